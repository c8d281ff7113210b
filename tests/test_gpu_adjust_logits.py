"""Histories of tokens, and logits changed by penalties, biases and masks, against the formulas in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
NINF = -math.inf


def ops():
    from from_scratch_inference_engine_b200.kernels import ops as module
    return module


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def flag():
    return ints([0])


def packed(bits):
    """[rows, n] truth values (host) as words of 32 on the device."""
    rows, n = bits.shape
    wide = torch.zeros(rows, -(-n // 32) * 32, dtype=torch.long)
    wide[:, :n] = bits.long()
    words = (wide.view(rows, -1, 32) << torch.arange(32)).sum(-1)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).int().cuda()


def unpacked(words, n):
    return ((words.cpu()[:, :, None] >> torch.arange(32)) & 1).bool().flatten(1)[:, :n]


def expected(logits, slots, penalties, counts, held, bias, mask_of, allowed):
    """Row by row and token by token in 64 bits; how far 32 bits may be off beside it."""
    z, bound = logits.double().cpu().clone(), torch.zeros_like(logits, dtype=torch.float64).cpu()
    half = torch.finfo(torch.float32).eps / 2
    for r in range(z.shape[0]):
        s = slots[r]
        if s >= 0:
            theta, presence, frequency = (float(p) for p in penalties[r])
            n, h = counts[s].double(), held[s]
            first = torch.where(z[r] > 0, z[r] / theta, z[r] * theta)
            second = first - presence * (n > 0)
            third = second - frequency * n
            # one rounding each of the scaled logit, of its difference from presence, of frequency * count, of the last difference
            size = first.abs() + second.abs() + (frequency * n).abs() + third.abs()
            z[r] = torch.where(h, third, z[r])
            bound[r] = torch.where(h, half * size * (1 + 1e-6), bound[r])
        for token, value in bias[r]:
            z[r, token] += value
            bound[r, token] += half * abs(float(z[r, token])) * (1 + 1e-6)
        if mask_of[r] >= 0:
            z[r, ~allowed[mask_of[r]]] = NINF
    return z, bound


def compare(got, want, bound):
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    finite = torch.isfinite(want)
    rest = ~finite & ~torch.isnan(want)
    assert torch.equal(got[rest], want[rest])
    bound = torch.nan_to_num(bound, nan=math.inf)
    assert (torch.isfinite(got) | ~finite).all() and ((got - want)[finite].abs() <= bound[finite]).all()


def problem(rows, vocab, histories, masks, biases, seed):
    g = torch.Generator().manual_seed(seed)
    logits = torch.randn(rows, vocab, generator=g) * 4
    held = torch.rand(histories, vocab, generator=g) < 0.3
    counts = (held & (torch.rand(histories, vocab, generator=g) < 0.5)) * torch.randint(1, 9, (histories, vocab), generator=g)
    penalties = torch.stack([0.5 + torch.rand(rows, generator=g) * 1.5, torch.randn(rows, generator=g),
                             torch.rand(rows, generator=g)], 1)
    penalties[::3] = torch.tensor([1.0, 0.0, 0.0])
    slots = torch.randint(-1, max(histories, 1), (rows,), generator=g).tolist() if histories else [-1] * rows
    allowed = torch.rand(masks, vocab, generator=g) < 0.5
    if masks > 1:
        allowed[0] = False                                     # nothing is left
        allowed[1] = True
    mask_of = torch.randint(-1, masks, (rows,), generator=g).tolist() if masks else [-1] * rows
    bias = []
    for r in range(rows):
        n = min(vocab, int(torch.randint(0, biases + 1, (1,), generator=g)))
        tokens = sorted(torch.randperm(vocab, generator=g)[:n].tolist())
        bias.append([(t, float(v)) for t, v in zip(tokens, (torch.randn(n, generator=g) * 3).float().tolist())])
    return logits, held, counts.int(), penalties, slots, allowed, mask_of, bias


def device_bias(bias):
    starts = [0]
    for entries in bias:
        starts.append(starts[-1] + len(entries))
    flat = [e for entries in bias for e in entries]
    return ints(starts), ints([t for t, _ in flat]), torch.tensor([v for _, v in flat], dtype=torch.float32, device="cuda")


# vocabularies of one token, around a word, of a part of a block's tokens, odd ones, rows that start on no 16 bytes
@pytest.mark.parametrize("vocab", [1, 3, 31, 32, 33, 4095, 4096, 4097, 5000, 12291])
@pytest.mark.parametrize("rows,histories,masks,biases", [(1, 1, 0, 0), (3, 0, 3, 0), (5, 0, 0, 40), (7, 4, 3, 300), (2, 2, 2, 1)])
def test_against_the_formula(vocab, rows, histories, masks, biases):
    logits, held, counts, penalties, slots, allowed, mask_of, bias = problem(rows, vocab, histories, masks, biases, vocab + rows)
    want, bound = expected(logits, slots, penalties, counts, held, bias, mask_of, allowed)
    got, error = logits.cuda(), flag()
    out = ops().adjust_logits(got, error, ints(slots) if histories else None, penalties.cuda() if histories else None,
                              counts.cuda() if histories else None, packed(held) if histories else None,
                              device_bias(bias) if biases else None, (ints(mask_of), packed(allowed)) if masks else None)
    assert out is got and int(error) == 0
    compare(got, want, bound)


def test_infinities_and_nan():
    """A mask wins over everything, a forbidden token is -inf whatever its logit, bias or history holds."""
    vocab = 40
    special = [math.inf, NINF, math.nan, 0.0, -0.0, 3.4e38, -3.4e38, torch.finfo(torch.float32).min]
    row = torch.tensor([special + [1.0] * (vocab - len(special))] * 2)
    held = torch.ones(1, vocab, dtype=torch.bool)
    counts = torch.ones(1, vocab, dtype=torch.int32)
    penalties = torch.tensor([[2.0, 0.5, 0.25], [2.0, 0.5, 0.25]])
    allowed = torch.zeros(1, vocab, dtype=torch.bool)
    allowed[0, 8:] = True
    bias = [[(9, math.inf), (10, NINF), (11, 3.0)], [(0, math.inf), (1, 5.0), (2, math.nan), (9, 2.0)]]
    want, bound = expected(row, [0, 0], penalties, counts, held, bias, [-1, 0], allowed)
    got, error = row.cuda(), flag()
    ops().adjust_logits(got, error, ints([0, 0]), penalties.cuda(), counts.cuda(), packed(held), device_bias(bias),
                        (ints([-1, 0]), packed(allowed)))
    # 3.4e38 halves, its negative doubles beyond 32 bits
    assert want[0, 6] == -6.8e38 * 1.0 - 0.75 or want[0, 6] < -6e38
    want[0, 6], want[0, 7] = NINF, NINF
    assert int(error) == 0
    compare(got, want, bound)
    assert (got[1, :8] == NINF).all()


def test_what_does_not_fit_is_left_out_and_reported():
    vocab = 70
    logits = torch.randn(2, vocab)
    held, counts = torch.ones(1, vocab, dtype=torch.bool), torch.ones(1, vocab, dtype=torch.int32)
    penalties = torch.tensor([[1.5, 0.0, 0.0]] * 2)
    none = [[], []]
    for case in ("history", "mask", "token", "order", "twice", "starts"):
        slots, mask_of, code = [0, -1], [-1, 0], 0
        bias = [[(1, 1.0), (4, 2.0)], [(0, 1.0)]]
        seen_slots, use_bias = list(slots), bias
        allowed = torch.ones(1, vocab, dtype=torch.bool)
        starts = None
        if case == "history":
            slots, seen_slots, code = [0, 1], [0, -1], 6
        elif case == "mask":
            mask_of, code = [-1, 1], 6
        elif case == "token":
            bias, use_bias, code = [[(1, 1.0), (vocab, 2.0)], [(-1, 1.0)]], [[(1, 1.0)], []], 1
        elif case == "order":
            bias, use_bias, code = [[(4, 1.0), (1, 2.0)], []], [[(4, 1.0)], []], 5
        elif case == "twice":
            bias, use_bias, code = [[(4, 1.0), (4, 2.0)], []], [[(4, 1.0)], []], 5
        elif case == "starts":
            starts = ints([-5, 2, 1000])                       # beyond the lists: what there is
        want, bound = expected(logits, seen_slots, penalties, counts, held, use_bias, [-1, -1], allowed)
        got, error = logits.cuda(), flag()
        lists = device_bias(bias)
        ops().adjust_logits(got, error, ints(slots), penalties.cuda(), counts.cuda(), packed(held),
                            (lists[0] if starts is None else starts, *lists[1:]), (ints(mask_of), packed(allowed)))
        assert int(error) == code, case
        compare(got, want, bound)
    assert none


def test_a_token_twice_in_a_bias_that_is_out_of_order():
    """What is above the one in front of it counts, one after the other: 32-bit sums in the order of the list."""
    vocab, low, high = 9000, 3, 8500
    values = torch.randn(1001, generator=torch.Generator().manual_seed(4))
    for tokens in ([high, low] * 500 + [high], [low, high] * 500 + [low], [low, high, low + 1] * 333, [high, low, high]):
        bias = [[(t, float(v)) for t, v in zip(tokens, values)], [(t, 1.0) for t in range(0, vocab, 10)]]
        want = torch.zeros(2, vocab)
        for i, (token, value) in enumerate(bias[0]):
            if i == 0 or tokens[i - 1] < token:
                want[0, token] += value                        # (a 32-bit sum)
        want[1, ::10] = 1
        for _ in range(5):
            got, error = torch.zeros(2, vocab, device="cuda"), flag()
            ops().adjust_logits(got, error, bias=device_bias(bias))
            assert int(error) == 5 and torch.equal(got.cpu(), want)


def test_nothing_around_the_rows_is_written():
    around = torch.full((5, 101), 7.0, device="cuda")
    held, counts = torch.ones(1, 101, dtype=torch.bool), torch.full((1, 101), 2, dtype=torch.int32)
    allowed = torch.zeros(1, 101, dtype=torch.bool)
    allowed[0, 100] = True
    ops().adjust_logits(around[2:3], flag(), ints([0]), torch.tensor([[2.0, 1.0, 0.5]], device="cuda"), counts.cuda(),
                        packed(held), None, (ints([0]), packed(allowed)))
    assert (around[:2] == 7).all() and (around[3:] == 7).all()
    assert (around[2, :100] == NINF).all() and float(around[2, 100]) == 7 / 2 - 1 - 1


@pytest.mark.parametrize("n,slots,vocab,generated", [(1, 1, 1, True), (70, 5, 33, True), (3000, 3, 2, True), (500, 9, 1001, False),
                                                     (20000, 40, 5003, True)])
def test_counts(n, slots, vocab, generated):
    g = torch.Generator().manual_seed(n)
    tokens, of = torch.randint(0, vocab, (n,), generator=g), torch.randint(-1, slots, (n,), generator=g)
    counts = torch.randint(0, 5, (slots, vocab), generator=g).int()
    held = torch.rand(slots, vocab, generator=g) < 0.1
    got_counts, got_seen, error = counts.cuda(), packed(held), flag()
    ops().count_tokens(tokens.int().cuda(), of.int().cuda(), got_counts, got_seen, error, generated=generated)
    for t, s in zip(tokens.tolist(), of.tolist()):
        if s >= 0:
            counts[s, t] += int(generated)
            held[s, t] = True
    assert torch.equal(got_counts.cpu(), counts) and torch.equal(unpacked(got_seen, vocab), held) and int(error) == 0


def test_counts_outside():
    counts, seen = torch.zeros(2, 33, dtype=torch.int32, device="cuda"), torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    for token, slot, code in ((33, 0, 1), (-1, 1, 1), (2 ** 31 - 1, 0, 1), (0, 2, 6), (0, 2 ** 31 - 1, 6), (40, -1, 0)):
        error = flag()
        ops().count_tokens(ints([token, 32]), ints([slot, 1]), counts, seen, error)
        assert int(error) == code
    assert int(counts.sum()) == 6 and int(counts[1, 32]) == 6 and int((seen != 0).sum()) == 1


def test_histories_beyond_2_31_counts():
    """Offsets of the counts pass 32 bits."""
    vocab, slots = 152064, 14200
    counts = torch.zeros(slots, vocab, dtype=torch.int32, device="cuda")
    seen = torch.zeros(slots, vocab // 32, dtype=torch.int32, device="cuda")
    error = flag()
    ops().count_tokens(ints([151000, 151000]), ints([14199, 14199]), counts, seen, error)
    logits = torch.full((1, vocab), 2.0, device="cuda")
    ops().adjust_logits(logits, error, ints([14199]), torch.tensor([[2.0, 0.0, 0.25]], device="cuda"), counts, seen)
    assert int(counts[14199, 151000]) == 2 and float(logits[0, 151000]) == 0.5 and int(error) == 0
    assert int((logits == 2).sum()) == vocab - 1


def test_replayed_in_a_graph_and_on_another_stream():
    rows, vocab = 3, 5001
    logits, held, counts, penalties, slots, allowed, mask_of, bias = problem(rows, vocab, 2, 2, 20, 5)
    slots = [0, 1, 0]
    state = [logits.cuda(), flag(), ints(slots), penalties.cuda(), counts.cuda(), packed(held), device_bias(bias),
             (ints(mask_of), packed(allowed))]
    token = ints([17, 4000, 17])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops().adjust_logits(*state)                            # (the library is loaded, the logits start anew below)
        state[0].copy_(logits)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops().adjust_logits(*state)
        ops().count_tokens(token, state[2], state[4], state[5], state[1])
    for _ in range(3):
        state[0].copy_(logits)
        want, bound = expected(logits, slots, penalties, counts, held, bias, mask_of, allowed)
        graph.replay()
        compare(state[0], want, bound)
        for t, s in zip(token.tolist(), slots):
            counts[s, t] += 1
            held[s, t] = True
        assert torch.equal(state[4].cpu(), counts) and torch.equal(unpacked(state[5], vocab), held)


def test_refusals():
    o = ops()
    logits, error = torch.zeros(2, 64, device="cuda"), flag()
    counts, seen = torch.zeros(3, 64, dtype=torch.int32, device="cuda"), torch.zeros(3, 2, dtype=torch.int32, device="cuda")
    slots, penalties = ints([0, 1]), torch.ones(2, 3, device="cuda")
    start, token, value = ints([0, 1, 1]), ints([3]), torch.ones(1, device="cuda")
    good = (slots, penalties, counts, seen)
    bad = [(logits.double(), error), (logits[:, ::2], error), (logits[0], error), (logits.cpu(), error), (logits, error.long()),
           (logits, error, slots), (logits, error, slots, penalties, counts), (logits, error, slots[:1], *good[1:]),
           (logits, error, slots, penalties[:, :2].contiguous(), counts, seen), (logits, error, slots, penalties, counts[:2], seen),
           (logits, error, slots, penalties, counts[:, :32].contiguous(), seen[:, :1].contiguous()),
           (logits, error, None, None, None, None, (start[:2], token, value)), (logits, error, None, None, None, None, (start, token, value[:0])),
           (logits, error, None, None, None, None, (start, token, value.double())),
           (logits, error, None, None, None, None, None, (slots, seen[:, :1].contiguous())),
           (logits, error, None, None, None, None, None, (slots[:1], seen))]
    for args in bad:
        with pytest.raises(o.KernelError):
            o.adjust_logits(*args)
    for args in [(slots, slots[:1], counts, seen, error), (slots.float(), slots, counts, seen, error), (slots, slots, counts, seen[:2], error),
                 (slots, slots, counts, seen.cpu(), error), (slots[None], slots[None], counts, seen, error)]:
        with pytest.raises(o.KernelError):
            o.count_tokens(*args)
    before = logits.clone()
    o.adjust_logits(logits, error)                             # nothing asked for
    o.adjust_logits(logits[:0], error, slots[:0], penalties[:0], counts, seen)
    o.adjust_logits(logits, error, None, None, None, None, (ints([0, 0, 0]), token[:0], value[:0]), (ints([-1, -1]), seen[:0]))
    o.count_tokens(slots[:0], slots[:0], counts, seen, error)
    assert torch.equal(logits, before) and int(error) == 0
