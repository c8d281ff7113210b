"""The gated delta rule against the formula in 64 bits, token by token.

Tolerances: the kernels work in 32 bits (unit 2^-24) and a token's step is a contraction of the state, so a rounding is not
amplified, only joined by those of the tokens that the state still remembers.  A step rounds sums of up to 256 products and
about ten single operations; with errors of either sign some 32 units of the result's 2-norm hold over a memory of a hundred
tokens, and 16 times that for a single number against the largest."""
import pytest
import torch

import plain_delta as plain

pytestmark = pytest.mark.gpu
UNIT = 2.0 ** -24
FEW, MANY = 1, 1 << 20           # what the caller says about the longest request: the recurrent form, the chunked one
CROWD = 1 << 21                  # the chunked one as among 400 more requests (padding entries): blocks share the SMs


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class Case:
    """Requests of `lengths` tokens at slots in no order, rows of q, k and v between other columns."""

    def __init__(self, lengths, heads, share, dim, vdim, dtype, seed=0, lead=8, gap=4, v_scale=1.0):
        g = torch.Generator(device="cuda").manual_seed(seed + 7 * dim + vdim)
        rand = lambda *shape: torch.randn(shape, generator=g, device="cuda")
        self.lengths, self.heads, self.share, self.dim, self.vdim = lengths, heads, share, dim, vdim
        self.tokens, self.narrow = sum(lengths), heads // share
        self.offs = (lead, lead + self.narrow * dim, lead + 2 * self.narrow * dim)
        width = lead + 2 * self.narrow * dim + heads * vdim + lead
        self.qkv = torch.nn.functional.silu(rand(self.tokens, width)).to(dtype)
        self.qkv[:, self.offs[2]:] *= v_scale
        self.decay = -torch.exp(rand(self.tokens, heads) - 2)
        self.beta = torch.sigmoid(rand(self.tokens, heads))
        self.items = len(lengths)
        self.slots = list(range(self.items, 0, -1))
        self.state = rand(self.items + 2, heads * dim * vdim + gap) * (0.1 * v_scale)
        self.starts = [sum(lengths[:i]) for i in range(self.items)]

    def run(self, longest, portions=None, early=False, scale=None, ones=0):
        """(out, state) of one call, or of one call per portion (lists of tokens per request)."""
        from from_scratch_inference_engine_b200.kernels import ops
        out = torch.full((self.tokens, self.heads * self.vdim), 7e7, device="cuda")
        state = self.state.clone()
        done = [0] * self.items
        padding = 400 if longest == CROWD else 0
        for part in portions or [self.lengths]:
            torch.cuda.synchronize()
            ops.gated_delta_rule(self.qkv, *self.offs, self.decay, self.beta,
                                 ints([s + d for s, d in zip(self.starts, done)] + [0] * padding), ints(part + [0] * padding),
                                 ints(self.slots + [-1] * padding), self.items + padding, state, out, self.heads, self.dim,
                                 self.vdim, share=self.share, scale=scale, longest=longest, early=early, ones=ones)
            done = [d + n for d, n in zip(done, part)]
        return out, state

    def want(self, scale=None, eps=1e-6):
        h, n, d, w = self.heads, self.narrow, self.dim, self.vdim
        q, k = (self.qkv[:, o:o + n * d].reshape(-1, n, d).repeat_interleave(self.share, 1) for o in self.offs[:2])
        v = self.qkv[:, self.offs[2]:self.offs[2] + h * w].reshape(-1, h, w)
        out = torch.full((self.tokens, h * w), 7e7, dtype=torch.float64, device="cuda")
        state = self.state.double()
        for start, length, slot in zip(self.starts, self.lengths, self.slots):
            if slot < 0:
                continue
            rows = slice(start, start + length)
            o, s = plain.rule(q[rows], k[rows], v[rows], self.decay[rows], self.beta[rows],
                              self.state[slot, :h * d * w].view(h, d, w), d ** -0.5 if scale is None else scale, eps)
            out[rows] = o.reshape(-1, h * w)
            state[slot, :h * d * w] = s.reshape(-1)
        return out, state


def near(got, want, units=32):
    error, size = (got.double() - want).norm(), want.norm()
    assert error <= units * UNIT * size, f"2-norm off by {float(error / size / UNIT):.1f} units"
    assert (got.double() - want).abs().max() <= 16 * units * UNIT * want.abs().max()


def check(case, longest, units=32, **given):
    for got, want in zip(case.run(longest, **given), case.want(**{k: v for k, v in given.items() if k == "scale"})):
        near(got, want, units)


SIZES = [  # lengths, heads, share, dim, vdim: chunks that are full, begun, one token over; heads that fill tiles and do not
    ([32, 31, 33], 2, 1, 128, 128), ([64, 96, 65, 63], 2, 1, 64, 64), ([32], 3, 3, 80, 17),
    ([16], 2, 1, 128, 128), ([1], 3, 1, 64, 64), ([17, 1, 33], 4, 2, 128, 128), ([5, 64, 100, 15], 6, 3, 64, 64),
    ([200], 2, 1, 96, 80), ([31, 2], 2, 2, 32, 160), ([20, 9], 2, 1, 48, 32), ([18], 1, 1, 36, 20), ([40], 2, 1, 33, 19),
    ([7, 19], 2, 1, 100, 1), ([35], 1, 1, 1, 5), ([12, 3], 2, 1, 200, 64), ([9], 1, 1, 256, 36), ([130], 1, 1, 112, 256)]


@pytest.mark.parametrize("longest", [FEW, MANY, CROWD])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lengths,heads,share,dim,vdim", SIZES)
def test_against_the_formula(lengths, heads, share, dim, vdim, dtype, longest):
    check(Case(lengths, heads, share, dim, vdim, dtype), longest)


@pytest.mark.parametrize("longest", [FEW, MANY, CROWD])
@pytest.mark.parametrize("lead,gap", [(3, 1), (4, 2), (8, 3)])
def test_rows_and_slots_off_the_16_bytes(lead, gap, longest):
    check(Case([21, 34], 2, 1, 64, 64, torch.bfloat16, lead=lead, gap=gap), longest)
    check(Case([21, 34], 2, 1, 64, 64, torch.float32, lead=lead, gap=gap), longest)


@pytest.mark.parametrize("longest", [FEW, MANY, CROWD])
def test_gates_at_their_ends(longest):
    case = Case([50, 33], 3, 1, 64, 96, torch.bfloat16)
    case.decay[::3], case.decay[1::7], case.decay[5], case.decay[11] = 0.0, -1e4, -float("inf"), -40.0
    case.beta[::4], case.beta[1::4], case.beta[2::8] = 0.0, 1.0, 2.0
    check(case, longest)


@pytest.mark.parametrize("longest", [FEW, MANY, CROWD])
@pytest.mark.parametrize("beta", [1.0, 2.0])
def test_the_same_key_again_and_again(beta, longest):
    """Nothing decays and every key is the first one: a chunk's triangular system is as far from the unit matrix as it gets.
    With beta = 2 a token mirrors the state and nothing is ever forgotten, and one key has one rounding of its length (three
    units), which counts twice in every token's mirror and always to the same side: six units a token."""
    case = Case([70], 2, 1, 128, 64, torch.bfloat16)
    k = slice(case.offs[1], case.offs[2])
    case.qkv[:, k] = case.qkv[:1, k].clone()
    case.decay.zero_()
    case.beta.fill_(beta)
    check(case, longest, units=32 if beta < 2 else 32 + 6 * 70)


@pytest.mark.parametrize("longest", [FEW, MANY, CROWD])
def test_keys_and_queries_of_nothing_and_of_all_sizes(longest):
    case = Case([60], 2, 1, 64, 64, torch.float32)
    factor = torch.tensor([0.0, 1e-6, 1e-3, 1.0, 300.0, 1e9], device="cuda")[torch.arange(60, device="cuda") % 6]
    case.qkv[:, case.offs[0]:case.offs[2]] *= factor[:, None]
    check(case, longest)


@pytest.mark.parametrize("longest", [FEW, MANY, CROWD])
@pytest.mark.parametrize("v_scale", [1e-25, 1e-6, 1e4, 1e20])
def test_values_of_all_sizes(v_scale, longest):
    check(Case([70], 2, 1, 64, 64, torch.float32, v_scale=v_scale), longest)
    case = Case([70], 2, 1, 64, 64, torch.float32, v_scale=v_scale)
    check(case, longest, scale=1.0)


@pytest.mark.parametrize("longest", [FEW, MANY, CROWD])
def test_columns_of_all_sizes_side_by_side(longest):
    """Every column of the state has its own size: a column's error is measured against that column."""
    case = Case([90], 1, 1, 64, 64, torch.float32, lead=8)
    sizes = torch.logspace(-18, 18, 64, device="cuda")
    v = slice(case.offs[2], case.offs[2] + 64)
    case.qkv[:, v] *= sizes
    case.state[:, :64 * 64] *= sizes.repeat(64)
    (out, state), (want_out, want_state) = case.run(longest), case.want()
    for col in range(64):
        near(out[:, col], want_out[:, col])
        near(state[1, col:64 * 64:64], want_state[1, col:64 * 64:64])


@pytest.mark.parametrize("longest", [FEW, MANY, CROWD])
def test_memories_that_fade_by_many_orders(longest):
    """A large state that a few tokens forget, and small values behind it."""
    case = Case([64], 2, 1, 64, 64, torch.float32)
    case.state *= 100
    case.decay[3], case.decay[20:24] = -60.0, -9.0
    out, state = case.run(longest)
    want_out, want_state = case.want()
    for rows in (slice(0, 3), slice(3, 16), slice(16, 20), slice(20, 32), slice(32, 64)):
        near(out[rows], want_out[rows])
    near(state[1], want_state[1])


@pytest.mark.parametrize("longest", [FEW, MANY, CROWD])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_a_value_that_is_not_finite_stays_in_its_column_and_behind_its_token(bad, longest):
    case = Case([45, 20], 2, 1, 64, 64, torch.bfloat16)
    want_out, want_state = case.want()
    token, head, col = 21, 1, 13
    case.qkv[token, case.offs[2] + head * 64 + col] = bad
    out, state = case.run(longest)
    hit = torch.zeros(65, 128, dtype=torch.bool, device="cuda")
    hit[token:45, head * 64 + col] = True
    assert torch.equal(~torch.isfinite(out), hit)
    near(out[~hit], want_out[~hit])
    first = state[case.slots[0], :2 * 64 * 64].view(2, 64, 64)
    held = torch.zeros_like(first, dtype=torch.bool)
    held[head, :, col] = True
    assert torch.equal(~torch.isfinite(first), held)
    near(state[case.slots[1]], want_state[case.slots[1]])


@pytest.mark.parametrize("longest", [FEW, MANY, CROWD])
@pytest.mark.parametrize("which", ["q", "k", "decay", "beta", "state"])
def test_what_is_not_finite_reaches_no_token_before_it(which, longest):
    case = Case([45], 2, 1, 64, 64, torch.bfloat16)
    want_out, _ = case.want()
    token, head = 21, 1
    if which == "decay":
        case.decay[token, head] = float("nan")
    elif which == "beta":
        case.beta[token, head] = float("nan")
    elif which == "state":
        case.state[case.slots[0], 64 * 64 + 5 * 64 + 9] = float("inf")          # head 1, row 5, column 9
    else:
        case.qkv[token, case.offs["qk".index(which)] + head * 64 + 3] = float("nan")
    out, _ = case.run(longest)
    hit = torch.zeros(45, 2, 64, dtype=torch.bool, device="cuda")
    if which == "q":
        hit[token, head] = True
    elif which == "state":
        hit[:, head, 9] = True
    else:
        hit[token:, head] = True
    hit = hit.view(45, 128)
    assert torch.equal(~torch.isfinite(out), hit)
    near(out[~hit], want_out[~hit])


@pytest.mark.parametrize("longest", [FEW, MANY, CROWD])
def test_requests_without_slot_or_tokens_change_nothing(longest):
    case = Case([20, 18, 0, 5], 2, 1, 64, 64, torch.bfloat16)
    case.slots = [3, -1, 1, 5]
    out, state = case.run(longest)
    want_out, want_state = case.want()
    assert (out[20:38] == 7e7).all()
    near(out[:20], want_out[:20])
    near(out[38:], want_out[38:])
    near(state[3], want_state[3])
    near(state[5], want_state[5])
    for slot in (0, 1, 2, 4):
        assert torch.equal(state[slot], case.state[slot])
    assert torch.equal(state[:, 2 * 64 * 64:], case.state[:, 2 * 64 * 64:])      # what else the slots hold


@pytest.mark.parametrize("longest", [FEW, MANY, CROWD])
def test_cut_into_portions(longest):
    case = Case([50, 23], 2, 1, 128, 64, torch.bfloat16)
    check(case, longest, portions=[[17, 0], [1, 16], [32, 7]])


@pytest.mark.parametrize("longest", [FEW, MANY, CROWD])
def test_long_and_the_same_bits_again(longest):
    """More tokens than the chunked form walks between two looks at the state's size, twice, and behind an early launch."""
    case = Case([1100], 1, 1, 64, 32, torch.bfloat16)
    case.decay *= 0.01
    first, state = case.run(longest)
    near(first, case.want()[0])
    for early in (False, True):
        again, other = case.run(longest, early=early)
        assert torch.equal(first, again) and torch.equal(state, other)


@pytest.mark.parametrize("longest", [FEW, MANY, CROWD])
def test_on_another_stream(longest):
    case = Case([40], 2, 1, 64, 64, torch.bfloat16)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = case.run(longest)
    torch.cuda.current_stream().wait_stream(stream)
    for have, want in zip(got, case.run(longest)):
        assert torch.equal(have, want)


MIXED = [[1] * 40 + [70], [1] * 20 + [11, 10, 12, 9, 17, 16, 18, 15], [90] + [1] * 33, [1, 5, 2, 40, 1, 0, 4, 7, 3, 6, 100, 1, 1], [1, 33], [6, 7, 5, 4, 1, 6], [0, 0, 50, 0, 1]]


@pytest.mark.parametrize("told", [False, True])
@pytest.mark.parametrize("dtype,dim,vdim", [(torch.bfloat16, 128, 128), (torch.bfloat16, 48, 20), (torch.float32, 64, 96),
                                            (torch.float32, 40, 7)])
@pytest.mark.parametrize("lengths", MIXED)
def test_few_tokens_beside_long_requests(lengths, dtype, dim, vdim, told):
    """Requests of few tokens go the recurrent way beside the others, wherever in the lists they stand."""
    check(Case(lengths, 4, 2, dim, vdim, dtype), max(lengths), ones=sum(n <= 1 for n in lengths) if told else 0)


@pytest.mark.parametrize("early", [False, True])
def test_few_tokens_beside_long_requests_call_after_call(early):
    """Each call reads the states that both launches of the one before left."""
    case = Case([260] + [9] * 50, 8, 1, 64, 64, torch.bfloat16)
    portions = [[100] + [1] * 50, [60] + [2] * 50, [1] + [1] * 50, [99] + [5] * 50]
    for got, want in zip(case.run(MANY, portions=portions, early=early, ones=0), case.want()):
        near(got, want)


def test_few_tokens_beside_long_requests_without_slot():
    case = Case([1, 40, 1, 64, 1, 2], 2, 1, 64, 64, torch.bfloat16)
    case.slots[0] = case.slots[3] = case.slots[5] = -1
    for got, want in zip(case.run(64, ones=3), case.want()):
        near(got, want)


def test_refusals():
    from from_scratch_inference_engine_b200.kernels import ops
    case = Case([4], 4, 2, 32, 32, torch.float32)
    out, lists = torch.empty(4, 128, device="cuda"), (ints([0]), ints([4]), ints([1]))

    def call(qkv=case.qkv, offs=case.offs, decay=case.decay, beta=case.beta, lists=lists, items=1, state=case.state, out=out,
             heads=4, dim=32, vdim=32, **given):
        ops.gated_delta_rule(qkv, *offs, decay, beta, *lists, items, state, out, heads, dim, vdim, **{"share": 2, **given})
    call()
    for wrong in (dict(qkv=case.qkv.half()), dict(qkv=case.qkv.cpu()), dict(qkv=case.qkv.t()), dict(offs=(8, 72, 152)),
                  dict(offs=(-8, 72, 136)), dict(decay=case.decay[:, :2].contiguous()), dict(beta=case.beta.double()),
                  dict(lists=(lists[0].long(),) + lists[1:]), dict(items=2), dict(state=case.state[:, :100]),
                  dict(state=case.state.bfloat16()), dict(out=out[:3]), dict(out=out.bfloat16()), dict(heads=3), dict(share=3),
                  dict(dim=0), dict(dim=257, heads=1, share=1), dict(eps=0.0), dict(ones=2), dict(ones=-1)):
        with pytest.raises(ops.KernelError):
            call(**wrong)
