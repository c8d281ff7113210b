"""The convolution and the gates in front of the gated delta rule against 64 bits.

Tolerances: a convolved value is a sum of at most 16 products in 32 bits, whose error is 17 units (2^-24) of the sum of the
products' sizes at most; silu has a slope below 1.1 and adds a few units of its own.  Stored in bfloat16 it lies between the
roundings of the two ends of that range.  The gates are five operations of a few units each, the first of them a sum that may cancel: its units count
against the sizes of its terms."""
import pytest
import torch

import plain_delta as plain

pytestmark = pytest.mark.gpu
UNIT = 2.0 ** -24


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class Case:
    def __init__(self, lengths, channels, heads, taps, dtype, lead=0, gap=0, tile=64, slots=None, tail_off=16):
        g = torch.Generator(device="cuda").manual_seed(channels + taps)
        rand = lambda *shape: torch.randn(shape, generator=g, device="cuda")
        self.lengths, self.channels, self.heads, self.taps, self.lead = lengths, channels, heads, taps, lead
        self.tile, self.tail_off, self.items = tile, tail_off, len(lengths)
        self.a_off = lead + channels + gap
        self.slots = slots or list(range(self.items, 0, -1))
        tokens = sum(lengths)
        self.proj = (2 * rand(tokens, lead + channels + gap + 2 * heads)).to(dtype)
        self.state = rand(self.items + 2, tail_off + (taps - 1) * channels + gap)
        self.conv, self.a_log, self.dt_bias = rand(taps, channels), rand(heads), 3 * rand(heads) - 3
        self.starts = [sum(lengths[:i]) for i in range(self.items)]

    def run(self, portions=None, early=False):
        from from_scratch_inference_engine_b200.kernels import ops
        tokens = len(self.proj)
        act = torch.full((tokens, self.channels), 5.0, dtype=self.proj.dtype, device="cuda")
        decay, beta = (torch.full((tokens, self.heads), 5.0, device="cuda") for _ in range(2))
        state, done = self.state.clone(), [0] * self.items
        for part in portions or [self.lengths]:
            tiles = [(i, r) for i, n in enumerate(part) for r in range(0, max(n, 1), self.tile)]
            torch.cuda.synchronize()
            ops.delta_prep(self.proj, self.lead, self.a_off, self.a_off + self.heads,
                           ints([s + d for s, d in zip(self.starts, done)]), ints(part), ints(self.slots), self.items,
                           ints([i for i, _ in tiles]), ints([r for _, r in tiles]), len(tiles), self.tile, state, self.tail_off,
                           self.conv, self.a_log, self.dt_bias, act, decay, beta, early=early)
            done = [d + n for d, n in zip(done, part)]
        return act, decay, beta, state

    def check(self, **given):
        act, decay, beta, state = self.run(**given)
        tails = self.state.double()
        for start, n, slot in zip(self.starts, self.lengths, self.slots):
            rows = slice(start, start + n)
            if slot < 0:
                assert (act[rows] == 5).all() and (decay[rows] == 5).all() and (beta[rows] == 5).all()
                continue
            inputs = self.proj[rows, self.lead:self.lead + self.channels]
            held = slice(self.tail_off, self.tail_off + (self.taps - 1) * self.channels)
            before = self.state[slot, held].view(self.taps - 1, self.channels)
            want, left = plain.convolved(inputs, before, self.conv)
            sizes = sum(self.conv[j].double().abs() * torch.cat([before, inputs.float()]).double().abs()[j:j + n]
                        for j in range(self.taps))
            slack = 24 * UNIT * sizes + 8 * UNIT * want.abs() + 1e-38
            low, high = (want - slack).to(act.dtype), (want + slack).to(act.dtype)
            assert ((act[rows] >= low) & (act[rows] <= high)).all()
            tails[slot, held] = left.reshape(-1)
            a, b = (self.proj[rows, o:o + self.heads].double() for o in (self.a_off, self.a_off + self.heads))
            want_decay, want_beta = plain.gates(a, b, self.a_log, self.dt_bias)
            slack = (16 + 2 * (a.abs() + self.dt_bias.double().abs())) * UNIT
            least = 2.0 ** -126 * self.a_log.double().exp()         # below 2^-126 float32 has fewer bits
            assert ((decay[rows].double() - want_decay).abs() <= slack * want_decay.abs() + least).all()
            assert ((beta[rows].double() - want_beta).abs() <= (8 + 2 * b.abs()) * UNIT * want_beta).all()
        assert torch.equal(state.double(), tails)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lengths,channels,heads,taps", [
    ([1], 64, 2, 4), ([1] * 9, 520, 3, 4), ([2, 1, 3, 64, 65, 130], 72, 5, 4), ([7, 8, 9], 1100, 1, 3), ([100], 1024, 8, 2),
    ([5, 70], 33, 2, 4), ([20], 60, 2, 3), ([66, 1], 40, 2, 5), ([17], 24, 2, 16), ([9, 3], 16, 4, 1)])
def test_against_64_bits(lengths, channels, heads, taps, dtype):
    Case(lengths, channels, heads, taps, dtype).check()


@pytest.mark.parametrize("lead,gap,tail_off", [(8, 8, 0), (3, 1, 5), (8, 5, 4), (0, 0, 2)])
def test_columns_and_slots_at_any_place(lead, gap, tail_off):
    for dtype in (torch.bfloat16, torch.float32):
        Case([30, 3], 64, 3, 4, dtype, lead=lead, gap=gap, tail_off=tail_off).check()


@pytest.mark.parametrize("taps", [4, 5])
def test_short_tiles_padding_and_empty_requests(taps):
    Case([10, 1, 0, 31], 64, 2, taps, torch.bfloat16, tile=max(4, taps - 1), slots=[2, -1, 4, 0]).check()


@pytest.mark.parametrize("taps", [3, 6])
def test_cut_into_portions(taps):
    case = Case([40, 9], 64, 2, taps, torch.bfloat16)
    whole = case.run()
    for early in (False, True):
        parts = case.run(portions=[[1, 0], [1, 2], [16, 1], [22, 6]], early=early)
        for got, want in zip(parts, whole):
            assert torch.equal(got, want)
    case.check()


def test_large_and_infinite_inputs():
    case = Case([12], 64, 4, 4, torch.float32)
    case.proj[3, case.a_off:case.a_off + 4] = torch.tensor([100.0, -100.0, 30.0, -30.0], device="cuda")
    case.proj[4, case.a_off + 4:] = torch.tensor([200.0, -80.0, 40.0, -40.0], device="cuda")
    case.check()
    case.proj[5, 7] = float("inf")
    act = case.run()[0]
    want = case.conv[3, 7] > 0
    assert torch.isfinite(act[:5]).all() and torch.isfinite(act[:, :7]).all() and torch.isfinite(act[9:]).all()
    assert bool(torch.isinf(act[5, 7]) if want else torch.isnan(act[5, 7]) or act[5, 7] == 0)


def test_refusals():
    from from_scratch_inference_engine_b200.kernels import ops
    case = Case([4], 32, 2, 4, torch.float32)
    act, decay, beta = torch.empty(4, 32, device="cuda"), torch.empty(4, 2, device="cuda"), torch.empty(4, 2, device="cuda")

    def call(proj=case.proj, conv_off=0, a_off=32, b_off=34, lists=(ints([0]), ints([4]), ints([1])), items=1,
             segs=(ints([0]), ints([0])), count=1, tile=64, state=case.state, tail_off=16, conv=case.conv, a_log=case.a_log,
             dt_bias=case.dt_bias, act=act, decay=decay, beta=beta):
        ops.delta_prep(proj, conv_off, a_off, b_off, *lists, items, *segs, count, tile, state, tail_off, conv, a_log, dt_bias, act,
                       decay, beta)
    call()
    for wrong in (dict(proj=case.proj.half()), dict(act=act.bfloat16()), dict(conv_off=8), dict(b_off=35), dict(a_off=-1),
                  dict(items=2), dict(count=2), dict(tile=2), dict(state=None), dict(tail_off=17), dict(conv=case.conv.double()),
                  dict(conv=torch.zeros(17, 32, device="cuda"), state=torch.zeros(3, 600, device="cuda"), tile=64),
                  dict(dt_bias=case.dt_bias[:1]), dict(decay=decay[:3]), dict(act=act[:2])):
        with pytest.raises(ops.KernelError if wrong.get("state", 0) is not None else (ops.KernelError, AttributeError)):
            call(**wrong)
