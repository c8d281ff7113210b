"""Calls of the gated delta rule and of what stands in front of it one behind the other, with nothing in between that would let
one finish first: every call's results are those, bit for bit, that it has when each kernel is waited for."""
import pytest
import torch

from test_gpu_delta_rule import ints

pytestmark = pytest.mark.gpu
TILE = 64
STEPS = {"mixed": [90] + [1] * 33 + [3] * 5, "short first": [1] * 40 + [260], "many long": [40, 33, 1, 64, 2, 100, 1],
         "decoded": [1] * 70}


class Chain:
    """A few projections, each run through the convolution into the SAME buffers and through the rule, on states that every step
    carries on."""

    def __init__(self, lengths, dtype, dim, vdim, steps=6, heads=4, share=2, taps=4):
        g = torch.Generator(device="cuda").manual_seed(len(lengths) + dim)
        rand = lambda *shape: torch.randn(shape, generator=g, device="cuda")
        self.lengths, self.heads, self.share, self.dim, self.vdim, self.taps = lengths, heads, share, dim, vdim, taps
        self.qk = heads // share * dim
        self.channels = 2 * self.qk + heads * vdim
        self.tokens, self.items = sum(lengths), len(lengths)
        width = -(-(self.channels + 2 * heads) // 8) * 8
        # every step's values have their own size: what another step's call read by mistake would show
        self.projections = [(rand(self.tokens, width) * (1 + i)).to(dtype) for i in range(steps)]
        self.conv, self.a_log, self.dt_bias = rand(taps, self.channels) / 2, rand(heads), rand(heads) - 2
        starts = [sum(lengths[:i]) for i in range(self.items)]
        self.lists = ints(starts), ints(lengths), ints(list(range(self.items, 0, -1)))
        tiles = [(i, r) for i, n in enumerate(lengths) for r in range(0, n, TILE)]
        self.tiles = ints([i for i, _ in tiles]), ints([r for _, r in tiles])
        self.matrix = heads * dim * vdim
        self.state = rand(self.items + 2, -(-(self.matrix + (taps - 1) * self.channels) // 8) * 8) * 0.1
        self.dtype, self.early, self.ones = dtype, False, 0

    def run(self, wait, early, ones):
        from from_scratch_inference_engine_b200.kernels import ops
        state = self.state.clone()
        act = torch.zeros(self.tokens, self.channels, dtype=self.dtype, device="cuda")
        decay, beta = torch.zeros(self.tokens, self.heads, device="cuda"), torch.zeros(self.tokens, self.heads, device="cuda")
        outs = [torch.zeros(self.tokens, self.heads * self.vdim, device="cuda") for _ in self.projections]
        torch.cuda.synchronize()
        for proj, out in zip(self.projections, outs):
            ops.delta_prep(proj, 0, self.channels, self.channels + self.heads, *self.lists, self.items, *self.tiles,
                           self.tiles[0].numel(), TILE, state, self.matrix, self.conv, self.a_log, self.dt_bias, act, decay,
                           beta, early=early)
            if wait:
                torch.cuda.synchronize()
            ops.gated_delta_rule(act, 0, self.qk, 2 * self.qk, decay, beta, *self.lists, self.items, state, out, self.heads,
                                 self.dim, self.vdim, share=self.share, longest=max(self.lengths), early=early, ones=ones)
            if wait:
                torch.cuda.synchronize()
        return outs, state


@pytest.mark.parametrize("dtype,dim,vdim", [(torch.bfloat16, 128, 128), (torch.bfloat16, 64, 64), (torch.float32, 48, 36)])
@pytest.mark.parametrize("step", list(STEPS))
def test_call_behind_call(step, dtype, dim, vdim):
    chain = Chain(STEPS[step], dtype, dim, vdim)
    told = sum(n <= 1 for n in chain.lengths)
    for ones in sorted({0, told}):
        want, want_state = chain.run(True, False, ones)
        for early in (False, True):
            for _ in range(10):
                got, state = chain.run(False, early, ones)
                assert all(torch.equal(a, b) for a, b in zip(got, want))
                assert torch.equal(state, want_state)


def test_call_behind_call_in_a_graph():
    """The same recorded once and replayed: the word that the launches hand on is cleared every time."""
    chain = Chain(STEPS["mixed"], torch.bfloat16, 64, 64)
    want, want_state = chain.run(True, False, 33)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        from from_scratch_inference_engine_b200.kernels import ops
        state = chain.state.clone()
        act = torch.zeros(chain.tokens, chain.channels, dtype=chain.dtype, device="cuda")
        decay, beta = (torch.zeros(chain.tokens, chain.heads, device="cuda") for _ in range(2))
        outs = [torch.zeros(chain.tokens, chain.heads * chain.vdim, device="cuda") for _ in chain.projections]
        room = torch.empty(ops.gated_delta_room(chain.tokens, chain.items, chain.heads, chain.dim, chain.dtype, chain.share),
                           dtype=torch.uint8, device="cuda")

        def step():
            for proj, out in zip(chain.projections, outs):
                ops.delta_prep(proj, 0, chain.channels, chain.channels + chain.heads, *chain.lists, chain.items, *chain.tiles,
                               chain.tiles[0].numel(), TILE, state, chain.matrix, chain.conv, chain.a_log, chain.dt_bias, act,
                               decay, beta, early=True)
                ops.gated_delta_rule(act, 0, chain.qk, 2 * chain.qk, decay, beta, *chain.lists, chain.items, state, out,
                                     chain.heads, chain.dim, chain.vdim, share=chain.share, longest=90, early=True, ones=33,
                                     room=room)
        step()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
        for _ in range(5):
            state.copy_(chain.state)
            graph.replay()
            stream.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, want)) and torch.equal(state, want_state)
