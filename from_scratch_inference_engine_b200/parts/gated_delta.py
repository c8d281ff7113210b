"""The gated delta rule as a mixer: a recurrence over a matrix per head from which a key takes out what it already holds
before its new value goes in."""

from __future__ import annotations

from typing import Dict, List, Optional

import torch

from ..kernels import ops
from ..weights.tensor_spec import TensorSpec
from .base import LayerCache, Mixer, StateNeed, register_part


@register_part("mixer", "gated_delta_rule")
class GatedDeltaRule(Mixer):
    """q, k = W_q y, W_k y [qk_heads, dim], v = W_v y [heads, vdim], each column through a short causal convolution of
    `taps` tokens and silu; per head a decay a = exp(-exp(A_log) softplus(W_a y + dt_bias)) and a step size
    b = sigmoid(W_b y); with q and k divided by their lengths, per head

        u_t = b_t (v_t - a_t S_(t-1)^T k_t)     S_t = a_t S_(t-1) + k_t u_t^T     o_t = S_t^T q_t * dim^(-1/2)

    heads / qk_heads heads in a row read the same q and k.  Every head of o is divided by its root mean square (`eps`
    inside the root, as inside the lengths' root), multiplied by a gain of vdim numbers that all heads share and by
    silu(W_g y), and the heads pass the output projection.

    Per request the slot holds S [heads, dim, vdim] and, behind it, the convolution's inputs of the last taps - 1 tokens;
    both are float32, zero when a request starts, and carried from step to step.  Gates, recurrence, norm and gate are 32-bit
    in both compute dtypes; the convolved q, k and v are stored as all activations are.  All projections of y are one
    matrix product over the stacked weight.  `names` gives the tensor names below the prefix.
    """

    capturable = True
    PREP_TOKENS = 64

    NAMES = {"q": "q", "k": "k", "v": "v", "gate": "g", "decay": "a", "step": "b", "conv": "conv", "a_log": "A_log",
             "dt_bias": "dt_bias", "norm": "norm", "o": "o"}

    def __init__(self, prefix: str, hidden_size: int, heads: int, dim: int, vdim: int, taps: int, eps: float,
                 qk_heads: Optional[int] = None, names: Optional[Dict[str, str]] = None):
        self.prefix, self.hidden_size = prefix, int(hidden_size)
        self.heads, self.dim, self.vdim = int(heads), int(dim), int(vdim)
        self.qk_heads = self.heads if qk_heads is None else int(qk_heads)
        self.taps, self.eps = int(taps), float(eps)
        if min(self.heads, self.qk_heads, self.dim, self.vdim) <= 0 or self.heads % self.qk_heads:
            raise ValueError("gated_delta_rule: heads, qk_heads, dim and vdim are positive and heads a multiple of qk_heads")
        if self.taps < 1 or self.eps <= 0:
            raise ValueError("gated_delta_rule: the convolution has at least one tap and eps is positive")
        self.qk_width, self.v_width = self.qk_heads * self.dim, self.heads * self.vdim
        self.channels = 2 * self.qk_width + self.v_width
        self.matrix_floats = self.heads * self.dim * self.vdim
        self.names = dict(self.NAMES)
        self.names.update(names or {})
        self.w_in = self.w_o = self.conv_by_tap = self.a_log = self.dt_bias = self.gain = None

    def tensor_specs(self) -> List[TensorSpec]:
        p, h, n = self.prefix, self.hidden_size, self.names
        return [TensorSpec(p + n["q"], (self.qk_width, h)), TensorSpec(p + n["k"], (self.qk_width, h)),
                TensorSpec(p + n["v"], (self.v_width, h)), TensorSpec(p + n["gate"], (self.v_width, h)),
                TensorSpec(p + n["decay"], (self.heads, h)), TensorSpec(p + n["step"], (self.heads, h)),
                TensorSpec(p + n["conv"], (self.channels, self.taps), role="vector", init="taps"),
                TensorSpec(p + n["a_log"], (self.heads,), role="vector", init="normal"),
                TensorSpec(p + n["dt_bias"], (self.heads,), role="vector", init="normal"),
                TensorSpec(p + n["norm"], (self.vdim,), role="vector", init="gain"),
                TensorSpec(p + n["o"], (h, self.v_width))]

    def state_need(self) -> Optional[StateNeed]:
        floats = self.matrix_floats + (self.taps - 1) * self.channels
        return StateNeed((-(-floats // 8) * 8,), torch.float32)      # slots start on 32 bytes

    def bind(self, tensors: Dict[str, torch.Tensor], runtime) -> None:
        self.runtime = runtime
        p, n = self.prefix, self.names
        if self.dim > ops.delta_max_dim():
            raise ValueError(f"gated_delta_rule: {self.dim} state rows per head, the kernels hold {ops.delta_max_dim()}")
        if self.taps > ops.delta_prep_max_taps():
            raise ValueError(f"gated_delta_rule: {self.taps} taps, the kernels hold {ops.delta_prep_max_taps()}")

        def vector(key):
            return tensors[p + n[key]].to(torch.float32).contiguous()
        stacked = [tensors[p + n[which]] for which in ("q", "k", "v", "gate", "decay", "step")]
        rows = sum(w.shape[0] for w in stacked)
        if rows % 8:                        # rows of the product's result start on 16 bytes
            stacked.append(torch.zeros(8 - rows % 8, self.hidden_size, dtype=stacked[0].dtype, device=stacked[0].device))
        self.w_in = torch.cat(stacked).contiguous()
        self.w_o = tensors[p + n["o"]].contiguous()
        self.conv_by_tap = vector("conv").t().contiguous()
        self.a_log, self.dt_bias, self.gain = vector("a_log"), vector("dt_bias"), vector("norm")
        runtime.prepare_weight(self.w_in)
        runtime.prepare_weight(self.w_o)

    def _room(self, tokens: int, requests: int) -> Optional[torch.Tensor]:
        size = ops.gated_delta_room(tokens, requests, self.heads, self.dim, self.runtime.dtype, self.heads // self.qk_heads)
        return self.runtime.buffer("gated_delta.room", 1, size, torch.uint8) if size else None

    def reserve(self, tokens: int, requests: int) -> None:
        self._room(tokens, requests)

    def forward(self, ctx, y: torch.Tensor, cache: LayerCache) -> torch.Tensor:
        rt = self.runtime
        tokens = y.shape[0]
        proj = rt.linear(y, self.w_in, None, "gated_delta.in")
        gate0 = self.channels
        decay0 = gate0 + self.v_width
        items = (ctx.item_qstart, ctx.item_qlen, ctx.item_slots, ctx.num_items)
        tiles = ctx.attention_tiles(1, self.PREP_TOKENS)
        act = rt.buffer("gated_delta.act", tokens, self.channels, proj.dtype)
        log_decay = rt.buffer("gated_delta.decay", tokens, self.heads, torch.float32)
        beta = rt.buffer("gated_delta.beta", tokens, self.heads, torch.float32)
        ops.delta_prep(proj, 0, decay0, decay0 + self.heads, *items, tiles.item, tiles.row0, tiles.count, self.PREP_TOKENS,
                       cache.state, self.matrix_floats, self.conv_by_tap, self.a_log, self.dt_bias, act, log_decay, beta,
                       early=True)
        o = rt.buffer("gated_delta.o", tokens, self.v_width, torch.float32)
        ops.gated_delta_rule(act, 0, self.qk_width, 2 * self.qk_width, log_decay, beta, *items, cache.state, o, self.heads,
                             self.dim, self.vdim, share=self.heads // self.qk_heads, eps=self.eps,
                             longest=ctx.longest, early=True, ones=ctx.ones,
                             room=self._room(tokens, ctx.num_items) if ctx.longest > 1 else None)
        gated = rt.buffer("gated_delta.gated", tokens, self.v_width, proj.dtype)
        ops.head_norm_silu(o, proj, gate0, self.gain, self.eps, gated, self.heads)
        return rt.linear(gated, self.w_o, None, "gated_delta.out")
