"""Greedy and temperature / top-k / top-p sampling on the device.

Options as the reference's `SamplingParams` (include/engine/sampler.hpp:9-13):
temperature (<= 0 selects the first largest logit), top_k (0 = off), top_p (>= 1 =
off), applied in that order (src/sampler/sampler.cpp:25-88).  Unlike the reference,
whose requests share one generator so that a request's tokens depend on what else is
in the batch (src/engine/engine.cpp:131-135), every draw here is a function of
(request seed, index of the output token): a request gives the same tokens alone, in
any batch, and when it is recomputed after a preemption.

Beyond the reference, before a token is chosen its row of logits is changed in place (`ops.adjust_logits`) by penalties for
tokens that the request's context holds, by a bias per token, and by the set of tokens that are allowed next, in this order.
"""

from __future__ import annotations

import operator
from dataclasses import dataclass
from typing import Callable, List, Mapping, Optional, Sequence, Tuple

import numpy as np
import torch

from ..kernels import ops

LEAST32, MOST32 = float(np.finfo(np.float32).tiny), float(np.finfo(np.float32).max)
_MASK = 0xFFFFFFFFFFFFFFFF


@dataclass
class SamplingParams:
    temperature: float = 1.0     # <= 0 selects greedy (argmax)
    top_k: int = 0               # 0 disables top-k
    top_p: float = 1.0           # >= 1 disables top-p (nucleus)
    seed: Optional[int] = None   # None: derived from the engine seed and the request id
    # of a token that prompt or answer hold: logit / penalty where it is above 0, else logit * penalty
    repetition_penalty: float = 1.0
    presence_penalty: float = 0.0     # taken from the logit of every token that the answer holds
    frequency_penalty: float = 0.0    # ... for every time that it does
    logit_bias: Optional[Mapping[int, float]] = None     # added to the logits of these tokens
    # Which tokens may come next, by the answer so far (a list that is not to be changed): their ids in any order, an array of a
    # bool per token of the vocabulary (the quickest for many), or None for all.  No token: the answer ends.  It is asked once per token, so a request with it has every step wait for the
    # token before.
    allowed: Optional[Callable[[Sequence[int]], Optional[Sequence[int]]]] = None

    @property
    def greedy(self) -> bool:
        return self.temperature <= 0.0

    @property
    def penalised(self) -> bool:
        return self.repetition_penalty != 1.0 or self.presence_penalty != 0.0 or self.frequency_penalty != 0.0

    def check(self, vocab: int) -> None:
        """ValueError where the options that change logits make no sense for this vocabulary, as the 32-bit numbers that they
        are applied as: a penalty that becomes infinite turns a count of zero into NaN, one that becomes zero a logit into inf."""
        if not LEAST32 <= self.repetition_penalty <= MOST32:
            raise ValueError(f"repetition_penalty must be positive and finite in 32 bits, not {self.repetition_penalty}")
        for name in ("presence_penalty", "frequency_penalty"):
            if not abs(getattr(self, name)) <= MOST32:
                raise ValueError(f"{name} must be finite in 32 bits, not {getattr(self, name)}")
        sorted_bias(self.logit_bias, vocab)
        if self.allowed is not None and not callable(self.allowed):
            raise ValueError("allowed must be a function of the answer so far")


def sorted_bias(bias: Optional[Mapping[int, float]], vocab: int) -> Optional[Tuple[np.ndarray, np.ndarray]]:
    """A bias per token as (ids in rising order, float32 values), None where there is none."""
    if not bias:
        return None
    try:
        tokens = np.asarray([operator.index(token) for token in bias], dtype=np.int64)
        values = np.asarray([float(value) for value in bias.values()], dtype=np.float32)
    except TypeError:
        raise ValueError("logit_bias: a number per token id is needed") from None
    if len(np.unique(tokens)) != len(tokens) or tokens.min() < 0 or tokens.max() >= vocab:
        raise ValueError(f"logit_bias: different token ids in [0, {vocab}) are needed")
    if not np.isfinite(values).all():
        raise ValueError("logit_bias: finite values are needed")
    order = np.argsort(tokens)
    return tokens[order].astype(np.int32), values[order]


def pack_allowed(tokens: Sequence[int], vocab: int) -> np.ndarray:
    """A set of tokens (their ids, or a bool per token of the vocabulary) as bits, int32 words: token v is bit v % 32 of word
    v // 32.  151,936 tokens of which a third are allowed, as bools 20 us, as an array of ids 100, as a list 1,400."""
    ids = np.asarray(tokens if isinstance(tokens, (np.ndarray, list, tuple)) else list(tokens))
    if isinstance(tokens, np.ndarray) and ids.dtype == bool and ids.shape == (vocab,):
        bits = np.zeros(32 * ops.bit_words(vocab), dtype=bool)
        bits[:vocab] = ids
        return np.packbits(bits, bitorder="little").view(np.int32)
    if ids.ndim != 1 or (ids.size and ids.dtype.kind not in "iu"):
        raise ValueError("allowed: a sequence of token ids is needed")
    if ids.size and (int(ids.min()) < 0 or int(ids.max()) >= vocab):
        raise ValueError(f"allowed: token ids must lie in [0, {vocab})")
    bits = np.zeros(32 * ops.bit_words(vocab), dtype=bool)
    bits[ids.astype(np.int64)] = True
    return np.packbits(bits, bitorder="little").view(np.int32)


def stage_changes(params: Sequence[SamplingParams], slots: Optional[Sequence[int]],
                  biases: Sequence[Optional[Tuple[np.ndarray, np.ndarray]]],
                  masks: Optional[Sequence[Optional[np.ndarray]]]):
    """What `ops.adjust_logits` needs to know of its rows, as one int32 array and where in it each part lies: slots and
    penalties, the lists of biases, which mask is whose (None where no row has any of it)."""
    rows = len(params)
    parts: List[np.ndarray] = []
    at = 0

    def put(array: np.ndarray) -> slice:
        nonlocal at
        parts.append(array.reshape(-1).view(np.int32))
        at += array.size
        return slice(at - array.size, at)
    histories = lists = mask_of = None
    if slots is not None:
        penalties = np.asarray([(p.repetition_penalty, p.presence_penalty, p.frequency_penalty) for p in params], dtype=np.float32)
        histories = put(np.asarray(slots, dtype=np.int32)), put(penalties)
    if any(bias is not None for bias in biases):
        start = np.zeros(rows + 1, dtype=np.int32)
        start[1:] = np.cumsum([0 if bias is None else len(bias[0]) for bias in biases])
        lists = put(start), put(np.concatenate([bias[0] for bias in biases if bias is not None])), \
            put(np.concatenate([bias[1] for bias in biases if bias is not None]))
    if masks is not None and any(mask is not None for mask in masks):
        has = np.asarray([mask is not None for mask in masks])
        mask_of = put(np.where(has, np.cumsum(has) - 1, -1).astype(np.int32))
    return np.concatenate(parts) if parts else None, histories, lists, mask_of


def _splitmix(x: int) -> int:
    x = (x + 0x9E3779B97F4A7C15) & _MASK
    x = ((x ^ (x >> 30)) * 0xBF58476D1CE4E5B9) & _MASK
    x = ((x ^ (x >> 27)) * 0x94D049BB133111EB) & _MASK
    return x ^ (x >> 31)


def uniform_draw(seed: int, index: int) -> float:
    """The uniform number in [0, 1) of output token `index` of a request with `seed`."""
    bits = _splitmix(_splitmix(seed & _MASK) ^ ((index + 1) * 0xD6E8FEB86659FD93 & _MASK))
    return float(np.float32((bits >> 40) / float(1 << 24)))   # 24 bits: exact in float32, < 1


def request_seed(engine_seed: int, request_id: int) -> int:
    return _splitmix((engine_seed & _MASK) ^ _splitmix(request_id + 0x51ED270B))


def any_short_list(params: Sequence[SamplingParams], longest: int) -> bool:
    """Whether some row draws from a top_k of at most `longest`, the rows that the sampler's first kernel is for."""
    return any(not p.greedy and 0 < p.top_k <= longest for p in params)


class Picked:
    """The tokens one sampling call chose: on the device at once (`device`, int32 [rows]), on
    the host after `result()`, which waits for the copy that was started with the call."""

    def __init__(self, device: torch.Tensor, host: np.ndarray, event, rows: int,
                 watches_fault: bool = False):
        self.device, self._host, self._event, self.rows = device, host, event, rows
        self._watches_fault = watches_fault
        self._list: Optional[List[int]] = None
        self.fault = 0          # after result(): the device's error flag as it stood after the kernels

    def result(self) -> List[int]:
        if self._list is None:
            self._event.synchronize()
            self._list = self._host[:self.rows].tolist()
            if self._watches_fault:
                self.fault = int(self._host[-1])
        return self._list


class Sampler:
    """Chooses one token per row of logits with the device kernels."""

    HOST_BUFFERS = 4           # pinned result buffers in rotation: a result is read at most two calls later

    def __init__(self, device):
        self.device = torch.device(device)
        self._scratch = None
        self._pinned: List[torch.Tensor] = []
        self._turn = 0
        from ..engine.context import PinnedRing
        self._ring = PinnedRing()    # staging of the sampling parameters
        self._mask_ring = PinnedRing(depth=4)
        self._no_error = None
        self.bytes_to_device = 0     # sampling parameters copied in (benchmarks read these)
        self.bytes_to_host = 0       # chosen ids copied out

    def sample(self, logits: torch.Tensor, params: Sequence[SamplingParams],
               seeds: Sequence[int], indices: Sequence[int]) -> List[int]:
        """logits float32 [rows, vocab]; row r is output token indices[r] of a request whose
        seed is seeds[r].  Returns the chosen ids (one device-to-host copy of rows ints)."""
        return self.sample_async(logits, params, seeds, indices).result()

    def _adjust(self, logits, params, error, slots, history, biases, masks):
        """Change the logits by what the rows' options say; returns the slots on the device, where there are any."""
        rows, vocab = logits.shape
        if history is None and any(p.penalised for p in params):
            raise ValueError("penalties need the history of every request's tokens")
        if masks is None and any(p.allowed is not None for p in params):
            raise ValueError("the masks of the allowed tokens are needed")
        if biases is None:
            biases = [sorted_bias(p.logit_bias, vocab) for p in params]
        if (slots is not None and len(slots) != rows) or len(biases) != rows or (masks is not None and len(masks) != rows):
            raise ValueError("a slot, a bias and a mask per row of logits are needed, each None or for all rows")
        if history is None or slots is None or max(slots) < 0:
            slots = None
        host, histories, lists, mask_of = stage_changes(params, slots, biases, masks)
        if host is None:
            return None
        staged = self._ring.stage(host, self.device)
        self.bytes_to_device += host.nbytes
        given = {}
        if histories is not None:
            given = dict(slots=staged[histories[0]], penalties=staged[histories[1]].view(torch.float32).view(rows, 3),
                         counts=history.counts, seen=history.seen)
        if lists is not None:
            given["bias"] = (staged[lists[0]], staged[lists[1]], staged[lists[2]].view(torch.float32))
        if mask_of is not None:
            if not all(mask is None or mask.any() for mask in masks):
                raise ValueError("no token is allowed in some row")
            bits = np.concatenate([mask for mask in masks if mask is not None])
            self.bytes_to_device += bits.nbytes
            given["masks"] = (staged[mask_of], self._mask_ring.stage(bits, self.device).view(-1, ops.bit_words(vocab)))
        ops.adjust_logits(logits, error, **given)
        return given.get("slots")

    def _host_buffer(self, rows: int) -> torch.Tensor:
        if not self._pinned or self._pinned[0].numel() - 1 < rows:
            size = max(256, 1 << (rows - 1).bit_length())
            # one more element: the device's error flag travels with the ids
            self._pinned = [torch.zeros(size + 1, dtype=torch.int32, pin_memory=True)
                            for _ in range(self.HOST_BUFFERS)]
        self._turn = (self._turn + 1) % self.HOST_BUFFERS
        return self._pinned[self._turn]

    def sample_async(self, logits: torch.Tensor, params: Sequence[SamplingParams],
                     seeds: Sequence[int], indices: Sequence[int],
                     error: Optional[torch.Tensor] = None, slots: Optional[Sequence[int]] = None,
                     history=None, biases: Optional[Sequence] = None,
                     masks: Optional[Sequence[Optional[np.ndarray]]] = None) -> Picked:
        """The same without waiting: the kernels and the copy to pinned host memory are queued,
        the chosen ids stay on the device for a step that feeds them back in.  `error` (int32
        [1], the flag that kernels set when they refuse an input or give up a wait) is copied
        along, so that whoever reads the ids learns of a fault without a transfer of its own.

        Rows whose options change logits have them changed in place.  For penalties `history` (a `TokenHistory`) and
        each row's slot in it (-1: none) are needed; the chosen tokens are taken into it.  biases: what `sorted_bias` makes
        of each row's options (None: made here); masks: the allowed tokens of each row as `pack_allowed` gives them, None
        where all are."""
        rows = logits.shape[0]
        if rows != len(params):
            raise ValueError("one SamplingParams per row of logits is needed")
        counted = None
        if slots is not None or masks is not None or any(p.penalised or p.logit_bias or p.allowed is not None for p in params):
            if error is None and self._no_error is None:
                self._no_error = torch.zeros(1, dtype=torch.int32, device=self.device)
            flag = self._no_error if error is None else error
            counted = self._adjust(logits, params, flag, slots, history, biases, masks)
        picks = torch.empty((2, rows), dtype=torch.int32, device=self.device)
        any_greedy = any(p.greedy for p in params)
        any_random = any(not p.greedy for p in params)
        if any_greedy:
            need = 2 * rows * ops.ARGMAX_PARTS
            if self._scratch is None or self._scratch.numel() < need:
                self._scratch = torch.empty(max(need, 4096), dtype=torch.float32,
                                            device=self.device)
            ops.argmax(logits, picks[0], self._scratch)
        if any_random:
            # one staged copy from pinned memory for all parameters: a copy from pageable memory
            # would wait for the stream and with it for the step that is still running
            host = np.empty((5, rows), dtype=np.float32)
            top_k = host[3].view(np.int32)
            for r, p in enumerate(params):
                host[0, r] = p.temperature if not p.greedy else 0.0
                host[1, r] = min(p.top_p, 1.0)
                host[2, r] = uniform_draw(seeds[r], indices[r])
                top_k[r] = max(0, int(p.top_k))
                host[4, r] = 1.0 if p.greedy else 0.0
            staged = self._ring.stage(host.reshape(-1).view(np.int32), self.device).view(5, rows)
            dev = staged.view(torch.float32)
            self.bytes_to_device += host.nbytes
            # the first of the sampler's two kernels would find no row to work on (2 to 3 us a step)
            ops.sample(logits, dev[0], staged[3], dev[1], dev[2], picks[1],
                       short_lists=any_short_list(params, ops.sample_short_top_k()))
            chosen = torch.where(dev[4] > 0, picks[0], picks[1]) if any_greedy else picks[1]
        else:
            chosen = picks[0]
        if counted is not None:
            ops.count_tokens(chosen, counted, history.counts, history.seen, flag)
        pinned = self._host_buffer(rows)
        pinned[:rows].copy_(chosen, non_blocking=True)
        if error is not None:
            pinned[-1:].copy_(error, non_blocking=True)
        event = torch.cuda.Event()
        event.record()
        self.bytes_to_host += 4 * rows + (4 if error is not None else 0)
        return Picked(chosen, pinned.numpy(), event, rows, error is not None)
