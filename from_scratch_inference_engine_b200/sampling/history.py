"""Which tokens each request's context holds, on the device: what the penalties for repeated tokens go by.

A history is a row of counts (how often the answer holds each token) and a row of bits (the token occurs at all, in the prompt
or in the answer).  A request's history is made when its first token is to be chosen, from its prompt and the answer so far,
follows every token chosen for it on the device (so that the next step need not wait for the host) and is given up when the
request is finished.  A request that is preempted keeps it; one that continues another (`Engine.fork`) gets one of its own.

Memory: 4 bytes and a bit per token of the vocabulary and slot (627 KB at 152,064 tokens), for as many slots as were in use
at once, rounded up to 8, 16, 32, ..; while it grows the old and the new lie side by side.
"""

from __future__ import annotations

from typing import Dict, List, Sequence, Tuple

import numpy as np
import torch

from ..kernels import ops


class TokenHistory:
    FIRST_SLOTS = 8            # doubled when more requests have one

    def __init__(self, device, vocab: int):
        self.device, self.vocab = torch.device(device), int(vocab)
        self.counts = self.seen = None
        self._slot_of: Dict[int, int] = {}
        self._free: List[int] = []
        from ..engine.context import PinnedRing
        self._ring = PinnedRing(depth=4)

    def __len__(self) -> int:
        return len(self._slot_of)

    def _grow(self, slots: int) -> None:
        old = 0 if self.counts is None else self.counts.shape[0]
        while len(self._free) < slots:
            size = max(self.FIRST_SLOTS, 2 * old)
            counts = torch.zeros((size, self.vocab), dtype=torch.int32, device=self.device)
            seen = torch.zeros((size, ops.bit_words(self.vocab)), dtype=torch.int32, device=self.device)
            if old:
                counts[:old].copy_(self.counts)
                seen[:old].copy_(self.seen)
            self.counts, self.seen = counts, seen
            self._free += range(size - 1, old - 1, -1)
            old = size

    def reserve(self, requests: Sequence[int]) -> None:
        """Take the memory that `slots` needs for these requests (ids), whatever of them it knows already."""
        self._grow(sum(request not in self._slot_of for request in requests))

    def slots(self, requests: Sequence[Tuple[int, Sequence[int], Sequence[int]]], error: torch.Tensor) -> List[int]:
        """The slots of `requests` (id, prompt, answer so far); those that have none get one, with both taken in."""
        fresh = [request for request in requests if request[0] not in self._slot_of]
        if fresh:
            if len({request[0] for request in fresh}) != len(fresh):
                raise ValueError("history: a request appears twice")
            self._grow(len(fresh))
            taken = self._free[-len(fresh):][::-1]
            for slot in taken:                            # (what the last owner left)
                self.counts[slot].zero_()
                self.seen[slot].zero_()
            for column, generated in ((1, False), (2, True)):
                lengths = [len(request[column]) for request in fresh]
                total = sum(lengths)
                if total:
                    host = np.empty((2, total), dtype=np.int32)
                    np.concatenate([np.asarray(request[column], dtype=np.int32) for request in fresh if request[column]], out=host[0])
                    host[1] = np.repeat(np.asarray(taken, dtype=np.int32), lengths)
                    staged = self._ring.stage(host.reshape(-1), self.device).view(2, total)
                    ops.count_tokens(staged[0], staged[1], self.counts, self.seen, error, generated=generated)
            del self._free[-len(fresh):]
            for (request, _, _), slot in zip(fresh, taken):
                self._slot_of[request] = slot
        return [self._slot_of[request[0]] for request in requests]

    def release(self, request: int) -> None:
        slot = self._slot_of.pop(request, None)
        if slot is not None:
            self._free.append(slot)
