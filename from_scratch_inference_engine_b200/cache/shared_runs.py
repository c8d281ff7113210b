"""Which keys the requests of a step share: their block tables cut into runs of pages.

Requests hold the same leading pages after `CacheManager.fork` and after `acquire_prefix`.  Seen as paths from the first page
on, their tables make a tree; a stretch of pages that several requests pass through is a run that attention reads once for
all of them, what is left of a request's table is a run of its own (see `ops.shared_attention`)."""

from __future__ import annotations

from dataclasses import dataclass
from typing import List, Tuple

import numpy as np


@dataclass(frozen=True)
class SharedRuns:
    """order [n] (tokens), runs [r, 6] and own_run [n] as `ops.shared_attention` takes them, int32; the shared runs come first.
    `shared`: how many those are; `levels`: at most so many lie around a token's own; `saved`: keys that need not be read
    again, over all requests."""

    order: np.ndarray
    runs: np.ndarray
    own_run: np.ndarray
    shared: int
    levels: int
    saved: int


def find_shared_runs(tables: np.ndarray, page_size: int, q_start: np.ndarray, q_len: np.ndarray, pos0: np.ndarray,
                     least_saved: int = 64, most_shared: int = 1 << 30, most_levels: int = 31) -> SharedRuns:
    """tables int32 [requests, width] (page ids, below 0 where there is none), and per request where its tokens start in the
    step, how many they are and the position of the first.  Only full pages in front of that position count as shared, only
    where sharing them saves reading `least_saved` keys, in at most `most_shared` runs and `most_levels` around a token."""
    full = np.asarray(pos0, dtype=np.int64) // page_size
    shared: List[Tuple[int, int, int, int, int, int]] = []       # runs, places counted in requests
    items: List[np.ndarray] = []
    begins: List[np.ndarray] = []
    parents: List[np.ndarray] = []
    placed = levels = saved = 0
    everyone = np.arange(len(q_len))
    # Still to do, the next one last: requests that hold the same pages in front of `column` (those from `begin` on are in no
    # run yet), the run around them and how many lie around each other there.  column -1: they are done and take their places.
    todo: List[Tuple[np.ndarray, int, int, int, int]] = []
    if len(everyone):
        todo.append((everyone, 0 if len(everyone) > 1 else -1, 0, -1, 0))
    while todo:
        members, column, begin, parent, depth = todo.pop()
        if column < 0:
            items.append(members)
            begins.append(np.full(len(members), begin * page_size, dtype=np.int64))
            parents.append(np.full(len(members), parent, dtype=np.int64))
            placed += len(members)
            continue
        upto = int(full[members].min())
        if upto > column:
            pages = tables[members, column:upto]
            same = (pages == pages[0]).all(axis=0) & (pages[0] >= 0)
            column = upto if same.all() else column + int(np.argmin(same))
        keys = (column - begin) * page_size
        if keys * (len(members) - 1) >= max(least_saved, 1) and len(shared) < most_shared and depth < most_levels:
            shared.append((placed, len(members), begin * page_size, column * page_size, int(members[0]), parent))
            begin, parent, depth = column, len(shared) - 1, depth + 1
            levels = max(levels, depth)
            saved += keys * (len(members) - 1)
        # those that go on with the same page stay together
        parts = []
        going = members[full[members] > column]
        if len(going) > 1:
            page = tables[going, column]
            going = going[page >= 0]
            values, which, counts = np.unique(tables[going, column], return_inverse=True, return_counts=True)
            together = np.nonzero(counts > 1)[0]
            if len(together):
                parts = [going[which == value] for value in together]
                members = np.setdiff1d(members, going[counts[which] > 1], assume_unique=True)
        if len(members):
            todo.append((members, -1, begin, parent, depth))
        todo += [(part, column, begin, parent, depth) for part in reversed(parts)]
    q_start, q_len = np.asarray(q_start, dtype=np.int64), np.asarray(q_len, dtype=np.int64)
    member = np.concatenate(items) if items else everyone
    lengths = q_len[member]
    first = np.cumsum(lengths) - lengths                           # place of each request's first token
    runs = np.empty((len(shared) + len(member), 6), dtype=np.int32)
    for index, (place, count, begin, end, item, parent) in enumerate(shared):
        start = first[place]
        runs[index] = (start, first[place + count - 1] + lengths[place + count - 1] - start, begin, end, item, parent)
    if len(member):
        runs[len(shared):] = np.stack([first, lengths, np.concatenate(begins), np.asarray(pos0, dtype=np.int64)[member] + lengths,
                                       member, np.concatenate(parents)], axis=1)
    total = int(lengths.sum())
    order = np.repeat(q_start[member] - first, lengths) + np.arange(total)
    own_run = np.repeat(np.arange(len(member)) + len(shared), lengths)
    return SharedRuns(order.astype(np.int32), runs, own_run.astype(np.int32), len(shared), levels, saved)
