"""Forked requests and compaction in the cache manager: pages, reference counts, tables and what is to be copied (host only)."""
import random

import pytest

from from_scratch_inference_engine_b200.cache.manager import CacheManager, CacheNeed
from from_scratch_inference_engine_b200.cache.pool import OutOfPages, PagePool


def manager(pages=20, slots=6, page=4, window=0, prefix=False):
    needs = [CacheNeed(1, 8), CacheNeed(1, 8, window, 2)] if window else [CacheNeed(1, 8)]
    return CacheManager(needs, page, pages, slots, enable_prefix_cache=prefix)


def grow(cache, handle, tokens):
    cache.reserve(handle, tokens)
    cache.commit(handle, tokens)


class Memory:
    """What the pages hold: every written token's owner-independent history, so that a wrong page shows."""

    def __init__(self, cache):
        self.cache, self.pages = cache, [{} for _ in cache.groups]

    def write(self, handle, tokens):
        start = handle.length
        self.cache.reserve(handle, len(tokens))
        for i, token in enumerate(tokens):
            block, place = divmod(start + i, self.cache.page_size)
            for g, table in enumerate(handle.tables):
                self.pages[g].setdefault(table[block], {})[place] = token
        self.cache.commit(handle, len(tokens))

    def copy(self, moves):
        for held, pairs in zip(self.pages, moves):
            old = {src: dict(held.get(src, {})) for src, _ in pairs}
            for src, dst in pairs:
                held[dst] = dict(old[src])

    def read(self, handle, g=0):
        out = []
        for at in range(handle.length):
            block, place = divmod(at, self.cache.page_size)
            page = handle.tables[g][block]
            out.append(None if page < 0 else self.pages[g][page][place])
        return out


@pytest.mark.parametrize("length", [0, 1, 3, 4, 5, 8, 11])
@pytest.mark.parametrize("window", [0, 5])
def test_forked_requests_hold_the_same_tokens_and_go_apart(length, window):
    cache = manager(window=window)
    memory = Memory(cache)
    parent = cache.open("parent")
    if length:
        memory.write(parent, list(range(length)))
    before = memory.read(parent)
    children, moves = cache.fork(parent, ["a", "b"])
    memory.copy(moves)
    cache.check()
    for g in range(len(cache.groups)):
        assert len(moves[g]) == (2 if length % 4 else 0)
        assert [memory.read(c, g) for c in children] == [memory.read(parent, g)] * 2
    for at, handle in enumerate([parent] + children):
        memory.write(handle, [100 * (at + 1) + i for i in range(6)])
    for at, handle in enumerate([parent] + children):
        kept = memory.read(handle)
        assert kept == before + [100 * (at + 1) + i for i in range(6)]
    cache.check()
    assert len({h.slot for h in [parent] + children}) == 3
    for handle in [parent] + children:
        cache.close(handle)
    cache.check()
    assert cache.free_pages() == [20] * len(cache.groups) and cache.slots.num_free == 6


def test_a_fork_that_finds_no_room_changes_nothing():
    cache = manager(pages=4, slots=3)
    parent = cache.open("parent")
    grow(cache, parent, 10)
    for ids in (["a", "b"], ["a", "b", "c"]):                 # one page is free; two slots are
        before = (cache.free_pages(), cache.slots.num_free, [list(t) for t in parent.tables])
        with pytest.raises(OutOfPages):
            cache.fork(parent, ids)
        assert before == (cache.free_pages(), cache.slots.num_free, [list(t) for t in parent.tables])
        cache.check()
    with pytest.raises(RuntimeError):
        cache.fork(parent, ["parent"])
    with pytest.raises(RuntimeError):
        cache.fork(parent, ["a", "a"])
    (child,), _ = cache.fork(parent, ["a"])
    cache.close(parent)
    with pytest.raises(RuntimeError):
        cache.fork(parent, ["b"])
    cache.check()
    assert cache.free_pages() == [1] and child.length == 10
    assert cache.fork(child, []) == ([], [[]])


def test_forks_share_cached_prefixes():
    cache = manager(pages=12, prefix=True)
    parent = cache.open("parent")
    grow(cache, parent, 9)
    cache.register_prefix(parent, list(range(9)))
    children, _ = cache.fork(parent, ["a"])
    cache.close(parent)
    cache.check()
    cache.close(children[0])
    cache.check()
    again = cache.open("again")
    assert cache.acquire_prefix(again, list(range(9))) == 8
    cache.check()


def test_compaction_of_a_pool():
    pool = PagePool(6)
    pages = [pool.allocate() for _ in range(6)]
    for page in (0, 2, 3):
        pool.free(page)
    pool.incref(4)
    assert pool.compact() == {4: 0, 5: 2}
    assert pool.compact() == {}
    pool.check()
    assert [pool.ref_count(p) for p in range(6)] == [2, 1, 1, 0, 0, 0] and pool.allocate() == 3
    assert pages == list(range(6)) and PagePool(3).compact() == {} and PagePool(0).compact() == {}


@pytest.mark.parametrize("seed", range(6))
def test_requests_forks_and_compactions_at_random(seed):
    rng = random.Random(seed)
    cache = manager(pages=40, slots=8, page=4, window=6 if seed % 2 else 0, prefix=seed % 2 == 0)
    memory, live, name = Memory(cache), {}, 0
    for _ in range(300):
        action = rng.random()
        if action < 0.25 and cache.can_open():
            name += 1
            live[name] = (cache.open(name), [])
        elif action < 0.6 and live:
            handle, tokens = live[rng.choice(list(live))]
            new = [rng.randrange(1000) for _ in range(rng.randint(1, 7))]
            if cache.can_reserve(handle, len(new)):
                memory.write(handle, new)
                tokens += new
                if rng.random() < 0.3:
                    cache.register_prefix(handle, tokens)
        elif action < 0.75 and live:
            handle, tokens = live[rng.choice(list(live))]
            try:
                children, moves = cache.fork(handle, [name + 1 + i for i in range(rng.randint(1, 3))])
            except OutOfPages:
                continue
            memory.copy(moves)
            for child in children:
                name += 1
                live[name] = (child, list(tokens))
        elif action < 0.9 and live:
            cache.close(live.pop(rng.choice(list(live)))[0])
        else:
            moves = cache.compact()
            for pairs in moves:
                assert not {s for s, _ in pairs} & {d for _, d in pairs}
            memory.copy(moves)
            for pool in cache.pools:
                used = pool.num_pages - pool.num_free
                assert all((pool.ref_count(p) > 0) == (p < used) for p in range(pool.num_pages))
        cache.check()
        for handle, tokens in live.values():
            assert memory.read(handle) == tokens               # the group that keeps everything
            for g, group in enumerate(cache.groups):
                if group.need.window:
                    seen = memory.read(handle, g)
                    assert all(got == want for got, want in zip(seen, tokens) if got is not None)
                    assert seen[-group.need.window + 1:] == tokens[-group.need.window + 1:] or len(tokens) < group.need.window
                array = handle.table_array(g)
                assert array.tolist() == handle.tables[g]
