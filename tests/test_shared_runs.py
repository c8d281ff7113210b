"""The runs of pages that requests share, found from their block tables."""
import random

import numpy as np
import pytest

from from_scratch_inference_engine_b200.cache.manager import CacheManager, CacheNeed
from from_scratch_inference_engine_b200.cache.shared_runs import find_shared_runs


def runs_of(tables, page, lengths, new=None, least=1, *most):
    width = max([len(t) for t in tables] + [1])
    array = np.full((len(tables), width), -1, dtype=np.int32)
    for i, t in enumerate(tables):
        array[i, :len(t)] = t
    new = new or [1] * len(tables)
    start = np.cumsum([0] + new[:-1]) if tables else []
    return find_shared_runs(array, page, np.asarray(start, dtype=np.int32), np.asarray(new, dtype=np.int32),
                            np.asarray([n - k for n, k in zip(lengths, new)], dtype=np.int32), least, *most)


def check(found, tables, page, lengths, new):
    """Every token's chain of runs holds its keys once, in pages that its request holds, and every run's places are together."""
    tokens = [(i, t) for i, n in enumerate(new) for t in range(n)]
    assert sorted(found.order.tolist()) == list(range(len(tokens)))
    for place, token in enumerate(found.order.tolist()):
        item, t = tokens[token]
        position = lengths[item] - new[item] + t
        run, chain, depth = int(found.own_run[place]), [], -1
        assert run >= found.shared
        while run >= 0:
            first, count, begin, end, row, parent = found.runs[run].tolist()
            assert first <= place < first + count and parent < run
            if run < found.shared:
                assert end <= lengths[item] - new[item] and begin % page == end % page == 0 and count > 1
            else:
                assert end == lengths[item] and row == item and count == new[item]
            chain.append((begin, end))
            for key in range(begin, min(end, position + 1)):
                assert tables[row][key // page] == tables[item][key // page] >= 0
            run, depth = parent, depth + 1
        assert depth <= found.levels
        chain.reverse()
        assert chain[0][0] == 0 and all(a[1] == b[0] for a, b in zip(chain, chain[1:]))


def test_nothing_shared():
    tables, lengths = [[0, 1], [2], [3, 4, 5]], [20, 3, 40]
    found = runs_of(tables, 16, lengths)
    assert found.shared == found.levels == found.saved == 0 and len(found.runs) == 3
    check(found, tables, 16, lengths, [1, 1, 1])
    assert len(runs_of([], 16, []).runs) == 0 and len(runs_of([[7]], 16, [1]).runs) == 1


def test_one_prompt():
    tables = [[5, 6, 7, 1], [5, 6, 7, 2], [5, 6, 7, 3, 4]]
    found = runs_of(tables, 4, [14, 13, 18])
    assert found.runs[0].tolist() == [0, 3, 0, 12, 0, -1] and found.shared == 1 and found.saved == 24
    check(found, tables, 4, [14, 13, 18], [1, 1, 1])


def test_only_full_pages_in_front_of_the_new_tokens():
    # the third page is the same, but request 1 is about to write its last slot and request 2 the one behind it
    tables = [[5, 6, 7], [5, 6, 7, 8]]
    found = runs_of(tables, 4, [12, 13])
    assert found.runs[0].tolist() == [0, 2, 0, 8, 0, -1]
    check(found, tables, 4, [12, 13], [1, 1])
    assert runs_of([[5], [5]], 4, [4, 4]).shared == 0
    assert runs_of([[-1, 5, 1], [-1, 5, 2]], 4, [10, 10]).shared == 0          # given back


def test_little_is_left_as_it_is():
    tables = [[1, 2], [1, 3], [1, 4]]
    assert runs_of(tables, 4, [6, 6, 6], least=8).shared == 1 and runs_of(tables, 4, [6, 6, 6], least=9).shared == 0


def test_a_little_common_start_goes_into_the_runs_behind_it():
    tables = [[1, 2, 3, 4, 10], [1, 5, 6, 7, 12], [1, 2, 3, 4, 11], [1, 5, 6, 7, 13]]
    for least, want in ((12, [[0, 4, 0, 4], [0, 2, 4, 16], [2, 2, 4, 16]]), (13, [[0, 2, 0, 16], [2, 2, 0, 16]]), (17, [])):
        found = runs_of(tables, 4, [18] * 4, least=least)
        assert [r[:4] for r in found.runs[:found.shared].tolist()] == want
        check(found, tables, 4, [18] * 4, [1] * 4)


@pytest.mark.parametrize("seed", range(60))
def test_random_trees(seed):
    rng = random.Random(seed)
    page, count = rng.choice([1, 4, 16]), rng.randint(1, 20)
    paths, fresh = [[]], iter(range(10 ** 6))
    for _ in range(rng.randint(0, 6)):                      # prefixes of prefixes
        paths.append(rng.choice(paths) + [next(fresh) for _ in range(rng.randint(1, 5))])
    tables, lengths, new = [], [], []
    for _ in range(count):
        path = list(rng.choice(paths))
        n = rng.choice([1, 1, 1, 2, 5])
        # tokens of its own, some of them in front of this step's
        own = n + rng.randint(0, 3 * page)
        length = len(path) * page + own
        tables.append(path + [next(fresh) for _ in range(-(-length // page) - len(path))])
        lengths.append(length)
        new.append(n)
    found = runs_of(tables, page, lengths, new, rng.choice([1, 1, page * 3]))
    check(found, tables, page, lengths, new)
    if found.shared:
        spared = sum((r[1] > 0) * (r[3] - r[2]) for r in found.runs[:found.shared].tolist())
        assert found.saved >= spared


def test_forked_requests_of_the_cache_manager():
    cache = CacheManager([CacheNeed(2, 16)], 4, 64, 16)
    root = cache.open("root")
    cache.reserve(root, 10)
    cache.commit(root, 10)
    children, _ = cache.fork(root, ["a", "b"])
    (grandchild,), _ = (cache.reserve(children[0], 7), cache.commit(children[0], 7), cache.fork(children[0], ["c"]))[2]
    handles = [root, *children, grandchild]
    for h in handles:
        cache.reserve(h, 1)
    tables, lengths = [h.tables[0] for h in handles], [h.length + 1 for h in handles]
    found = runs_of(tables, 4, lengths)
    check(found, tables, 4, lengths, [1] * 4)
    assert found.shared == 2 and found.levels == 2 and found.saved == 3 * 8 + 8


@pytest.mark.parametrize("most,levels", [(0, 31), (1, 31), (5, 31), (700, 3), (1000, 31), (1000, 1), (1000, 0)])
def test_no_more_runs_and_levels_than_asked_for(most, levels):
    """Request i holds the first i pages of one chain: without a limit a run around a run around a run.."""
    count, page = 300, 4
    tables = [list(range(i)) + [1000 + i] for i in range(count)]
    lengths = [i * page + 1 for i in range(count)]
    found = runs_of(tables, page, lengths, None, 1, most, levels)
    check(found, tables, page, lengths, [1] * count)
    assert found.shared == min(most, levels, count - 2) and found.levels == found.shared
