"""Runs of shared keys in a step's context, and tiles without requests of one token (no GPU needed)."""
import types

import numpy as np
import torch

from from_scratch_inference_engine_b200.engine.context import StepContext


class Ring:
    def stage(self, host, device, out=None):
        return torch.from_numpy(host.copy())


def test_lists_of_shared_runs():
    """One copy brings them along; for a captured step they are padded: places that see no key, runs without places."""
    from from_scratch_inference_engine_b200.cache.shared_runs import SharedRuns
    runs = SharedRuns(np.array([1, 0], np.int32), np.array([[0, 2, 0, 8, 0, -1], [0, 1, 8, 10, 1, 0], [1, 1, 8, 12, 0, 0]], np.int32),
                      np.array([1, 2], np.int32), 1, 1, 8)
    tables = [(4, [[0, 1, 2], [0, 1, 3], []]), (8, [[4, 5], [4, 6], []])]
    for room, order, own, count in (((0, 0), [1, 0], [1, 2], 3), ((5, 4), [1, 0, 2], [1, 2, -1], 5)):
        ctx = StepContext(types.SimpleNamespace(device="cpu"), Ring(), {}, None, [7, 7, 0], [0, 1, 2], [1, 1, 1], [11, 9, 0],
                          [0, 1, -1], tables, shared=[runs, None], shared_room=room)
        lists = ctx.shared_lists[0]
        assert ctx.shared_lists[1] is None
        assert lists.order.tolist() == order and lists.own_run.tolist() == own
        assert lists.runs.tolist() == runs.runs.tolist() + [[0] * 6] * (count - 3)
        assert (lists.shared, lists.levels) == ((1, 1) if room == (0, 0) else room)
        assert ctx.groups[0].slot_of.tolist() == [11, 13, -1]


def test_how_many_runs_of_a_captured_step_may_be_shared():
    """Working memory goes by it: of the runs that a list is padded to most are requests' own."""
    from from_scratch_inference_engine_b200.cache.shared_runs import SharedRuns
    runs = SharedRuns(np.array([0, 1], np.int32), np.array([[0, 2, 0, 8, 0, -1], [0, 1, 8, 10, 0, 0], [1, 1, 8, 12, 1, 0]], np.int32),
                      np.array([1, 2], np.int32), 1, 1, 8)
    for most in (1, 3):
        ctx = StepContext(types.SimpleNamespace(device="cpu"), Ring(), {}, None, [7] * 4, [0, 1, 2, 3], [1] * 4, [9, 11, 0, 0],
                          [0, 1, -1, -1], [(4, [[0, 1, 2], [0, 1, 3], [], []])], shared=[runs], shared_room=(7, 4), most_shared=most)
        lists = ctx.shared_lists[0]
        assert (lists.shared, lists.levels, lists.runs.shape[0], lists.order.shape[0]) == (most, 4, 7, 4)


def test_requests_of_one_token_can_be_left_out_of_the_tiles():
    ctx = StepContext(types.SimpleNamespace(device="cpu"), Ring(), {}, None, [0] * 24, [0, 1, 21, 22], [1, 20, 1, 2], [3, 0, 8, 5],
                      [0, 1, 2, 3], [(4, [list(range(8)) for _ in range(4)])])
    assert ctx.attention_tiles(2, 16).item.tolist() == [0, 1, 1, 1, 2, 3]
    assert ctx.attention_tiles(2, 16, True).item.tolist() == [1, 1, 1, 3]
    classes = ctx.attention_row_classes(2, (16, 32), True)
    assert [c[0] for c in classes] == [0, 1]
    assert classes[0][1].item.tolist() == [3] and classes[0][2].tolist() == [22, 23]
    assert classes[1][1].item.tolist() == [1, 1] and classes[1][2].tolist() == list(range(1, 21))
    assert len(ctx.attention_row_classes(2, (16, 32))[0][2]) == 4
