"""Keys that several running requests hold, read once for all of them, through the runner and the engine."""

import numpy as np
import pytest
import torch

import helpers
from helpers import TINY

pytestmark = pytest.mark.gpu

# As for every other way of cutting the work (test_gpu_replay.py): 32-bit sums in another order, and results stored in
# bfloat16 after every operation, relative to max(1, the largest |logit|).  The shared form rounds where the other forms of
# the attention do: weights against a running maximum, and the result.
FLOAT32_BOUND = 1e-4
BFLOAT16_BOUND = {"A": 6.4e-3, "C": 3.0e-2, "E": 3.9e-2, "F": 2.2e-2}


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    root = tmp_path_factory.mktemp("models")
    return {name: helpers.make_model_dir(root, name) for name in ("A", "C", "E", "F")}


def runner_of(folder, dtype, page_size, pages=400, max_requests=32, graphs=True, shared=True):
    from from_scratch_inference_engine_b200.engine import LoadedModel, ModelRunner
    model = LoadedModel.from_pretrained(folder, dtype=dtype, max_positions=512)
    runner = ModelRunner(model.model, model.runtime, page_size=page_size, num_pages=pages, max_requests=max_requests,
                         cuda_graphs=graphs, shared_attention=shared)
    runner.shared_min_bytes = runner.shared_min_part = runner.shared_least_keys = 0
    return runner


@pytest.fixture
def calls(monkeypatch):
    """How often attention over shared pages was launched or captured, and with how many runs."""
    from from_scratch_inference_engine_b200.kernels import ops
    seen = []
    real = ops.shared_attention

    def counting(*args, **kwargs):
        seen.append(args[9].shape[0])
        return real(*args, **kwargs)
    monkeypatch.setattr(ops, "shared_attention", counting)
    return seen


def step(runner, *pairs):
    from from_scratch_inference_engine_b200 import StepEntry
    logits = runner.step([StepEntry(handle, ids, [len(ids) - 1]) for handle, ids in pairs]).cpu().numpy()
    runner.raise_on_device_error()
    return logits


def check(name, folder, dtype, seqs, rows):
    bound = FLOAT32_BOUND if dtype == "float32" else BFLOAT16_BOUND[name]
    for seq, row in zip(seqs, rows):
        want = helpers.plain_logits(folder, seq)[-1]
        assert np.abs(row - want).max() < bound * max(1.0, np.abs(want).max())


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("name,page_size", [("A", 4), ("C", 16), ("E", 16), ("F", 32)])
def test_forks_of_forks(folders, calls, name, page_size, graphs, dtype):
    """A tree of requests, steps of single tokens beside requests that share nothing and beside prompts, requests that end."""
    folder, vocab = folders[name], TINY[name]["config"]["vocab_size"]
    runner = runner_of(folder, dtype, page_size, graphs=graphs)
    ids = helpers.random_ids(vocab, 2 * page_size + 3, 1)
    parent, other = runner.cache.open("parent"), runner.cache.open("other")
    apart = helpers.random_ids(vocab, 9, 2)
    check(name, folder, dtype, [ids, apart], step(runner, (parent, ids), (other, apart)))
    handles, seqs = [other, parent], [list(apart), list(ids)]

    def turn(count, seed):
        fresh = [helpers.random_ids(vocab, count, 1000 * seed + i) for i in range(len(handles))]
        rows = step(runner, *zip(handles, fresh))
        for seq, more in zip(seqs, fresh):
            seq += more
        check(name, folder, dtype, seqs, rows)
    handles += runner.fork(parent, ["b", "c", "d"])
    seqs += [list(ids) for _ in range(3)]
    for seed in range(3):
        turn(1, seed + 1)
    assert calls
    turn(page_size, 4)                                         # everyone in a portion: no single tokens
    grown = seqs[2]
    handles += runner.fork(handles[2], ["e", "f"])             # a second level
    seqs += [list(grown) for _ in range(2)]
    turn(1, 5)
    late = helpers.random_ids(vocab, 2 * page_size + 1, 3)      # a prompt beside single tokens
    fresh = [helpers.random_ids(vocab, 1, 60 + i) for i in range(len(handles))]
    handles.append(runner.cache.open("late"))
    seqs.append([])
    fresh.append(late)
    before = len(calls)
    rows = step(runner, *zip(handles, fresh))
    assert len(calls) > before
    for seq, more in zip(seqs, fresh):
        seq += more
    check(name, folder, dtype, seqs, rows)
    runner.cache.close(handles.pop(1))                         # the first one ends: others hold its pages
    seqs.pop(1)
    runner.compact()
    for seed in range(2):
        turn(1, seed + 6)
    for handle in handles:
        runner.cache.close(handle)
    assert all(pool.num_free == pool.num_pages for pool in runner.cache.pools)


@pytest.mark.parametrize("graphs", [True, False])
def test_a_step_shares_only_where_it_pays(folders, calls, graphs):
    runner = runner_of(folders["E"], "bfloat16", 16, graphs=graphs)
    vocab = TINY["E"]["config"]["vocab_size"]
    parent = runner.cache.open("parent")
    step(runner, (parent, helpers.random_ids(vocab, 70, 4)))
    handles = [parent] + runner.fork(parent, ["b", "c"])
    # 64 keys of 2 heads of 64, keys and values of 2 bytes, for two requests: 65,536 bytes; of 213, 216 and 219 keys in all
    for least, part, shares in ((65537, 0.0, False), (65536, 0.62, False), (65536, 0.58, True)):
        calls.clear()
        runner.shared_min_bytes, runner.shared_min_part = least, part
        step(runner, *[(handle, [5]) for handle in handles])
        assert bool(calls) == shares
        for handle in handles[1:]:
            runner.cache.close(handle)
        handles = [parent] + runner.fork(parent, ["b", "c"])
    calls.clear()
    step(runner, (handles[0], [7]))                             # one alone
    assert not calls


def test_without_the_option_nothing_is_shared(folders, calls):
    runner = runner_of(folders["E"], "bfloat16", 16, shared=False)
    parent = runner.cache.open("parent")
    step(runner, (parent, [3] * 40))
    step(runner, *[(handle, [5]) for handle in [parent] + runner.fork(parent, ["b", "c"])])
    assert not calls and len(runner._graphs) == 1


def test_a_model_whose_layers_cannot_is_refused(folders, tmp_path):
    import json
    from from_scratch_inference_engine_b200 import Engine, LoadedModel, write_random_model
    from from_scratch_inference_engine_b200.config import config_from_dict
    config = dict(TINY["C"]["config"], max_window_layers=0)      # every layer keeps a window of the keys
    folder = write_random_model(tmp_path / "windows", config_from_dict(config), 1, 0.05)
    model = LoadedModel.from_pretrained(folder, max_positions=256)
    assert Engine(model, block_size=4, num_blocks=64, max_batch=2).runner.shareable == [False]
    with pytest.raises(ValueError, match="shared_attention"):
        Engine(model, block_size=4, num_blocks=64, max_batch=2, shared_attention=True)


def test_graphs_are_captured_ahead_for_both_forms(folders, calls):
    from from_scratch_inference_engine_b200 import Engine, LoadedModel, SamplingParams
    model = LoadedModel.from_pretrained(folders["F"], max_positions=1024)
    engine = Engine(model, num_blocks=64, max_batch=4, shared_attention=True)
    engine.runner.shared_min_bytes = engine.runner.shared_min_part = engine.runner.shared_least_keys = 0
    assert engine.warm_up(100) == 5                             # one request alone; two and four, either way
    calls.clear()
    ids = engine.add_samples(helpers.random_ids(300, 50, 1), [SamplingParams(seed=i) for i in range(4)], 6)
    engine.run_until_done()
    assert not calls and all(len(engine.output(i)) == 6 for i in ids)


@pytest.mark.parametrize("pipeline", [True, False])
@pytest.mark.parametrize("blocks", [200, 24])
def test_answers_are_those_of_requests_alone(folders, blocks, pipeline, calls):
    """Answers to two prompts with a common beginning; with 24 blocks some wait or are run again."""
    from from_scratch_inference_engine_b200 import Engine, LoadedModel, SamplingParams
    model = LoadedModel.from_pretrained(folders["A"], dtype="float32", max_positions=512)
    engine = Engine(model, block_size=4, num_blocks=blocks, max_batch=8, max_step_tokens=16, pipeline=pipeline,
                    enable_prefix_cache=True, shared_attention=True)
    engine.runner.shared_min_bytes = engine.runner.shared_min_part = engine.runner.shared_least_keys = 0
    common = helpers.random_ids(256, 21, 1)
    prompts = [common + helpers.random_ids(256, n, 2 + n) for n in (5, 11)]
    params = [SamplingParams(temperature=0.8, seed=40 + i) for i in range(6)]
    ids = engine.add_samples(prompts[0], params[:4], 9) + engine.add_samples(prompts[1], params[4:], 9)
    engine.run_until_done()
    engine.runner.raise_on_device_error()
    engine.runner.cache.check()
    assert calls
    alone = Engine(model, block_size=4, num_blocks=200, max_batch=8, max_step_tokens=16)
    for index, (rid, own) in enumerate(zip(ids, params)):
        assert engine.output(rid) == alone.generate(prompts[index >= 4], own, 9)


def test_working_memory_is_taken_before_serving(folders, calls):
    """A runner that has reserved its memory has that of steps outside of graphs, whose requests share and prompts run beside."""
    runner = runner_of(folders["E"], "bfloat16", 16, graphs=False)
    runner.reserve_step_memory(100)
    room = runner.runtime._buffers["attention.shared_room", torch.uint8]
    parent = runner.cache.open("parent")
    step(runner, (parent, [3] * 70))
    handles = [parent] + runner.fork(parent, list("bcdefg"))
    step(runner, *[(handle, [5]) for handle in handles], (runner.cache.open("other"), [1, 2, 3]))
    assert calls and runner.runtime._buffers["attention.shared_room", torch.uint8] is room


@pytest.mark.parametrize("requests", [7, 40, 200])
def test_captured_steps_find_the_working_memory_that_was_taken(folders, calls, requests):
    """Graphs of padded batches (8, 48, 256), captured ahead or while serving: none is given more than was reserved, and what a
    step of as many requests as there may be needs is what was reserved."""
    from from_scratch_inference_engine_b200.engine import runner as module
    runner = runner_of(folders["E"], "bfloat16", 16, pages=500, max_requests=requests)
    runner.reserve_step_memory(300)
    room = runner.runtime._buffers["attention.shared_room", torch.uint8]
    runner.capture_decode_graphs(100)
    assert calls and runner.runtime._buffers["attention.shared_room", torch.uint8] is room
    graphs = {batch: graph for (batch, _, shared), graph in runner._graphs.items() if shared}
    largest = max(graphs)
    assert largest >= requests
    for batch, graph in graphs.items():
        lists = graph.context.shared_lists[runner.shareable.index(True)]
        assert lists.shared == min(batch - 1, module.MOST_SHARED_RUNS) and lists.runs.shape[0] == batch + lists.shared
    parent = runner.cache.open("parent")
    step(runner, (parent, [3] * 70))
    handles = [parent] + runner.fork(parent, list(range(requests - 1)))
    step(runner, *[(handle, [5]) for handle in handles])
    assert len(runner._graphs) == 2 * len(graphs) + 1
    assert runner.runtime._buffers["attention.shared_room", torch.uint8] is room


def test_behind_the_attention_that_lets_its_successor_go_early(folders, monkeypatch):
    """Requests of two tokens on `attention_tc_decode` in front of those of one that share keys, step after step."""
    from from_scratch_inference_engine_b200.kernels import ops
    runner = runner_of(folders["F"], "bfloat16", 16)
    runner.runtime.decode_tcgen05_min_blocks = 1
    order = []
    for name in ("attention_tc_decode", "shared_attention"):
        monkeypatch.setattr(ops, name, lambda *args, real=getattr(ops, name), name=name, **kwargs: (order.append(name), real(*args, **kwargs))[1])
    prompt = helpers.random_ids(300, 100, 1)
    parent = runner.cache.open("parent")
    step(runner, (parent, prompt))
    handles = [parent] + runner.fork(parent, list("bcdefg"))
    seqs = [list(prompt) for _ in handles]
    apart = [runner.cache.open(f"apart {i}") for i in range(9)]
    handles += apart
    seqs += [[] for _ in apart]
    for turn in range(6):
        order.clear()
        fresh = [helpers.random_ids(300, 1 if i < 7 else 2, 100 * turn + i) for i in range(len(handles))]
        rows = step(runner, *zip(handles, fresh))
        assert order == ["attention_tc_decode", "shared_attention"] * 2
        for seq, more in zip(seqs, fresh):
            seq += more
        check("F", folders["F"], "bfloat16", seqs, rows)
