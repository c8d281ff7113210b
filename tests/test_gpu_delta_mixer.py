"""The gated delta rule as a mixer beside attention, and requests that are continued several times: the example's architecture
against a plain implementation in 64 bits, under every cutting of the work, through forks and compaction."""
import json
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

import helpers
import plain_delta
import plain_qwen2 as plain

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))
import delta_samples as example  # noqa: E402

pytestmark = pytest.mark.gpu
VOCAB = 97


def plain_logits(folder, ids):
    """Logits of every position."""
    cfg = example.DeltaHybridConfig.from_dict(json.loads((folder / "config.json").read_text()))
    w = plain.read_safetensors(folder / "model.safetensors")
    x = plain.embedding(w["embed.weight"], ids)
    n, h, qk = len(ids), cfg.heads, cfg.qk_heads
    for i in range(cfg.layers):
        p = f"layers.{i}.mixer."
        y = plain.rms_norm(x, w[f"layers.{i}.mixer_norm.weight"], cfg.eps)
        if cfg.attends(i):
            positions = list(range(n))
            q = plain.rope(plain.linear(y, w[p + "q_proj.weight"]), h, cfg.dim, cfg.theta, positions)
            k = plain.rope(plain.linear(y, w[p + "k_proj.weight"]), qk, cfg.dim, cfg.theta, positions)
            v = plain.linear(y, w[p + "v_proj.weight"])
            x = x + plain.linear(plain.attention(q, k, v, h, qk, cfg.dim), w[p + "o_proj.weight"])
        else:
            stacked = torch.cat([plain.linear(y, w[p + name]) for name in "qkv"], -1)
            act, _ = plain_delta.convolved(stacked, torch.zeros(cfg.taps - 1, stacked.shape[1]), w[p + "conv"].t())
            q, k = (act[:, j * qk * cfg.dim:(j + 1) * qk * cfg.dim].reshape(n, qk, cfg.dim).repeat_interleave(h // qk, 1)
                    for j in range(2))
            v = act[:, 2 * qk * cfg.dim:].reshape(n, h, cfg.vdim)
            decay, beta = plain_delta.gates(plain.linear(y, w[p + "a"]), plain.linear(y, w[p + "b"]), w[p + "A_log"],
                                            w[p + "dt_bias"])
            o, _ = plain_delta.rule(q, k, v, decay, beta, torch.zeros(h, cfg.dim, cfg.vdim), cfg.dim ** -0.5, cfg.eps)
            g = plain.linear(y, w[p + "g"]).reshape(n, h, cfg.vdim)
            o = o / (o.square().mean(-1, keepdim=True) + cfg.eps).sqrt() * w[p + "norm"].double() * g / (1 + (-g).exp())
            x = x + plain.linear(o.reshape(n, -1), w[p + "o"])
        y = plain.rms_norm(x, w[f"layers.{i}.feed_forward_norm.weight"], cfg.eps)
        p = f"layers.{i}.feed_forward."
        x = x + plain.linear(plain.silu_mul(plain.linear(y, w[p + "gate_proj.weight"]), plain.linear(y, w[p + "up_proj.weight"])),
                             w[p + "down_proj.weight"])
    return plain.linear(plain.rms_norm(x, w["final_norm.weight"], cfg.eps), w["embed.weight"])


SHAPES = {"wide": dict(width=96, layers=3, heads=4, qk_heads=2, dim=32, vdim=48, attention_every=2),
          "odd": dict(width=40, layers=2, heads=3, qk_heads=3, dim=20, vdim=12, taps=3, attention_every=9)}


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    from from_scratch_inference_engine_b200 import register_architecture, write_random_model
    from from_scratch_inference_engine_b200.config import unregister_architecture
    register_architecture(example.NAME, example.DeltaHybridConfig)
    root = tmp_path_factory.mktemp("delta")
    yield {name: write_random_model(root / name, example.DeltaHybridConfig(vocab=VOCAB, **shape), seed=3, std=0.2)
           for name, shape in SHAPES.items()}
    unregister_architecture(example.NAME)


def runner_of(folder, dtype="float32", page=4, pages=96, requests=6):
    from from_scratch_inference_engine_b200 import LoadedModel, ModelRunner
    model = LoadedModel.from_pretrained(folder, dtype=dtype, max_positions=512)
    return ModelRunner(model.model, model.runtime, page_size=page, num_pages=pages, max_requests=requests)


def step(runner, *entries):
    from from_scratch_inference_engine_b200 import StepEntry
    logits = runner.step([StepEntry(handle, tokens, [len(tokens) - 1]) for handle, tokens in entries])
    runner.raise_on_device_error()
    return logits.cpu().double().numpy()


# float32: sums over the widths in 32 bits through a few layers, as the package's other designs are held to
@pytest.mark.parametrize("name", list(SHAPES))
def test_logits_under_every_cutting(folders, name):
    folder = folders[name]
    requests = {k: helpers.random_ids(VOCAB, n, i) for i, (k, n) in enumerate({"a": 75, "b": 9, "c": 40, "d": 61}.items())}
    wanted = {key: plain_logits(folder, ids).numpy() for key, ids in requests.items()}
    runner = runner_of(folder)
    rows = helpers.run_trace_in_process(runner, helpers.trace_mixed(requests, seed=2, max_live=3))
    assert len(rows) == 185
    for (key, pos), row in rows.items():
        want = wanted[key][pos]
        assert np.abs(row - want).max() < 1e-4 * max(1.0, np.abs(want).max())
    runner.cache.check()


def test_whole_prompts_in_bfloat16(folders):
    """Every activation is rounded to 8 bits between the kernels: a few layers leave a few hundredths of the largest logit."""
    ids = helpers.random_ids(VOCAB, 70, 5)
    want = plain_logits(folders["wide"], ids).numpy()
    runner = runner_of(folders["wide"], "bfloat16")
    got = step(runner, (runner.cache.open("a"), ids))[0]
    assert np.abs(got - want[-1]).max() < 0.08 * np.abs(want).max()


@pytest.mark.parametrize("name", list(SHAPES))
@pytest.mark.parametrize("length", [1, 4, 18, 37])
def test_forked_requests_go_on_by_themselves(folders, name, length):
    folder = folders[name]
    ids = helpers.random_ids(VOCAB, length, 7)
    runner = runner_of(folder)
    parent = runner.cache.open("parent")
    step(runner, (parent, ids))
    children = runner.fork(parent, ["x", "y"])
    grandchild = runner.fork(children[0], ["z"])[0]
    handles = [parent] + children + [grandchild]
    seqs = [list(ids) for _ in handles]
    for turn in range(3):
        # a step of single tokens, of several tokens each, and once more, with the pages moved in between
        count = (1, 5, 2)[turn]
        fresh = [helpers.random_ids(VOCAB, count, 100 + 10 * turn + i) for i in range(len(handles))]
        rows = step(runner, *zip(handles, fresh))
        for seq, more, row in zip(seqs, fresh, rows):
            seq += more
            want = plain_logits(folder, seq)[-1].numpy()
            assert np.abs(row - want).max() < 1e-4 * max(1.0, np.abs(want).max())
        if turn == 0:
            runner.cache.close(handles.pop(1))               # one goes: holes in the pools
            seqs.pop(1)
            used = runner.compact()
            runner.cache.check()
            for pool, n in zip(runner.cache.pools, used):
                assert all((pool.ref_count(p) > 0) == (p < n) for p in range(pool.num_pages))
    for handle in handles:
        runner.cache.close(handle)
    assert runner.cache.slots.num_free == 6 and all(p.num_free == p.num_pages for p in runner.cache.pools)


def test_a_request_that_has_run_nothing_can_be_forked(folders):
    runner = runner_of(folders["odd"])
    used = runner.cache.open("used")
    step(runner, (used, [5, 6, 7]))                          # leaves something in its slot
    runner.cache.close(used)
    child, = runner.fork(runner.cache.open("parent"), ["child"])
    row = step(runner, (child, [9, 3]))[0]
    want = plain_logits(folders["odd"], [9, 3])[-1].numpy()
    assert np.abs(row - want).max() < 1e-4 * max(1.0, np.abs(want).max())


def engine_of(folder, max_batch=8, **given):
    from from_scratch_inference_engine_b200 import Engine, LoadedModel
    model = LoadedModel.from_pretrained(folder, dtype="float32", max_positions=512)
    return Engine(model, block_size=4, num_blocks=given.pop("num_blocks", 200), max_batch=max_batch, max_step_tokens=16, **given)


@pytest.mark.parametrize("pipeline", [True, False])
@pytest.mark.parametrize("max_batch", [8, 3, 1])
@pytest.mark.parametrize("length", [1, 2, 37])
def test_samples_of_one_prompt(folders, length, max_batch, pipeline):
    """The answers are those of requests that run the prompt each by themselves, which happens once here where there is room."""
    from from_scratch_inference_engine_b200 import SamplingParams
    folder, count = folders["wide"], 5
    prompt = helpers.random_ids(VOCAB, length, 11)
    params = [SamplingParams(temperature=0.8, seed=40 + i) for i in range(count)]
    engine = engine_of(folder, max_batch, pipeline=pipeline)
    other = engine.add_request(helpers.random_ids(VOCAB, 20, 12), SamplingParams(temperature=0.0), 4)
    ids = engine.add_samples(prompt, params, 7)
    engine.run_until_done()
    engine.runner.cache.check()
    alone = engine_of(folder)
    for rid, own in zip(ids, params):
        assert engine.output(rid) == alone.generate(prompt, own, 7)
    assert len(engine.output(other)) == 4
    if length > 1 and max_batch == 8:
        assert engine.stats()["tokens_prefilled"] == 20 + (length - 1) + count
    assert engine.runner.cache.slots.num_free == max_batch


def test_continuations_of_a_running_request(folders):
    from from_scratch_inference_engine_b200 import SamplingParams
    from from_scratch_inference_engine_b200.cache.pool import OutOfPages
    engine = engine_of(folders["wide"], max_batch=4)
    prompt = helpers.random_ids(VOCAB, 30, 13)
    first = engine.add_request(prompt, SamplingParams(temperature=0.0), 12)
    while len(engine.output(first)) < 5:
        engine.step()
    greedy, drawn = engine.fork(first, 2, [SamplingParams(temperature=0.0), SamplingParams(temperature=1.5, seed=3)])
    shared = list(engine.output(first))
    assert engine.output(greedy) == shared == engine.output(drawn)
    engine.compact()
    engine.run_until_done()
    assert engine.output(greedy) == engine.output(first) and len(engine.output(first)) == 12
    assert engine.output(drawn)[:len(shared)] == shared and engine.output(drawn) != engine.output(first)
    engine.runner.cache.check()
    for wrong in (lambda: engine.fork(first), lambda: engine.fork(drawn, 2, [SamplingParams()])):
        with pytest.raises(ValueError):
            wrong()
    running = engine.add_request(prompt, SamplingParams(temperature=0.0), 12)
    engine.step()
    with pytest.raises(RuntimeError):
        engine.fork(running, 4)
    tight = engine_of(folders["wide"], max_batch=4, num_blocks=9)
    rid = tight.add_request(prompt, SamplingParams(temperature=0.0), 4)
    while not tight.output(rid):
        tight.step()
    with pytest.raises(OutOfPages):
        tight.fork(rid, 3)
    tight.run_until_done()
    assert tight.output(rid) == engine.output(first)[:4]


def test_the_example_runs(capsys):
    from from_scratch_inference_engine_b200.config import unregister_architecture
    try:
        assert example.main(["--layers", "4", "--width", "256", "--prompt-len", "90", "--samples", "3", "--max-tokens", "6"]) == 0
    finally:
        unregister_architecture(example.NAME)
    lines = capsys.readouterr().out.splitlines()
    assert len(lines) == 5 and "prompt tokens run: 92 for 3 answers to a prompt of 90" in lines[3]
