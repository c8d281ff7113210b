"""Penalties, biases and allowed tokens through the sampler, the engine, `LLM` and the command line."""

import json

import numpy as np
import pytest
import torch

import helpers
import plain_qwen2 as plain
from helpers import TINY

pytestmark = pytest.mark.gpu
VOCAB = {"A": 256, "B": 384}


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    root = tmp_path_factory.mktemp("models")
    return {name: helpers.make_model_dir(root, name) for name in ("A", "B", "E")}


def plainly(row, prompt, output, params):
    """float64 logits as the options leave them."""
    row = np.array(row, dtype=np.float64)
    count = np.bincount(np.asarray(output, dtype=np.int64), minlength=len(row))
    seen = np.bincount(np.asarray(list(prompt) + list(output), dtype=np.int64), minlength=len(row)) > 0
    theta = np.float64(np.float32(params.repetition_penalty))
    row = np.where(seen, np.where(row > 0, row / theta, row * theta), row)
    row -= np.float32(params.presence_penalty) * (count > 0) + np.float64(np.float32(params.frequency_penalty)) * count
    for token, value in (params.logit_bias or {}).items():
        row[token] += np.float32(value)
    allowed = params.allowed(output) if params.allowed else None
    if allowed is not None:
        mask = np.full(len(row), -np.inf)
        mask[list(allowed)] = 0
        row = row + mask
    return row


# ------------------------------------------------------------------------------------ the sampler
def test_histories_follow_the_chosen_tokens():
    """Nine steps over fifteen rows, greedy and drawn, some with a history and some without; a row in the middle ends and
    another request takes its slot."""
    from from_scratch_inference_engine_b200.sampling import Sampler, SamplingParams, TokenHistory
    vocab, rows = 1003, 15
    gen = torch.Generator(device="cuda").manual_seed(5)
    sampler, history = Sampler("cuda:0"), TokenHistory("cuda:0", vocab)
    error = torch.zeros(1, dtype=torch.int32, device="cuda")
    forms = [SamplingParams(temperature=0.0), SamplingParams(temperature=0.0, repetition_penalty=1.7),
             SamplingParams(temperature=0.0, presence_penalty=1.5), SamplingParams(temperature=0.0, frequency_penalty=0.8),
             SamplingParams(temperature=0.0, repetition_penalty=0.6, presence_penalty=-0.5, frequency_penalty=-0.25, logit_bias={3: 2.0, 900: -1.0})]
    params = [forms[r % 5] for r in range(rows)]
    prompts = [[int(t) for t in np.random.default_rng(r).integers(0, vocab, 1 + 40 * (r % 4))] for r in range(rows)]
    outputs, ids = [[] for _ in range(rows)], list(range(rows))
    base = torch.randn(rows, vocab, device="cuda", generator=gen) * 2
    for step in range(9):
        if step == 5:
            history.release(ids[6])
            ids[6], prompts[6], outputs[6] = 100, [1, 2, 3], []
        logits = (base + 0.3 * torch.randn(rows, vocab, device="cuda", generator=gen)).contiguous()
        before = logits.double().cpu().numpy()
        slots = [-1] * rows
        known = iter(history.slots([(ids[r], prompts[r], outputs[r]) for r in range(rows) if params[r].penalised], error))
        slots = [next(known) if p.penalised else -1 for p in params]
        picked = sampler.sample_async(logits, params, [0] * rows, [step] * rows, error, slots, history)
        chosen = picked.result()
        assert picked.fault == 0
        for r, token in enumerate(chosen):
            want = plainly(before[r], prompts[r], outputs[r], params[r])
            # a few roundings of 32 bits of numbers below 16
            assert want[token] >= want.max() - 1e-5
            outputs[r].append(token)
    assert any(len(set(o)) < len(o) for o in outputs) and len(history) == sum(p.penalised for p in params)
    for slot, r in zip(history.slots([(ids[r], prompts[r], outputs[r]) for r in range(rows) if params[r].penalised], error),
                       [r for r in range(rows) if params[r].penalised]):
        assert history.counts[slot].tolist() == np.bincount(outputs[r], minlength=vocab).tolist()


@pytest.mark.parametrize("vocab", [151936, 32003, 50])
@pytest.mark.parametrize("top_k,top_p", [(0, 1.0), (40, 1.0), (40, 0.9), (0, 0.9), (300, 0.5), (1, 1.0)])
def test_draws_stay_inside_what_is_allowed(vocab, top_k, top_p):
    """From 1 token to all of them; what is forbidden has the largest logits."""
    from from_scratch_inference_engine_b200.sampling import Sampler, SamplingParams, pack_allowed
    sampler = Sampler("cuda:0")
    rng = np.random.default_rng(vocab + top_k)
    sets = [rng.choice(vocab, size=max(1, min(vocab, n)), replace=False) for n in (1, 2, 3, 7, 39, 41, 299, 400, 20000, vocab)]
    logits = torch.randn(len(sets) + 1, vocab, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) * 3
    for r, tokens in enumerate(sets):
        logits[r] += 30
        logits[r, torch.from_numpy(tokens).cuda()] -= 30
    everything = lambda output: None
    params = [SamplingParams(1.3, top_k, top_p, allowed=everything)] * len(logits)
    masks = [pack_allowed(tokens, vocab) for tokens in sets] + [None]
    for index in range(12):
        chosen = sampler.sample_async(logits.clone(), params, list(range(len(logits))), [index] * len(logits), masks=masks).result()
        for r, tokens in enumerate(sets):
            assert chosen[r] in tokens


def test_the_sampler_refuses_what_it_cannot_do():
    from from_scratch_inference_engine_b200.sampling import Sampler, SamplingParams, TokenHistory, pack_allowed
    sampler, history = Sampler("cuda:0"), TokenHistory("cuda:0", 40)
    logits = torch.zeros(2, 40, device="cuda")
    penalised, masked = SamplingParams(repetition_penalty=1.1), SamplingParams(allowed=lambda output: [1])
    error = torch.zeros(1, dtype=torch.int32, device="cuda")
    for params, given in (([penalised] * 2, {}), ([masked] * 2, {}), ([penalised] * 2, dict(slots=[0], history=history)),
                          ([masked] * 2, dict(masks=[pack_allowed([1], 40)])), ([SamplingParams()] * 2, dict(slots=[0, 1], biases=[None]))):
        with pytest.raises(ValueError):
            sampler.sample_async(logits, params, [0, 0], [0, 0], error, **given)
    with pytest.raises(ValueError, match="no token is allowed"):
        sampler.sample_async(logits, [masked] * 2, [0, 0], [0, 0], error, masks=[pack_allowed([1], 40), pack_allowed([], 40)])
    with pytest.raises(ValueError):
        history.slots([(1, [2], []), (1, [2], [])], error)
    assert len(history) == 0
    # a history of another vocabulary
    history.slots([(1, [2], []), (2, [], [])], error)
    with pytest.raises(Exception, match="vocabulary"):
        sampler.sample_async(torch.zeros(2, 41, device="cuda"), [penalised] * 2, [0, 0], [0, 0], error, [0, 1], history)
    assert not error.item()


# ------------------------------------------------------------------------------------- the engine
def engine_for(folder, dtype="float32", **kwargs):
    from from_scratch_inference_engine_b200 import Engine, LoadedModel
    options = dict(block_size=4, num_blocks=128, seed=0, max_batch=8, max_step_tokens=16)
    options.update(kwargs)
    model = LoadedModel.from_pretrained(folder, dtype=dtype, max_positions=options["block_size"] * options["num_blocks"])
    return Engine(model, **options)


def assert_greedy_agrees(folder, prompt, got, params, stop=None):
    """Token for token, or near ties: 1e-4 of the largest logit, what 32-bit sums in another order may come to, times what a
    penalty multiplies it by."""
    config, weights = plain.load(folder)
    output = []
    for token in got:
        row = plain.forward(config, weights, list(prompt) + output)[-1].numpy()
        want = plainly(row, prompt, output, params)
        assert want[token] >= want.max() - 2e-4 * max(1.0, np.abs(row).max())
        output.append(token)


def even_then_odd(output):
    """Even tokens, odd ones, everything, and after six tokens nothing."""
    if len(output) >= 6:
        return []
    return (range(0, 256, 2), np.arange(1, 256, 2), None)[len(output) % 3]


PARAMS = [dict(repetition_penalty=1.8), dict(presence_penalty=0.4, frequency_penalty=0.3), dict(logit_bias={7: 0.6, 250: 0.5, 3: -2.0}), {},
          dict(allowed=even_then_odd), dict(repetition_penalty=0.7, frequency_penalty=0.5, logit_bias={9: 0.3}, allowed=even_then_odd)]


@pytest.mark.parametrize("pipeline", [True, False])
@pytest.mark.parametrize("blocks,max_batch", [(128, 8), (14, 8), (128, 2)])
@pytest.mark.parametrize("masked", [False, True])
def test_greedy_answers_under_options(folders, pipeline, blocks, max_batch, masked):
    """Requests with and without options in one batch; with 14 blocks some are preempted and run again, with a batch of two
    they wait."""
    from from_scratch_inference_engine_b200 import SamplingParams
    engine = engine_for(folders["A"], num_blocks=blocks, max_batch=max_batch, pipeline=pipeline)
    params = [SamplingParams(temperature=0.0, **given) for given in PARAMS[:len(PARAMS) if masked else 4]]
    prompts = [helpers.random_ids(256, n, 20 + n) for n in (5, 17, 1, 9, 12, 3)][:len(params)]
    ids = [engine.add_request(p, q, 12) for p, q in zip(prompts, params)]
    engine.run_until_done()
    engine.runner.raise_on_device_error()
    engine.runner.cache.check()
    assert blocks > 14 or engine.preemptions() > 0
    for rid, prompt, own in zip(ids, prompts, params):
        output = engine.output(rid)
        assert len(output) == (6 if own.allowed else 12)
        assert_greedy_agrees(folders["A"], prompt, output, own)
    assert len(engine.history) == 0 and engine.runner.cache.slots.num_free == max_batch


def test_more_histories_than_there_were_slots(folders):
    """Twenty requests at once, twice: histories grow, and a second request finds nothing of the first in its slot."""
    from from_scratch_inference_engine_b200 import SamplingParams
    engine = engine_for(folders["A"], max_batch=24, num_blocks=256)
    own = SamplingParams(temperature=0.0, frequency_penalty=0.2, repetition_penalty=1.3)
    for turn in range(2):
        prompts = [helpers.random_ids(256, 4 + i, 50 * turn + i) for i in range(20)]
        ids = [engine.add_request(p, own, 6) for p in prompts]
        engine.run_until_done()
        for rid, prompt in list(zip(ids, prompts))[::4]:
            assert_greedy_agrees(folders["A"], prompt, engine.output(rid), own)
        assert len(engine.history) == 0


def test_continuations_have_histories_of_their_own(folders):
    from from_scratch_inference_engine_b200 import SamplingParams
    engine = engine_for(folders["A"])
    prompt = helpers.random_ids(256, 21, 3)
    first = engine.add_request(prompt, SamplingParams(temperature=0.0), 10)
    while len(engine.output(first)) < 4:
        engine.step()
    params = [SamplingParams(temperature=0.0, **given) for given in PARAMS[:3]]
    ids = engine.fork(first, 3, params)
    begun = list(engine.output(first))
    engine.run_until_done()
    for rid, own in zip(ids, params):
        output = engine.output(rid)
        assert output[:len(begun)] == begun and len(output) == 10
        config, weights = plain.load(folders["A"])
        for at in range(len(begun), 10):
            row = plain.forward(config, weights, prompt + output[:at])[-1].numpy()
            want = plainly(row, prompt, output[:at], own)
            assert want[output[at]] >= want.max() - 2e-4 * max(1.0, np.abs(row).max())


@pytest.mark.parametrize("pipeline", [True, False])
def test_what_a_callback_raises(folders, pipeline):
    """It comes out of `step`; that request has ended, the others have lost nothing."""
    from from_scratch_inference_engine_b200 import SamplingParams, SeqStatus
    engine = engine_for(folders["A"], pipeline=pipeline)
    prompts = [helpers.random_ids(256, n, n) for n in (6, 9, 4)]

    def breaks(output):
        if len(output) == 3:
            raise KeyError("grammar")
        return None
    params = [SamplingParams(temperature=0.0), SamplingParams(temperature=0.0, allowed=breaks),
              SamplingParams(temperature=0.0, allowed=lambda output: [5, 300] if len(output) == 5 else None)]
    ids = [engine.add_request(p, q, 9) for p, q in zip(prompts, params)]
    with pytest.raises(KeyError, match="grammar"):
        engine.run_until_done()
    with pytest.raises(ValueError, match="allowed"):
        engine.run_until_done()
    engine.run_until_done()
    assert [len(engine.output(i)) for i in ids] == [9, 3, 5]
    assert all(engine.status(i) is SeqStatus.Finished for i in ids)
    alone = engine_for(folders["A"])
    for rid, prompt in zip(ids, prompts):
        assert engine.output(rid) == alone.generate(prompt, params[0], 9)[:len(engine.output(rid))]
    engine.runner.cache.check()
    assert engine.runner.cache.slots.num_free == 8


def test_what_a_callback_raises_while_another_request_is_sampled(folders):
    """`add_samples` runs steps of other requests: it returns its ids, the next step raises.  Of two that raise in one step the
    first comes out, both requests have ended."""
    from from_scratch_inference_engine_b200 import SamplingParams, SeqStatus
    engine = engine_for(folders["A"])

    def breaks(output):
        raise KeyError(f"after {len(output)}")
    broken = [engine.add_request([5, 6, 7 + i], SamplingParams(temperature=0.0, allowed=breaks), 5) for i in range(2)]
    prompt = helpers.random_ids(256, 40, 3)
    ids = engine.add_samples(prompt, [SamplingParams(temperature=0.9, seed=i) for i in range(3)], 4)
    assert len(ids) == 3
    with pytest.raises(KeyError, match="after 0"):
        engine.step()
    engine.run_until_done()
    assert [len(engine.output(i)) for i in ids] == [4, 4, 4]
    assert all(engine.status(i) is SeqStatus.Finished and not engine.output(i) for i in broken)


@pytest.mark.parametrize("pipeline", [True, False])
def test_what_several_callbacks_raise(folders, pipeline):
    """The first comes out; its notes say whose it was, and what the others raised, in the same step and in later ones of
    `add_samples`."""
    from from_scratch_inference_engine_b200 import SamplingParams, SeqStatus
    engine = engine_for(folders["A"], pipeline=pipeline)

    def breaks_after(count, error):
        def allowed(output):
            if len(output) == count:
                raise error
        return allowed
    errors = [KeyError("one"), ValueError("two"), KeyError("three")]
    broken = [engine.add_request([5, 6, 7 + i], SamplingParams(temperature=0.0, allowed=breaks_after(i // 2, error)), 5)
              for i, error in enumerate(errors)]
    ids = engine.add_samples(helpers.random_ids(256, 40, 3), [SamplingParams(temperature=0.9, seed=i) for i in range(3)], 4)
    assert len(ids) == 3
    with pytest.raises(KeyError, match="one") as caught:
        engine.step()
    assert caught.value is errors[0]
    notes = caught.value.__notes__
    assert len(notes) == 3
    for rid, note, text in zip(broken, notes, ("request", "ValueError('two')", "KeyError('three')")):
        assert f"request {rid}" in note and text in note
    engine.run_until_done()
    assert [len(engine.output(i)) for i in broken + ids] == [0, 0, 1, 4, 4, 4]
    assert all(engine.status(i) is SeqStatus.Finished for i in broken)


@pytest.mark.parametrize("pipeline", [True, False])
def test_a_callback_that_is_interrupted(folders, pipeline):
    """What is no Exception comes out of `step` as well once the step is recorded, in front of what others raised, and of
    `add_samples` at once; the others lose nothing."""
    from from_scratch_inference_engine_b200 import SamplingParams, SeqStatus

    class Stop(BaseException):
        pass
    engine = engine_for(folders["A"], pipeline=pipeline)
    prompts = [helpers.random_ids(256, n, n) for n in (6, 5, 4)]      # one step's tokens

    def breaks_after(count, error):
        def allowed(output):
            if len(output) == count:
                raise error
        return allowed
    greedy = SamplingParams(temperature=0.0)
    params = [greedy, SamplingParams(temperature=0.0, allowed=breaks_after(3, KeyError("other"))),
              SamplingParams(temperature=0.0, allowed=breaks_after(3, Stop("now")))]
    ids = [engine.add_request(p, q, 9) for p, q in zip(prompts, params)]
    with pytest.raises(Stop, match="now") as caught:
        engine.run_until_done()
    assert [f"request {i}" in note for i, note in zip((ids[2], ids[1]), caught.value.__notes__)] == [True, True]
    engine.run_until_done()
    assert [len(engine.output(i)) for i in ids] == [9, 3, 3]
    alone = engine_for(folders["A"])
    for rid, prompt in zip(ids, prompts):
        assert engine.output(rid) == alone.generate(prompt, greedy, 9)[:len(engine.output(rid))]
    stopping = engine.add_request(prompts[0], params[2], 9)
    prompt = helpers.random_ids(256, 100, 3)
    with pytest.raises(Stop, match="now"):
        engine.add_samples(prompt, [greedy] * 2, 4)
    engine.run_until_done()
    assert engine.status(stopping) is SeqStatus.Finished and len(engine.output(stopping)) == 3
    assert engine.output(stopping + 1) == alone.generate(prompt, greedy, 4)
    engine.runner.cache.check()
    assert engine.runner.cache.slots.num_free == 8 and len(engine.history) == 0


@pytest.mark.parametrize("pipeline", [True, False])
def test_no_memory_for_a_history(folders, pipeline, monkeypatch):
    """It comes out of `step` before anything of the step has run: tried again, every request gives the tokens that it gives alone."""
    from from_scratch_inference_engine_b200 import SamplingParams
    from from_scratch_inference_engine_b200.sampling import TokenHistory
    engine = engine_for(folders["A"], pipeline=pipeline, num_blocks=200, max_batch=20, max_step_tokens=40)
    params = [SamplingParams(temperature=0.0, **PARAMS[i % 4]) for i in range(18)]
    prompts = [helpers.random_ids(256, 3 + i, i) for i in range(18)]
    grow, fails = TokenHistory._grow, [0]

    def scarce(self, slots):
        if len(self._free) < slots and fails[0] < 6:               # three times for the first slots, twice for more
            fails[0] += 1
            if fails[0] % 4:
                raise torch.OutOfMemoryError("CUDA out of memory")
        return grow(self, slots)
    monkeypatch.setattr(TokenHistory, "_grow", scarce)
    ids = [engine.add_request(p, q, 7) for p, q in zip(prompts, params)]
    raised = 0
    while engine.has_work():
        try:
            assert engine.step() > 0
        except torch.OutOfMemoryError:
            raised += 1
    assert raised == 5 and fails[0] == 6
    engine.runner.cache.check()
    assert engine.runner.cache.slots.num_free == 20 and len(engine.history) == 0
    alone = engine_for(folders["A"], num_blocks=200)
    for rid, prompt, own in zip(ids, prompts, params):
        assert engine.output(rid) == alone.generate(prompt, own, 7)


def test_options_are_refused_before_anything_is_kept(folders):
    from from_scratch_inference_engine_b200 import SamplingParams
    engine = engine_for(folders["A"])
    for wrong in (dict(repetition_penalty=0.0), dict(logit_bias={256: 1.0}), dict(allowed=3), dict(presence_penalty=float("nan"))):
        with pytest.raises(ValueError):
            engine.add_request([1, 2], SamplingParams(**wrong))
        with pytest.raises(ValueError):
            engine.add_samples([1, 2, 3], [SamplingParams(), SamplingParams(**wrong)])
    running = engine.add_request([1, 2, 3, 4, 5], SamplingParams(temperature=0.0), 8)
    engine.step()
    with pytest.raises(ValueError):
        engine.fork(running, 1, [SamplingParams(logit_bias={-1: 0.0})])
    assert list(engine.scheduler.sequences) == [running]
    engine.run_until_done()
    assert len(engine.output(running)) == 8


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_all_of_it_together(folders, dtype):
    """Answers to one prompt that read its keys once, with penalties, a bias and a grammar: in float32 the tokens of requests
    that run alone and share nothing."""
    from from_scratch_inference_engine_b200 import GenerationConfig, LLM
    config = GenerationConfig(max_tokens=11, temperature=0.9, top_k=20, seed=70, repetition_penalty=1.4, presence_penalty=0.2,
                              frequency_penalty=0.3, logit_bias={5: 1.0, 77: -3.0},
                              allowed=lambda output: range(len(output) % 3, 300, 3))
    prompt = helpers.random_ids(300, 150, 8)
    llm = LLM(folders["E"], num_blocks=200, dtype=dtype, eos_id=-1, max_batch=16, shared_attention=True)
    runner = llm.engine.runner
    runner.shared_min_bytes = runner.shared_min_part = runner.shared_least_keys = 0
    answers = llm.generate_samples(prompt, 12, config)
    runner.raise_on_device_error()
    assert any(shared for _, _, shared in runner._graphs)
    for answer in answers:
        assert len(answer) == 11 and all(token % 3 == at % 3 for at, token in enumerate(answer))
    assert len(set(map(tuple, answers))) == 12
    if dtype == "float32":
        from dataclasses import replace
        alone = LLM(folders["E"], num_blocks=200, dtype=dtype, eos_id=-1, max_batch=16)
        for i, answer in enumerate(answers):
            assert answer == alone.generate_ids(prompt, replace(config, seed=70 + i))


def test_the_command_line_has_the_options(tmp_path, capsys):
    from from_scratch_inference_engine_b200 import cli
    config_path = tmp_path / "config_in.json"
    config_path.write_text(json.dumps(TINY["E"]["config"]))
    folder = tmp_path / "model"
    common = ["--model-dir", str(folder), "--prompt-ids", "5,17,3,88,41", "--num-requests", "2", "--max-tokens", "9", "--num-blocks", "32",
              "--json"]
    assert cli.main(common + ["--random-weights", str(config_path), "--std", "0.08", "--allowed-ids", "4,9,33,100,101,102,103,104,105",
                              "--shared-attention", "1", "--presence-penalty", "1000"]) == 0
    outputs = json.loads(capsys.readouterr().out)["outputs"]
    assert sorted(outputs[0]) == [4, 9, 33, 100, 101, 102, 103, 104, 105] and outputs[0] == outputs[1]
    assert cli.main(common + ["--logit-bias", "7:100,8:99.5", "--frequency-penalty", "0.2", "--repetition-penalty", "1.0"]) == 0
    assert set(json.loads(capsys.readouterr().out)["outputs"][0]) == {7, 8}
    for wrong in (["--logit-bias", "7"], ["--allowed-ids", "4,x"]):
        with pytest.raises(SystemExit):
            cli.main(common + wrong)
