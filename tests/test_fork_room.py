"""How often a request can be continued, and answers to one prompt where room lacks or a step fails."""
import random
import sys
from pathlib import Path

import pytest

import helpers
from test_cache_fork import grow, manager
from from_scratch_inference_engine_b200.cache.pool import OutOfPages

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))
import delta_samples as example  # noqa: E402

VOCAB = 97


@pytest.mark.parametrize("window", [0, 5])
@pytest.mark.parametrize("prefix", [False, True])
def test_room_is_what_fork_can_make(window, prefix):
    """As many as `fork_room` says can be made, one more cannot, wherever the request stands."""
    rng = random.Random(window)
    for length in list(range(12)) * 3:
        cache = manager(pages=rng.randint(6, 14), slots=rng.randint(1, 9), window=window, prefix=prefix and not window)
        parent = cache.open("parent")
        if length:
            grow(cache, parent, length)
        if cache.prefix_enabled and rng.random() < 0.7:        # pages that only the prefix cache holds count as free
            other = cache.open("other") if cache.can_open() else None
            if other is not None:
                if cache.can_reserve(other, 9):
                    grow(cache, other, 9)
                    cache.register_prefix(other, list(range(50, 59)))
                cache.close(other)
        room = cache.fork_room(parent)
        with pytest.raises(OutOfPages):
            cache.fork(parent, range(room + 1))
        children, _ = cache.fork(parent, range(room))
        assert len(children) == room
        cache.check()


@pytest.fixture(scope="module")
def folder(tmp_path_factory):
    from from_scratch_inference_engine_b200 import register_architecture, write_random_model
    from from_scratch_inference_engine_b200.config import unregister_architecture
    register_architecture(example.NAME, example.DeltaHybridConfig)
    yield write_random_model(tmp_path_factory.mktemp("samples") / "m", example.DeltaHybridConfig(
        vocab=VOCAB, width=96, layers=3, heads=4, qk_heads=2, dim=32, vdim=48, attention_every=2), seed=3, std=0.2)
    unregister_architecture(example.NAME)


def engine_of(folder, num_blocks, max_batch=8, pipeline=True):
    from from_scratch_inference_engine_b200 import Engine, LoadedModel
    model = LoadedModel.from_pretrained(folder, dtype="float32", max_positions=512)
    return Engine(model, block_size=4, num_blocks=num_blocks, max_batch=max_batch, max_step_tokens=16, pipeline=pipeline)


def params_of(count):
    from from_scratch_inference_engine_b200 import SamplingParams
    return [SamplingParams(temperature=0.8, seed=40 + i) for i in range(count)]


@pytest.mark.gpu
@pytest.mark.parametrize("pipeline", [True, False])
def test_as_many_answers_share_the_prompt_as_pages_allow(folder, pipeline):
    """Eleven pages: the prompt's eight leave three, for three of four more answers; the fourth runs the prompt by itself."""
    prompt, params = helpers.random_ids(VOCAB, 30, 11), params_of(5)
    engine = engine_of(folder, 11, pipeline=pipeline)
    ids = engine.add_samples(prompt, params, 3)
    engine.run_until_done()
    engine.runner.cache.check()
    alone = engine_of(folder, 200)
    assert [engine.output(i) for i in ids] == [alone.generate(prompt, p, 3) for p in params]
    assert engine.stats()["tokens_prefilled"] == 29 + 4 + 30 and engine.preemptions() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("pipeline", [True, False])
def test_a_step_that_fails_holds_nothing_back(folder, pipeline, monkeypatch):
    prompt, params = helpers.random_ids(VOCAB, 37, 11), params_of(3)
    engine = engine_of(folder, 200, pipeline=pipeline)
    step, calls = engine.step, []

    def failing():
        calls.append(1)
        if len(calls) == 2:
            raise RuntimeError("lost")
        return step()
    monkeypatch.setattr(engine, "step", failing)
    with pytest.raises(RuntimeError, match="lost"):
        engine.add_samples(prompt, params, 5)
    monkeypatch.undo()
    engine.run_until_done()
    assert engine.output(0) == engine_of(folder, 200).generate(prompt, params[0], 5)
    engine.runner.cache.check()
