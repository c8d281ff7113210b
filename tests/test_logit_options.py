"""What the sampler and the scheduler make of the options that change logits (no GPU needed)."""

import numpy as np
import pytest

from from_scratch_inference_engine_b200.cache import CacheManager, CacheNeed
from from_scratch_inference_engine_b200.engine.scheduler import Scheduler, SeqStatus
from from_scratch_inference_engine_b200.sampling import SamplingParams, pack_allowed, sorted_bias
from from_scratch_inference_engine_b200.sampling.sampler import stage_changes


@pytest.mark.parametrize("vocab", [1, 31, 32, 33, 151936])
@pytest.mark.parametrize("kind", [list, tuple, set, np.asarray, range, lambda ids: iter(ids)])
def test_allowed_tokens_as_bits(vocab, kind):
    rng = np.random.default_rng(vocab)
    ids = [int(t) for t in rng.choice(vocab, size=(vocab + 1) // 2, replace=False)]
    if kind is range:
        ids = range(0, vocab, 2)
    words = pack_allowed(kind(ids) if kind is not range else ids, vocab)
    assert words.dtype == np.int32 and words.shape == (-(-vocab // 32),)
    bits = words.view(np.uint32)
    for token in range(vocab) if vocab < 100 else rng.integers(0, vocab, 200):
        assert (int(bits[token // 32]) >> int(token) % 32 & 1) == (token in ids)
    if vocab % 32:
        assert int(bits[-1]) >> (vocab % 32) == 0


def test_allowed_tokens_that_are_none():
    assert not pack_allowed([], 50).any() and not pack_allowed(np.zeros(0, np.int64), 50).any()
    assert pack_allowed(np.arange(50) % 7 == 3, 50).tolist() == pack_allowed(range(3, 50, 7), 50).tolist()
    assert not pack_allowed(np.zeros(50, bool), 50).any()
    assert pack_allowed([7, 7, 7], 50).tolist() == [128, 0]              # twice is once
    for wrong in ([50], [-1], [1.5], [[1, 2]], [True, False], ["a"], np.ones(49, bool), np.ones((1, 50), bool)):
        with pytest.raises(ValueError):
            pack_allowed(wrong, 50)


def test_bias_lists():
    tokens, values = sorted_bias({9: 1.5, 0: -2, np.int64(4): 1e-3}, 10)
    assert tokens.tolist() == [0, 4, 9] and tokens.dtype == np.int32
    assert values.tolist() == np.asarray([-2, 1e-3, 1.5], np.float32).tolist()
    assert sorted_bias(None, 10) is None and sorted_bias({}, 10) is None
    for wrong in ({10: 1.0}, {-1: 1.0}, {3: float("inf")}, {3: float("nan")}, {1.5: 2.0}, {3: None}, {"x": 1.0}):
        with pytest.raises(ValueError):
            sorted_bias(wrong, 10)


@pytest.mark.parametrize("options", [dict(repetition_penalty=0.0), dict(repetition_penalty=-1.0), dict(repetition_penalty=float("inf")),
                                     dict(repetition_penalty=float("nan")), dict(presence_penalty=float("inf")),
                                     dict(frequency_penalty=float("nan")), dict(logit_bias={100: 1.0}), dict(allowed=[1, 2])])
def test_options_that_make_no_sense(options):
    with pytest.raises(ValueError):
        SamplingParams(**options).check(100)
    SamplingParams(repetition_penalty=1.2, presence_penalty=-0.5, frequency_penalty=2, logit_bias={99: -1e9}, allowed=lambda o: None).check(100)


@pytest.mark.parametrize("name", ["repetition_penalty", "presence_penalty", "frequency_penalty"])
def test_penalties_are_checked_as_the_numbers_they_are_applied_as(name):
    """What is finite, or positive, in 64 bits only is refused; the ends of the range of 32 bits are taken."""
    top, low = float(np.finfo(np.float32).max), float(np.finfo(np.float32).tiny)
    wrong = [1e39, top * (1 + 2.0 ** -24), np.inf, np.nan, -np.inf]
    wrong += [1e-50, low / 2, 0.0, -0.0, -1.0] if name == "repetition_penalty" else [-1e39]
    for value in wrong:
        with pytest.raises(ValueError, match=name):
            SamplingParams(**{name: value}).check(100)
    for value in [top, 1] + ([low, np.float32(1.5)] if name == "repetition_penalty" else [-top, 1e-50, 0, np.float32(-2)]):
        params = SamplingParams(**{name: value})
        params.check(100)
        host, histories, _, _ = stage_changes([params], [0], [None], None)
        staged = host[histories[1]].view(np.float32)
        assert np.isfinite(staged).all() and staged[0] >= low


def test_what_is_staged_for_the_rows():
    params = [SamplingParams(), SamplingParams(repetition_penalty=1.5, frequency_penalty=0.25), SamplingParams(presence_penalty=2.0)]
    biases = [sorted_bias({5: 1.0, 2: 3.0}, 40), None, sorted_bias({39: -4.0}, 40)]
    masks = [None, pack_allowed([1], 40), pack_allowed([2], 40)]
    host, histories, lists, mask_of = stage_changes(params, [-1, 4, 0], biases, masks)
    assert host.dtype == np.int32 and host.size == 3 + 9 + 4 + 3 + 3 + 3
    assert host[histories[0]].tolist() == [-1, 4, 0]
    assert host[histories[1]].view(np.float32).tolist() == [1, 0, 0, 1.5, 0, 0.25, 1, 2, 0]
    assert host[lists[0]].tolist() == [0, 2, 2, 3] and host[lists[1]].tolist() == [2, 5, 39]
    assert host[lists[2]].view(np.float32).tolist() == [3, 1, -4]
    assert host[mask_of].tolist() == [-1, 0, 1]
    assert stage_changes(params[:1], None, [None], [None]) == (None, None, None, None)
    host, histories, lists, mask_of = stage_changes(params[:2], None, [None, biases[0]], None)
    assert histories is None and mask_of is None and host[lists[0]].tolist() == [0, 0, 2]


@pytest.mark.parametrize("overlapped", [False, True])
def test_a_request_to_which_no_token_may_come_ends_without_one(overlapped):
    """As the engine does it: the item is marked before its token is recorded; the step that was planned behind it runs for
    nothing."""
    cache = CacheManager([CacheNeed(1, 16)], 4, 32, 4)
    s = Scheduler(cache, 4, 16)
    first, second = (s.add([1, 2, 3], SamplingParams(temperature=0.0), 5, -1, seed=0) for _ in range(2))

    def run(items):
        for item in items:
            cache.reserve(item.seq.handle, len(item.tokens))
            cache.commit(item.seq.handle, len(item.tokens))
    items = s.plan()
    run(items)
    s.finish_step(items, [7, 8])
    items = s.plan()
    run(items)
    items[0].ends = True
    s.begin_step(items)
    if overlapped:
        behind = s.plan(can_preempt=False)
        assert [i.seq.id for i in behind] == [first, second]
        run(behind)
    s.resolve_step(items, [9, 9])
    assert s.sequences[first].output == [7] and s.sequences[first].status is SeqStatus.Finished
    assert s.sequences[second].output == [8, 9]
    if overlapped:
        s.begin_step(behind)
        s.resolve_step(behind, [3, 3])
        assert s.sequences[first].output == [7] and s.sequences[second].output == [8, 9, 3]
    assert s.running == [second]
    cache.check()
