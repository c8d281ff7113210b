"""Working memory of the chunked gated delta rule: as much as the requests that go in chunks need, and all of it there before
serving starts."""
import random
import sys
from pathlib import Path

import pytest
import torch

from test_gpu_delta_rule import Case, near

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))
import delta_samples as example  # noqa: E402

gpu = pytest.mark.gpu


def test_the_chunks_of_any_step_fit():
    """Counted, for requests of any lengths (host only)."""
    from from_scratch_inference_engine_b200.kernels.ops import _delta_chunks
    rng = random.Random(0)
    tight = 0
    for _ in range(4000):
        few = rng.choice([0, 4, 6, 10, 16])
        lengths = [rng.choice([0, 1, 1, 1, few, few + 1, 32, 33, 64, rng.randint(1, 300)]) for _ in range(rng.randint(1, 40))]
        told = rng.randint(0, sum(n <= 1 for n in lengths)) if few else 0
        chunks = sum(-(-n // 32) for n in lengths if n > few)
        room = _delta_chunks(sum(lengths), len(lengths), told, few, 32)
        assert chunks <= room
        tight += chunks == room
    assert tight > 0


def test_mixers_that_know_nothing_of_reserving():
    """A registered mixer of the older interface, beside one that takes memory (host only)."""
    from types import SimpleNamespace
    from from_scratch_inference_engine_b200.parts.model import DecoderModel
    seen = []
    mixers = [object(), SimpleNamespace(reserve=lambda tokens, requests: seen.append((tokens, requests)))]
    DecoderModel.reserve(SimpleNamespace(blocks=[SimpleNamespace(mixer=m) for m in mixers]), 7, 3)
    assert seen == [(7, 3)]


def chunk_bytes(case):
    from from_scratch_inference_engine_b200.kernels import ops
    return ops.delta().fsie_delta_chunk_bytes(case.heads, case.share, case.dim, ops._tag(case.qkv.dtype))


@gpu
@pytest.mark.parametrize("singles,long", [(255, 1793), (63, 512), (200, 40)])
def test_decoded_tokens_beside_a_portion_take_no_chunks(singles, long):
    case = Case([1] * singles + [long], 4, 1, 64, 64, torch.bfloat16)
    want = case.want()
    for ones in (0, singles):
        case.run(long, ones=ones)                              # the allocator's other pieces
        out = torch.full((case.tokens, case.heads * case.vdim), 7e7, device="cuda")
        from test_gpu_delta_rule import ints
        from from_scratch_inference_engine_b200.kernels import ops
        lists = ints(case.starts), ints(case.lengths), ints(case.slots)
        state = case.state.clone()
        torch.cuda.reset_peak_memory_stats()                   # (asked for, not what the allocator rounds it to)
        before = torch.cuda.memory_stats()["requested_bytes.all.current"]
        ops.gated_delta_rule(case.qkv, *case.offs, case.decay, case.beta, *lists, case.items, state, out, case.heads,
                             case.dim, case.vdim, longest=long, ones=ones)
        taken = torch.cuda.memory_stats()["requested_bytes.all.peak"] - before
        # the portion's chunks; without `ones` as many more as requests of more than ten tokens could have begun
        most = case.tokens // 32 + (1 if ones else min(case.items, case.tokens // 11))
        assert taken <= most * chunk_bytes(case) + 1024
        near(out, want[0])
        near(state[case.slots[-1]], want[1][case.slots[-1]])


@gpu
def test_memory_given_by_the_caller():
    from from_scratch_inference_engine_b200.kernels import ops
    from test_gpu_delta_rule import ints
    case = Case([70, 1, 12, 33], 2, 1, 64, 64, torch.float32)
    lists = ints(case.starts), ints(case.lengths), ints(case.slots)
    size = ops.gated_delta_room(case.tokens, case.items, case.heads, case.dim, torch.float32)
    assert ops.gated_delta_room(100, 4, 2, 200, torch.float32) == 0

    def call(room):
        out, state = torch.empty(case.tokens, case.heads * case.vdim, device="cuda"), case.state.clone()
        ops.gated_delta_rule(case.qkv, *case.offs, case.decay, case.beta, *lists, case.items, state, out, case.heads,
                             case.dim, case.vdim, longest=70, room=room)
        return out, state
    room = torch.full((size + 64,), 171, dtype=torch.uint8, device="cuda")
    for got, want in zip(call(room[:size]), case.want()):
        near(got, want)
    assert (room[size:] == 171).all()
    for wrong in (room[:100], room[8:], room.int(), room.cpu(), room[::2]):
        with pytest.raises(ops.KernelError):
            call(wrong)


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_no_step_needs_more_than_was_reserved(dtype, tmp_path):
    from from_scratch_inference_engine_b200 import LoadedModel, ModelRunner, StepEntry, register_architecture, write_random_model
    from from_scratch_inference_engine_b200.config import unregister_architecture
    register_architecture(example.NAME, example.DeltaHybridConfig)
    try:
        config = example.DeltaHybridConfig(vocab=97, width=96, layers=3, heads=4, qk_heads=2, dim=32, vdim=48, attention_every=2)
        model = LoadedModel.from_pretrained(write_random_model(tmp_path / "m", config, seed=3, std=0.2), dtype=dtype, max_positions=512)
        runner = ModelRunner(model.model, model.runtime, page_size=4, num_pages=600, max_requests=64, max_step_tokens=400)
        assert runner.reserve_step_memory() == 400
        key = ("gated_delta.room", torch.uint8)
        held = model.runtime._buffers[key].data_ptr()
        for lengths in ([400], [1] * 39 + [361], [11] * 36, [17] * 23, [33] * 12, [5] * 30 + [7] * 30, [2] * 20 + [40] * 9):
            handles = [runner.cache.open(i) for i in range(len(lengths))]
            runner.step([StepEntry(h, [3] * n, [n - 1]) for h, n in zip(handles, lengths)])
            runner.raise_on_device_error()
            assert model.runtime._buffers[key].data_ptr() == held
            for handle in handles:
                runner.cache.close(handle)
    finally:
        unregister_architecture(example.NAME)
