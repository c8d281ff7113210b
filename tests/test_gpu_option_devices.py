"""Launches go to the current device: tensors that live on another one are refused, not handed to it."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_tensors_of_another_device(monkeypatch):
    from from_scratch_inference_engine_b200.kernels import ops
    ints = lambda *shape: torch.zeros(shape, dtype=torch.int32, device="cuda")
    pages, q = torch.zeros(2, 2, 1, 16, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(1, 64, dtype=torch.bfloat16, device="cuda")
    runs = torch.tensor([[0, 1, 0, 1, 0, -1]], dtype=torch.int32, device="cuda")
    room = torch.zeros(ops.shared_attention_room(1, 1, 0, 1, 1, 64, torch.bfloat16), dtype=torch.uint8, device="cuda")
    error, logits = ints(1), torch.zeros(1, 32, device="cuda")
    calls = [lambda: ops.shared_attention(q, 64, pages[:, 0], pages[:, 1], pages.stride(0), 16, ints(1, 2), ints(1), ints(1), runs, ints(1),
                                          q.clone(), 1, 1, 64, 1.0, room, error),
             lambda: ops.count_tokens(ints(1), ints(1), ints(1, 32), ints(1, 1), error),
             lambda: ops.adjust_logits(logits, error, None, None, None, None, None, (ints(1), ints(1, 1)))]
    for call in calls:
        call()
    # as it looks from a thread whose current device is the second one
    monkeypatch.setattr(ops, "_device", lambda: torch.cuda.current_device() + 1)
    for call in calls:
        with pytest.raises(ops.KernelError, match="current device"):
            call()
    assert not error.item()
