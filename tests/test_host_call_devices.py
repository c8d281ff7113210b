"""Which device tensors live on, asked without ctypes (no GPU needed)."""
import pytest
import torch

from from_scratch_inference_engine_b200.csrc import build


@pytest.mark.parametrize("calls", [build.host_call(), build._PlainCalls])
def test_which_device_tensors_live_on(calls):
    assert calls.on(-1, torch.zeros(2), None, torch.zeros(3)) is True              # (torch's number of the CPU)
    assert calls.on(0, None) is True and calls.on(0) is True
    assert calls.on(0, torch.zeros(2)) is False and calls.on(1, None, torch.zeros(2)) is False
    with pytest.raises(AttributeError):
        calls.on(0, 5)


def test_what_is_refused():
    calls = build.host_call()
    if calls is build._PlainCalls:
        pytest.skip("no headers of this Python")
    for wrong in ((), ("x",)):
        with pytest.raises(TypeError):
            calls.on(*wrong)
