"""Several tensors checked in one call without ctypes (no GPU needed)."""
import pytest
import torch

from from_scratch_inference_engine_b200.csrc import build


@pytest.mark.parametrize("calls", [build.host_call(), build._PlainCalls])
def test_tensors_that_fit(calls):
    floats, ints = torch.zeros(4, 6), torch.zeros(3, dtype=torch.int32)
    here = -1                                                                     # torch's number of the CPU
    assert calls.all_fit(here, None, False, floats, None, ints, floats[:, ::2]) is True
    assert calls.all_fit(here, torch.float32, True, floats, None, floats[1:]) is True
    assert calls.all_fit(0, torch.float32, True) is True and calls.all_fit(0, None, True, None) is True
    assert calls.all_fit(here, torch.float32, True, floats, floats[:, ::2]) is False
    assert calls.all_fit(here, torch.float32, False, floats, ints) is False
    assert calls.all_fit(0, None, False, floats) is False and calls.all_fit(1, torch.int32, True, None, ints) is False
    with pytest.raises(AttributeError):
        calls.all_fit(here, None, False, floats, 5)


def test_what_is_refused():
    calls = build.host_call()
    if calls is build._PlainCalls:
        pytest.skip("no headers of this Python")
    for wrong in ((), (0, None), ("x", None, False)):
        with pytest.raises(TypeError):
            calls.all_fit(*wrong)
