"""The sequence operators' plans as the C ABI describes them, on the host."""

import ctypes

import pytest
import torch

from torch_convnd import _capi
from torch_convnd._toolchain import HIP_LIBRARY


@pytest.fixture(scope="module")
def lib():
    if not HIP_LIBRARY.exists():
        pytest.skip("native libraries not built (python __graft_entry__.py)")
    return _capi.bind(ctypes.CDLL(str(HIP_LIBRARY)))


def test_descriptions(lib):
    assert _capi.linear_plan(lib, 4, 1024, 4096, torch.bfloat16) == {"kernel": "few_rows", "workgroups": 256}
    for which in (1, 2):
        plan = _capi.linear_plan(lib, 100, 64, 64, torch.float32, which)
        assert plan["kernel"] == "tiles" and plan["tile"] == 64 and plan["splits"] >= 1
    plan = _capi.linear_plan(lib, 8192, 1024, 4096, torch.bfloat16, 3)
    assert plan["kernel"] == "both_gradients" and plan["workgroups"] >= 1
    assert _capi.recurrence_plan(lib, 32, 1, 1024, torch.bfloat16)["kernel"] == "step"
    assert _capi.recurrence_plan(lib, 1, 65536, 512, torch.float32)["kernel"] == "chain"
    assert _capi.recurrence_plan(lib, 64, 512, 4096, torch.float32, True)["kernel"] == "whole"


def test_refusals(lib):
    with pytest.raises(RuntimeError, match="which must be 0 to 3"):
        _capi.linear_plan(lib, 4, 16, 16, torch.float32, 4)
    with pytest.raises(RuntimeError, match="rows positive"):
        _capi.linear_plan(lib, 0, 16, 16, torch.float32)
    with pytest.raises(RuntimeError, match="2\\^32 threads"):
        _capi.linear_plan(lib, (1 << 31) - 1, 16, 16, torch.float32)
    with pytest.raises(RuntimeError, match="supports float16, bfloat16 and float32"):
        _capi.recurrence_plan(lib, 1, 16, 16, torch.float64)
    buffer = ctypes.create_string_buffer(8)
    p = _capi.LinearProblem(rows=4, inputs=16, outputs=16, input_stride=16)
    assert lib.convnd_hip_linear_plan_describe(_capi.FLOAT32, ctypes.byref(p), 0, buffer, 8) == _capi.SUCCESS
    assert len(buffer.value) == 7  # truncated, with its end
