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


# Batch and tokens of 1024 channels where one of the two forward kernels was at least 8 % faster.
FASTER = {
    ("whole", torch.bfloat16): [(6, 1024), (7, 1024), (8, 1024), (12, 1024), (16, 1024), (6, 1536), (7, 1536), (8, 1536)],
    ("whole", torch.float32): [(3, 1024), (4, 1024), (6, 1024), (8, 1024), (12, 1024), (15, 1024), (4, 2048), (6, 2048)],
    ("chain", torch.bfloat16): [(2, 1536), (2, 2048), (4, 2560), (6, 2560), (9, 1536), (10, 2048), (4, 4096), (7, 4096)],
    ("chain", torch.float32): [(2, 2048), (2, 4096), (3, 4096), (5, 4096)],
}


@pytest.mark.parametrize(("kernel", "dtype", "sizes"), [(*k, v) for k, v in FASTER.items()])
def test_forward_takes_the_faster_kernel(lib, kernel, dtype, sizes):
    for batch, tokens in sizes:
        assert _capi.recurrence_plan(lib, batch, tokens, 1024, dtype)["kernel"] == kernel, (batch, tokens)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_neighbouring_sizes_take_one_kernel(lib, dtype):
    """No single count of workgroups, tokens or channels has a rule of its own."""
    for batch, tokens in ((7, 1200), (8, 2048), (15, 1100), (4, 6000)):
        kernels = {
            _capi.recurrence_plan(lib, batch, t, c, dtype)["kernel"]
            for t in range(tokens - 3, tokens + 4)
            for c in (992, 1008, 1024)
        }
        assert len(kernels) == 1, (batch, tokens, kernels)
    for batch in range(1, 16):
        kernels = [_capi.recurrence_plan(lib, batch, t, 1024, dtype)["kernel"] for t in range(1024, 9000, 97)]
        assert kernels == sorted(kernels, reverse=True), batch  # whole sequences, from some length on chunks
