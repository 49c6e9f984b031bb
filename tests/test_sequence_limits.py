"""Sizes of the sequence operators past what one launch can hold: refused with the reason before any
device work."""

import ctypes

import pytest

from torch_convnd import _capi
from torch_convnd._toolchain import HIP_LIBRARY

ONE = ctypes.c_void_p(16)
BIG = 1 << 62  # a workspace that is never too small
TOO_MANY = "2^32 threads"


@pytest.fixture(scope="module")
def lib():
    if not HIP_LIBRARY.exists():
        pytest.skip("native libraries not built (python __graft_entry__.py)")
    return _capi.bind(ctypes.CDLL(str(HIP_LIBRARY)))


def refused(lib, status, text):
    assert status == _capi.INVALID_ARGUMENT, lib.convnd_hip_last_error()
    assert text in lib.convnd_hip_last_error().decode()


@pytest.mark.parametrize("dtype", [_capi.BFLOAT16, _capi.FLOAT32])
def test_linear(lib, dtype):
    rows = (1 << 31) - 1
    p = _capi.LinearProblem(rows=rows, inputs=16, outputs=16, input_stride=16, residual_stride=16, grad_stride=16)
    at = ctypes.byref(p)
    refused(lib, lib.convnd_hip_linear(dtype, at, ONE, ONE, None, None, ONE, None, ONE, BIG, None), TOO_MANY)
    for grads in ((ONE, ONE, ONE), (ONE, None, None)):
        refused(lib, lib.convnd_hip_linear_backward(dtype, at, ONE, ONE, ONE, None, *grads, ONE, BIG, None), TOO_MANY)


@pytest.mark.parametrize("dtype", [_capi.BFLOAT16, _capi.FLOAT32])
@pytest.mark.parametrize(
    ("backward", "batch", "tokens", "channels"),
    [(0, 1 << 23, 9, 16), (0, 1 << 28, 1, 16), (1, 1 << 23, 9, 16), (1, 1 << 26, 8, 16)],
)
def test_recurrence(lib, dtype, backward, batch, tokens, channels):
    p = _capi.RecurrenceProblem(batch=batch, tokens=tokens, channels=channels, input_batch=tokens * channels,
                                input_token=channels, gate_batch=tokens * channels, gate_token=channels)
    at = ctypes.byref(p)
    if backward:
        status = lib.convnd_hip_recurrence_backward(dtype, at, ONE, None, ONE, ONE, None, ONE, ONE, ONE, None, ONE, BIG, None)
    else:
        status = lib.convnd_hip_recurrence(dtype, at, ONE, ONE, None, None, ONE, ONE, None, ONE, BIG, None)
    refused(lib, status, TOO_MANY)


def test_layer_norm_parameters(lib):
    channels = 1 << 27
    refused(lib, lib.convnd_hip_layer_norm_backward(_capi.BFLOAT16, _capi.BFLOAT16, ONE, channels, ONE, channels, None,
                                                    ONE, ONE, ONE, ONE, None, 2, channels, ONE, BIG, None), "2^27 channels")
