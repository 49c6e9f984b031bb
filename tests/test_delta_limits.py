"""Sizes of the delta rule that its kernels cannot address, refused by the C ABI before anything is launched."""

import ctypes

import pytest

from test_delta_cpu import BIG, ONE, expect, lib  # noqa: F401
from torch_convnd import _capi


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize(("tensor", "heads", "key_size", "value_size"), [
    ("value", 1 << 22, 8, 1), ("key", 1 << 19, 64, 8), ("query", 1 << 19, 64, 8)
])
def test_copies_past_32_bits(lib, tensor, heads, key_size, value_size, backward):  # noqa: F811
    """Broadcast heads, whose rows are copied with 16 bytes each at least: a token 2^26 bytes from the next."""
    key_heads = 1 if tensor == "value" else heads
    p = _capi.DeltaProblem.make(1, 20, key_heads, heads, key_size, value_size, _capi.BFLOAT16)
    for name in ("query", "key", "value", "grad"):
        for axis in ("batch", "token", "head"):
            setattr(p, f"{name}_{axis}", 0)
    q, k, v = (ctypes.c_void_p(18 if tensor == name else 16) for name in ("query", "key", "value"))
    run = lib.convnd_hip_delta
    args = (q, k, v, ONE, ONE, None, None, ONE, ONE, None)
    if backward:
        run = lib.convnd_hip_delta_backward
        args = (ONE, None, q, k, v, ONE, ONE, None, ONE, ONE, ONE, ONE, ONE, ONE, None)
    expect(lib, run(_capi.BFLOAT16, ctypes.byref(p), *args, ONE, BIG, None), _capi.INVALID_ARGUMENT, "2^25 bytes a token")
