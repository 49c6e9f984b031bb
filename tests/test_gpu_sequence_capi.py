"""The sequence operators called straight through the C ABI (ctypes, device pointers, the current
stream), as a program that manages its own memory calls them, against their 64-bit definitions."""

import ctypes

import pytest
import torch

from sequence_helpers import assert_within, linear_reference, norm_reference, recurrence_reference
from torch_convnd import _build, _capi, load_native

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    load_native()
    return _build.hip_library()


def ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def scratch(size):
    return torch.empty(max(size, 8), dtype=torch.uint8, device="cuda").fill_(0xFF)


def ok(lib, status):
    assert status == _capi.SUCCESS, lib.convnd_hip_last_error().decode()


def randn(*shape, dtype=torch.float32, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_layer_norm(lib, dtype):
    rows, c, eps, code = 37, 70, 1e-5, _capi.dtype_code(dtype)
    wide = randn(rows, 90, dtype=dtype)
    x, dy, w, b = wide[:, 11:81], randn(rows, c, dtype=dtype, seed=1), randn(c, seed=2), randn(c, seed=3)
    y, dx = torch.empty(rows, c, dtype=dtype, device="cuda"), torch.empty(rows, c, dtype=dtype, device="cuda")
    mean, rstd, dw, db = (torch.empty(n, device="cuda") for n in (rows, rows, c, c))
    ok(lib, lib.convnd_hip_layer_norm(code, _capi.FLOAT32, ptr(x), 90, ptr(w), ptr(b), ptr(y), ptr(mean), ptr(rstd),
                                      rows, c, eps, stream()))
    size = lib.convnd_hip_layer_norm_backward_workspace_size(code, rows, c)
    ws = scratch(size)
    ok(lib, lib.convnd_hip_layer_norm_backward(code, _capi.FLOAT32, ptr(dy), c, ptr(x), 90, ptr(w), ptr(mean),
                                               ptr(rstd), ptr(dx), ptr(dw), ptr(db), rows, c, ptr(ws), size, stream()))
    ref = norm_reference(x, w, b, eps, dy)
    for name, got in (("y", y), ("dx", dx), ("dw", dw), ("db", db)):
        assert_within(got, *ref[name], name)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("m", [9, 130])
def test_linear(lib, m, dtype):
    k, n, code = 75, 50, _capi.dtype_code(dtype)
    x, w, b, r = randn(m, k, dtype=dtype), randn(n, k, dtype=dtype, seed=1) / 8, randn(n, dtype=dtype, seed=2), None
    dy = randn(m, n, dtype=dtype, seed=3)
    y, dx, dw, db = (torch.empty(s, dtype=dtype, device="cuda") for s in ((m, n), (m, k), (n, k), (n,)))
    slope = torch.empty(m, n, dtype=torch.float32 if dtype == torch.float32 else torch.int16, device="cuda")
    p = _capi.LinearProblem(rows=m, inputs=k, outputs=n, input_stride=k, residual_stride=0, grad_stride=n, activation=2)
    at = ctypes.byref(p)
    size = lib.convnd_hip_linear_workspace_size(code, at, ptr(x), ptr(w))
    ws = scratch(size)
    ok(lib, lib.convnd_hip_linear(code, at, ptr(x), ptr(w), ptr(b), ptr(r), ptr(y), ptr(slope), ptr(ws), size, stream()))
    size = lib.convnd_hip_linear_backward_workspace_size(code, at, ptr(dy), ptr(x), ptr(w), 1, 1, 1)
    ws = scratch(size)
    ok(lib, lib.convnd_hip_linear_backward(code, at, ptr(dy), ptr(x), ptr(w), ptr(slope), ptr(dx), ptr(dw), ptr(db),
                                           ptr(ws), size, stream()))
    ref = linear_reference(x, w, b, r, "gelu", dy)
    for name, got in (("y", y), ("dx", dx), ("dw", dw), ("db", db)):
        assert_within(got, *ref[name], name)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens", [1, 90, 2100])
@pytest.mark.parametrize("wide", [0, 1])
def test_recurrence(lib, tokens, wide, dtype):
    batch, c, code = 3, 34, _capi.dtype_code(dtype)
    x, gate, dy = (randn(batch, tokens, c, dtype=dtype, seed=s) for s in (0, 1, 2))
    first, dlast = randn(batch, c, seed=3), randn(batch, c, seed=4)
    lengths = torch.tensor([tokens, 0, tokens // 2], dtype=torch.int64 if wide else torch.int32, device="cuda")
    y, dx, dg = (torch.empty_like(x) for _ in range(3))
    last, df = torch.empty_like(first), torch.empty_like(first)
    carries = torch.empty(batch, lib.convnd_hip_recurrence_carries(tokens), c, device="cuda")
    p = _capi.RecurrenceProblem(batch=batch, tokens=tokens, channels=c, input_batch=tokens * c, input_token=c,
                                gate_batch=tokens * c, gate_token=c, wide_lengths=wide)
    at = ctypes.byref(p)
    size = lib.convnd_hip_recurrence_workspace_size(code, at)
    ws = scratch(size)
    ok(lib, lib.convnd_hip_recurrence(code, at, ptr(x), ptr(gate), ptr(first), ptr(lengths), ptr(y), ptr(last),
                                      ptr(carries), ptr(ws), size, stream()))
    ok(lib, lib.convnd_hip_recurrence_backward(code, at, ptr(dy), ptr(dlast), ptr(x), ptr(gate), ptr(lengths),
                                               ptr(carries), ptr(dx), ptr(dg), ptr(df), ptr(ws), size, stream()))
    ref = recurrence_reference(x, gate, first, lengths, dy, dlast)
    for name, got in (("h", y), ("last", last), ("dx", dx), ("dgate", dg), ("dfirst", df)):
        assert_within(got, *ref[name], name)
