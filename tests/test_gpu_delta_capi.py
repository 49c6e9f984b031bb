"""The delta rule and the gated linear layer called straight through the C ABI (ctypes, device pointers, the current
stream, workspaces filled with NaN), as a program that manages its own memory calls them, against their 64-bit
definitions; and rows next to the results, which stay as they were."""

import ctypes

import pytest
import torch

from delta_helpers import assert_rows, delta_reference, make_delta
from gated_linear_helpers import gated_reference
from sequence_helpers import assert_within
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


class Fenced:
    """A tensor between two bands of ones that a call must leave alone."""

    def __init__(self, *shape, dtype):
        count = torch.Size(shape).numel()
        self.whole = torch.ones(count + 512, dtype=dtype, device="cuda")
        self.part = self.whole[256 : 256 + count].view(shape)
        self.part.fill_(float("nan"))

    def intact(self):
        return bool((self.whole[:256] == 1).all() and (self.whole[-256:] == 1).all())


def ok(lib, status):
    assert status == _capi.SUCCESS, lib.convnd_hip_last_error().decode()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize(
    ("tokens", "key_size", "value_size"), [(1, 64, 64), (7, 33, 21), (90, 64, 64), (150, 128, 40), (77, 21, 97), (1100, 32, 48)]
)
@pytest.mark.parametrize("wide", [0, 1])
def test_delta(lib, wide, tokens, key_size, value_size, dtype):
    batch, key_heads, heads, code = 3, 1, 2, _capi.dtype_code(dtype)
    data = make_delta(batch, tokens, key_heads, heads, key_size, value_size, dtype, normalize=True)
    q, k, v, decay, beta, first, dy, dlast = (t.cuda() for t in data)
    lengths = torch.tensor([tokens, 0, tokens // 2], dtype=torch.int64 if wide else torch.int32, device="cuda")
    o, dq, dk, dv = (Fenced(*t.shape, dtype=dtype) for t in (v, q, k, v))
    last, df, dg, db = (Fenced(*t.shape, dtype=torch.float32) for t in (first, first, decay, beta))
    p = _capi.DeltaProblem.make(batch, tokens, key_heads, heads, key_size, value_size, _capi.FLOAT32)
    p.scale, p.normalize, p.wide_lengths = 0.3, 1, wide
    at = ctypes.byref(p)
    saved = Fenced(lib.convnd_hip_delta_saved(code, at), dtype=dtype)
    inputs = [ptr(t) for t in (q, k, v, decay, beta)]
    ref = delta_reference(q, k, v, decay, beta, first, lengths, 0.3, True, dy, dlast)
    sizes = (key_size, value_size)
    for keep in (0, 1):
        size = lib.convnd_hip_delta_workspace_size(code, at, *inputs[:3], keep)
        ws = scratch(size)
        o.part.fill_(float("nan")), last.part.fill_(float("nan"))
        ok(lib, lib.convnd_hip_delta(code, at, *inputs, ptr(first), ptr(lengths), ptr(o.part), ptr(last.part),
                                     ptr(saved.part) if keep else None, ptr(ws), size, stream()))
        for name, got in (("o", o), ("last", last)):
            assert got.intact()
            assert_rows(name, got.part, ref, dtype, sizes)
    size = lib.convnd_hip_delta_backward_workspace_size(code, at, ptr(dy), *inputs[:3])
    ws = scratch(size)
    ok(lib, lib.convnd_hip_delta_backward(code, at, ptr(dy), ptr(dlast), *inputs, ptr(lengths), ptr(saved.part),
                                          ptr(dq.part), ptr(dk.part), ptr(dv.part), ptr(dg.part), ptr(db.part),
                                          ptr(df.part), ptr(ws), size, stream()))
    assert saved.intact()
    for name, got in (("dq", dq), ("dk", dk), ("dv", dv), ("ddecay", dg), ("dbeta", db), ("dfirst", df)):
        assert got.intact(), name
        assert_rows(name, got.part, ref, dtype, sizes)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize(("m", "k", "n"), [(1, 70, 33), (9, 64, 40), (130, 75, 50), (700, 128, 96)])
def test_gated_linear(lib, m, k, n, dtype):
    code = _capi.dtype_code(dtype)
    g = torch.Generator().manual_seed(1)
    x, w, b, dy = ((torch.randn(s, generator=g) / d).to(dtype).cuda()
                   for s, d in (((m, k), 1), ((2 * n, k), 8), ((2 * n,), 1), ((m, n), 1)))
    p = _capi.LinearProblem(rows=m, inputs=k, outputs=n, input_stride=k, grad_stride=n, activation=4)
    at = ctypes.byref(p)
    y, dx, dw, db = (Fenced(*s, dtype=dtype) for s in ((m, n), (m, k), (2 * n, k), (2 * n,)))
    kept_size = lib.convnd_hip_gated_linear_kept_size(code, at)
    kept = scratch(kept_size + 256)
    ref = gated_reference(x, w, b, "silu", dy)
    size = lib.convnd_hip_gated_linear_workspace_size(code, at, ptr(x), ptr(w))
    ws = scratch(size)
    for factors in (None, ptr(kept)):
        y.part.fill_(float("nan"))
        ok(lib, lib.convnd_hip_gated_linear(code, at, ptr(x), ptr(w), ptr(b), ptr(y.part), factors, ptr(ws), size, stream()))
        assert y.intact()
        assert_within(y.part, *ref["y"], "y")
    assert (kept[kept_size:] == 0xFF).all()
    for wanted in ((1, 1, 1), (1, 0, 0), (0, 1, 0), (0, 0, 1)):
        grads = [t if take else None for t, take in zip((dx, dw, db), wanted)]
        size = lib.convnd_hip_gated_linear_backward_workspace_size(code, at, ptr(x), ptr(w), *wanted)
        ws = scratch(size)
        for t in (dx, dw, db):
            t.part.fill_(float("nan"))
        ok(lib, lib.convnd_hip_gated_linear_backward(code, at, ptr(dy), ptr(x), ptr(w), ptr(kept),
                                                     *(None if t is None else ptr(t.part) for t in grads), ptr(ws), size,
                                                     stream()))
        for name, got in zip(("dx", "dw", "db"), grads):
            if got is not None:
                assert got.intact()
                assert_within(got.part, *ref[name], name)
