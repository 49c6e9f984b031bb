"""The delta rule, the gated linear layer and their block without a GPU: the PyTorch path against 64-bit
definitions, refusals, shapes of the operators' fake kernels, the C ABI's checks and plans, and the block fed whole,
in parts and token by token."""

import ctypes
import subprocess
import sys
from pathlib import Path

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import torch_convnd
from delta_helpers import assert_rows, delta_reference, make_delta
from gated_linear_helpers import gated_reference
from sequence_helpers import assert_within
from torch_convnd import _capi, gated_delta_rule, gated_linear
from torch_convnd._toolchain import HIP_LIBRARY

ROOT = Path(__file__).resolve().parent.parent
ONE = ctypes.c_void_p(16)
BIG = 1 << 62  # a workspace that is never too small


def randn(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("normalize", [False, True])
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("tokens", [0, 1, 37])
def test_delta_rule(tokens, ragged, normalize):
    data = make_delta(4, tokens, 2, 4, 8, 6, torch.float32)
    *inputs, first, dy, dlast = data
    lengths = None
    if ragged:
        lengths = torch.tensor([tokens, 0, 7, 99])
        for t in (*inputs, dy):
            t[1] = float("nan")
    if tokens > 9:
        inputs[3][:, 9] = -float("inf")
        inputs[3][:, 11] = -150.0
    leaves = [t.requires_grad_() for t in (*inputs, first)]
    o, last = gated_delta_rule(*leaves, lengths=lengths, normalize=normalize)
    ref = delta_reference(*inputs, first, lengths, None, normalize, dy, dlast)
    grads = torch.autograd.grad((o, last), leaves, (dy, dlast), allow_unused=True)
    names = ("o", "last", "dq", "dk", "dv", "ddecay", "dbeta", "dfirst")
    for name, got in zip(names, (o, last, *grads)):
        if got is not None:  # without tokens
            assert_rows(name, got, ref, torch.float32, (8, 6))


def test_delta_rule_of_other_types():
    data = make_delta(2, 20, 1, 2, 8, 6, torch.bfloat16)
    o, last = gated_delta_rule(*data[:6], scale=0.5)
    ref = delta_reference(*data[:6], scale=0.5)
    assert o.dtype == torch.bfloat16 and last.dtype == torch.float32
    assert_rows("o", o, ref, torch.bfloat16, (8, 6))
    assert_rows("last", last, ref, torch.float32, (8, 6))
    wide = [t.double().requires_grad_() for t in make_delta(1, 5, 1, 2, 3, 2, torch.float32)[:6]]
    assert torch.autograd.gradcheck(lambda *a: gated_delta_rule(*a, normalize=True), wide)
    assert torch.autograd.gradgradcheck(lambda *a: gated_delta_rule(*a)[0], wide)


@pytest.mark.parametrize("kind", ["silu", "relu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gated_linear(kind, dtype):
    x, w, b = (randn(*s, seed=i, dtype=dtype) for i, s in enumerate([(6, 20), (18, 20), (18,)]))
    y = gated_linear(x, w, b, activation=kind)
    assert y.dtype == dtype and y.shape == (6, 9)
    assert_within(y, *gated_reference(x, w, b, kind)["y"], "y")
    if dtype == torch.float32:
        dy = randn(6, 9, seed=5)
        leaves = [t.requires_grad_() for t in (x, w, b)]
        ref = gated_reference(x, w, b, kind, dy)
        grads = torch.autograd.grad(gated_linear(*leaves, activation=kind), leaves, dy)
        for name, got in zip(("dx", "dw", "db"), grads):
            assert_within(got, *ref[name], name)


def test_refusals():
    q, k, v, decay, beta, first, _, _ = make_delta(2, 6, 2, 4, 16, 8, torch.bfloat16)

    def refused(match, call, *inputs, kind=RuntimeError, **options):
        with pytest.raises(kind, match=match):
            call(*inputs, **options)

    rule = gated_delta_rule
    refused("Invalid backend", rule, q, k, v, decay, beta, kind=ValueError, backend="cuda")
    refused("runs on ROCm GPUs", rule, q, k, v, decay, beta, backend="native")
    refused(r"query and key of \[batch", rule, q[0], k[0], v, decay, beta)
    refused(r"query and key of \[batch", rule, q, k[..., :8], v, decay, beta)
    refused("a value of", rule, q, k, v[:, :, :3], decay[..., :3], beta[..., :3])
    refused("decay and beta of", rule, q, k, v, decay[..., :2], beta)
    refused("same device and dtype", rule, q, k.half(), v, decay, beta)
    refused("both of their dtype or float32", rule, q, k, v, decay, beta.bfloat16())
    refused("initial_state must be float32", rule, q, k, v, decay, beta, first.bfloat16())
    refused("lengths must be int32 or int64", rule, q, k, v, decay, beta, lengths=torch.ones(2))
    x, w, b = randn(6, 16), randn(16, 16), randn(16)
    refused("Invalid activation", gated_linear, x, w, kind=ValueError, activation="tanh")
    refused("runs on ROCm GPUs", gated_linear, x, w, backend="native")
    refused("expects an input", gated_linear, x, w[:15])
    refused("bias must match", gated_linear, x, w, b[:8])
    refused("same device and dtype", gated_linear, x, w.half())
    refused("positive", torch_convnd.GatedLinear, 0, 3, kind=ValueError)
    refused("Invalid activation", torch_convnd.GatedLinear, 3, 3, activation="tanh", kind=ValueError)
    refused("multiple of heads", torch_convnd.GatedDeltaBlock, 12, 5, kind=ValueError)


def test_fake_kernels():
    ops = torch.ops.torch_convnd
    with FakeTensorMode():
        q = torch.empty(3, 70, 2, 16, device="cuda", dtype=torch.bfloat16)
        v, gate = q.new_empty(3, 70, 4, 20), q.new_empty(3, 70, 4, dtype=torch.float32)
        o, last, saved = ops.gated_delta_rule(q, q, v, gate, gate, None, None, 1.0, True, True)
        assert o.shape == v.shape and last.shape == (3, 4, 16, 20) and last.dtype == torch.float32
        assert saved.shape == (3 * 4 * 2 * (32 * 128 + (4 * 64 * 128 + 36 * 64 + 32) // 2),) and saved.dtype == torch.bfloat16
        assert ops.gated_delta_rule(q, q, v, gate, gate, None, None, 1.0, True, False)[2].numel() == 0
        grads = ops.gated_delta_rule_backward(o, last, q, q, v, gate, gate, None, saved, 1.0, True, True)
        for got, t in zip(grads, (q, q, v, gate, gate, last)):
            assert got.shape == t.shape and got.dtype == t.dtype
        x, w = torch.empty(3, 70, 16, device="cuda", dtype=torch.bfloat16), q.new_empty(24, 16)
        y, kept = ops.gated_linear(x, w, None, "silu", True)
        assert y.shape == (3, 70, 12) and kept.shape == (3 * 70 * 24 * 3,) and kept.dtype == torch.uint8
        dx, dw, db = ops.gated_linear_backward(y, x, w, kept, "silu", [True, False, True])
        assert dx.shape == x.shape and dw is None and db.shape == (24,)


@pytest.fixture(scope="module")
def lib():
    if not HIP_LIBRARY.exists():
        pytest.skip("native libraries not built (python __graft_entry__.py)")
    return _capi.bind(ctypes.CDLL(str(HIP_LIBRARY)))


def expect(lib, status, code, text):
    assert status == code, lib.convnd_hip_last_error()
    assert text in lib.convnd_hip_last_error().decode()


def test_saved_sizes_are_the_fake_kernels(lib):
    """What the forward keeps is allocated by the shapes traced and by the library alike."""
    from torch_convnd._autograd import delta_saved

    for dtype, code in ((torch.bfloat16, _capi.BFLOAT16), (torch.float32, _capi.FLOAT32)):
        for tokens, key_size, value_size in ((1, 1, 1), (64, 64, 64), (65, 65, 100), (500, 128, 257)):
            q, v = (torch.empty(2, tokens, n, s, dtype=dtype, device="meta") for n, s in ((2, key_size), (6, value_size)))
            p = _capi.DeltaProblem.make(2, tokens, 2, 6, key_size, value_size, code)
            assert lib.convnd_hip_delta_saved(code, ctypes.byref(p)) == delta_saved(q, v)


def test_c_abi_checks(lib):
    bf16, f32, f64 = _capi.BFLOAT16, _capi.FLOAT32, _capi.FLOAT64
    bad, small = _capi.INVALID_ARGUMENT, _capi.WORKSPACE_TOO_SMALL

    def delta(dtype=bf16, query=ONE, last=ONE, saved=None, workspace=ONE, size=BIG, backward=False, **fields):
        p = _capi.DeltaProblem.make(2, 100, 2, 4, 64, 64, f32)
        for name, value in fields.items():
            setattr(p, name, value)
        p = ctypes.byref(p)
        if backward:
            return lib.convnd_hip_delta_backward(dtype, p, ONE, None, query, ONE, ONE, ONE, ONE, None, saved, ONE, ONE,
                                                 ONE, ONE, ONE, None, workspace, size, None)
        return lib.convnd_hip_delta(dtype, p, query, ONE, ONE, ONE, ONE, None, None, ONE, last, saved, workspace, size,
                                    None)

    for backward in (False, True):
        expect(lib, delta(dtype=f64, backward=backward), bad, "float16, bfloat16 and float32")
        expect(lib, delta(batch=-1, backward=backward), bad, "batch")
        expect(lib, delta(heads=3, backward=backward), bad, "multiple")
        expect(lib, delta(key_heads=0, backward=backward), bad, "multiple")
        expect(lib, delta(key_size=129, backward=backward), bad, "1 to 128")
        expect(lib, delta(value_size=0, backward=backward), bad, "1 to 65535")
        expect(lib, delta(gate_dtype=f64, backward=backward), bad, "inputs' dtype or float32")
        expect(lib, delta(query_token=1 << 21, backward=backward), bad, "2^21")
        expect(lib, delta(key_head=-1, backward=backward), bad, "overflow")
        expect(lib, delta(value_batch=1 << 62, backward=backward), bad, "overflow")
        expect(lib, delta(tokens=1 << 31, backward=backward), bad, "2^31")
        expect(lib, delta(heads=1 << 17, key_heads=1, backward=backward), bad, "2^23 values")
        expect(lib, delta(batch=1 << 24, backward=backward, saved=ONE), bad, "2^32 threads")
        expect(lib, delta(query=None, backward=backward), bad, "must not be null")
        assert delta(batch=0, backward=backward) == _capi.SUCCESS
    expect(lib, delta(last=None), bad, "must not be null")
    expect(lib, delta(backward=True), bad, "must not be null")  # saved
    expect(lib, delta(workspace=ctypes.c_void_p(20)), bad, "aligned to 16 bytes")
    expect(lib, delta(saved=ctypes.c_void_p(20)), bad, "saved must be aligned")
    expect(lib, delta(saved=ctypes.c_void_p(20), backward=True), bad, "saved must be aligned")
    p = ctypes.byref(_capi.DeltaProblem.make(2, 100, 2, 4, 64, 64, f32))
    size = lib.convnd_hip_delta_workspace_size(bf16, p, ONE, ONE, ONE, 0)
    assert size > 0
    expect(lib, delta(size=size - 1), small, str(size))
    # Rows that do not start on 4 bytes are copied.
    assert lib.convnd_hip_delta_workspace_size(bf16, p, ctypes.c_void_p(18), ONE, ONE, 0) > size
    back = lib.convnd_hip_delta_backward_workspace_size(bf16, p, ONE, ONE, ONE, ONE)
    assert back > lib.convnd_hip_delta_workspace_size(bf16, p, ONE, ONE, ONE, 1)
    expect(lib, delta(backward=True, saved=ONE, size=back - 1), small, str(back))
    p = ctypes.byref(_capi.DeltaProblem.make(2, 3, 2, 4, 64, 64, f32))
    assert lib.convnd_hip_delta_workspace_size(bf16, p, ONE, ONE, ONE, 0) == 0

    def gated(dtype=bf16, x=ONE, workspace=ONE, size=BIG, **fields):
        q = _capi.LinearProblem(rows=100, inputs=64, outputs=32, input_stride=64, grad_stride=32, activation=4)
        for name, value in fields.items():
            setattr(q, name, value)
        return lib.convnd_hip_gated_linear(dtype, ctypes.byref(q), x, ONE, None, ONE, None, workspace, size, None)

    expect(lib, gated(dtype=f64), bad, "float16, bfloat16 and float32")
    expect(lib, gated(outputs=0), bad, "outputs")
    expect(lib, gated(outputs=1 << 20), bad, "2^20")
    expect(lib, gated(activation=0), bad, "'silu'")
    expect(lib, gated(activation=5), bad, "'silu'")
    expect(lib, gated(rows=-1), bad, "rows")
    expect(lib, gated(input_stride=63), bad, "apart")
    expect(lib, gated(x=None), bad, "must not be null")
    assert gated(rows=0) == _capi.SUCCESS
    q = _capi.LinearProblem(rows=100, inputs=63, outputs=32, input_stride=63, grad_stride=32, activation=4)
    at = ctypes.byref(q)
    size = lib.convnd_hip_gated_linear_workspace_size(bf16, at, ONE, ONE)
    expect(lib, gated(inputs=63, input_stride=63, size=size - 1), small, str(size))
    assert lib.convnd_hip_gated_linear_kept_size(bf16, at) == 100 * 64 * 3
    assert lib.convnd_hip_gated_linear_kept_size(f32, at) == 100 * 64 * 4
    size = lib.convnd_hip_gated_linear_backward_workspace_size(bf16, at, ONE, ONE, 1, 1, 1)
    call = lib.convnd_hip_gated_linear_backward
    expect(lib, call(bf16, at, ONE, ONE, ONE, ONE, ONE, ONE, ONE, ONE, size - 1, None), small, str(size))
    expect(lib, call(bf16, at, ONE, ONE, ONE, None, ONE, ONE, ONE, ONE, size, None), bad, "kept must not be null")
    q.grad_stride = 31
    expect(lib, call(bf16, at, ONE, ONE, ONE, ONE, ONE, ONE, ONE, ONE, size, None), bad, "apart")
    # The linear layer has no silu.
    q = _capi.LinearProblem(rows=4, inputs=64, outputs=32, input_stride=64, residual_stride=32, grad_stride=32, activation=4)
    expect(lib, lib.convnd_hip_linear(bf16, ctypes.byref(q), ONE, ONE, None, None, ONE, None, None, 0, None), bad,
           "activation must be")


def test_plans(lib):
    plan = lambda *sizes, **kw: _capi.delta_plan(lib, *sizes, torch.bfloat16, **kw)  # noqa: E731
    assert plan(32, 1, 8, 8, 128, 128)["kernel"] == "step"
    assert plan(32, 1, 8, 8, 128, 128, saving=True)["kernel"] == "chunks"
    assert plan(8, 2048, 8, 8, 128, 128)["segments"] == 1
    long = plan(1, 32768, 8, 8, 128, 128)
    assert long["segments"] == 16 and long["segment_chunks"] == 32
    assert plan(1, 2047, 8, 8, 128, 128)["segments"] == 4 and plan(1, 1984, 8, 8, 128, 128)["segments"] == 1
    assert plan(1, 4095, 32, 32, 128, 128)["segments"] == 4 and plan(1, 4032, 32, 32, 128, 128)["segments"] == 1
    for tokens in (1000, 1024, 5000, 65536):
        got = plan(1, tokens, 1, 1, 64, 64)
        chunks = (tokens + 63) // 64
        assert got["segments"] * got["segment_chunks"] >= chunks > (got["segments"] - 1) * got["segment_chunks"]


def block(**kw):
    torch.manual_seed(3)
    return torch_convnd.GatedDeltaBlock(12, 3, kernel_size=3, hidden=20, dtype=torch.float64, **kw)


def test_block_in_parts_and_steps():
    """A prompt at once, in two parts and token by token gives the same outputs and state."""
    model = block()
    x = randn(2, 9, 12).double()
    whole, state = model(x)
    first, middle = model(x[:, :5])
    second, parts = model(x[:, 5:], middle)
    steps, running = [], None
    for t in range(9):
        y, running = model(x[:, t : t + 1], running)
        steps.append(y)
    for other, end in ((torch.cat((first, second), 1), parts), (torch.cat(steps, 1), running)):
        torch.testing.assert_close(other, whole, rtol=1e-9, atol=1e-9)
        for a, b in zip(end, state):
            torch.testing.assert_close(a, b, rtol=1e-9, atol=1e-9)


def test_block_with_lengths():
    """Padded sequences give each one's own outputs and state."""
    model = block()
    x = randn(3, 8, 12).double()
    lengths = torch.tensor([8, 1, 5])
    padded, (window, hidden) = model(x, None, lengths)
    for i, n in enumerate(lengths.tolist()):
        alone, state = model(x[i : i + 1, :n])
        torch.testing.assert_close(padded[i : i + 1, :n], alone, rtol=1e-9, atol=1e-9)
        torch.testing.assert_close(window[i : i + 1], state[0], rtol=1e-9, atol=1e-9)
        torch.testing.assert_close(hidden[i : i + 1], state[1], rtol=1e-9, atol=1e-9)


def test_block_is_causal_and_refuses_other_shapes():
    model = block()
    x = randn(1, 6, 12).double()
    changed = x.clone()
    changed[:, 4:] += 1
    assert torch.equal(model(x)[0][:, :4], model(changed)[0][:, :4])
    with pytest.raises(ValueError, match="expected an input"):
        model(x[0])
    assert torch_convnd.GatedDeltaBlock(16, 2).gated.out_features == 48


def test_example_runs_with_heads():
    command = [sys.executable, str(ROOT / "examples" / "byte_model.py"), "--steps", "5", "--channels", "32",
               "--blocks", "1", "--batch", "2", "--length", "24", "--write", "4", "--heads", "2"]
    result = subprocess.run(command, capture_output=True, text=True, timeout=300)
    assert result.returncode == 0, result.stderr
    assert "bytes/s in writing" in result.stdout
