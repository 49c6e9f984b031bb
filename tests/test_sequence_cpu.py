"""The sequence operators and modules without a GPU: the PyTorch path against 64-bit definitions, its
refusals, shapes of the operators' fake kernels, the C ABI's checks, and the block fed whole, in
parts and token by token."""

import ctypes
import subprocess
import sys
from pathlib import Path

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import torch_convnd
from sequence_helpers import assert_within, linear_reference, norm_reference, recurrence_reference
from torch_convnd import _capi, gated_recurrence, layer_norm, linear_act
from torch_convnd._toolchain import HIP_LIBRARY

ROOT = Path(__file__).resolve().parent.parent


def randn(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layer_norm(dtype):
    x, w, b, dy = (randn(*s, seed=i, dtype=dtype) for i, s in enumerate([(5, 40), (40,), (40,), (5, 40)]))
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = layer_norm(*leaves, 1e-5)
    ref = norm_reference(x, w, b, 1e-5, dy)
    assert_within(y, *ref["y"], "y")
    for name, got in zip(("dx", "dw", "db"), torch.autograd.grad(y, leaves, dy)):
        assert_within(got, *ref[name], name)


@pytest.mark.parametrize("kind", [None, "relu", "gelu", "gelu_tanh"])
def test_linear_act(kind):
    x, w, b, r, dy = (randn(*s, seed=i) for i, s in enumerate([(6, 20), (9, 20), (9,), (6, 9), (6, 9)]))
    leaves = [t.requires_grad_() for t in (x, w, b, r)]
    y = linear_act(*leaves, activation=kind)
    ref = linear_reference(x, w, b, r, kind, dy)
    assert_within(y, *ref["y"], "y")
    grads = torch.autograd.grad(y, leaves, dy)
    for name, got in zip(("dx", "dw", "db"), grads):
        assert_within(got, *ref[name], name)
    assert torch.equal(grads[3], dy)


@pytest.mark.parametrize("ragged", [False, True])
def test_gated_recurrence(ragged):
    x, gate, first, dy, dlast = (
        randn(*s, seed=i) for i, s in enumerate([(4, 30, 5), (4, 30, 5), (4, 5), (4, 30, 5), (4, 5)])
    )
    gate[:, 11] = -float("inf")
    lengths = torch.tensor([30, 0, 7, 99]) if ragged else None
    if ragged:
        x[1], gate[2, 7:] = float("nan"), float("nan")
    leaves = [t.requires_grad_() for t in (x, gate, first)]
    h, last = gated_recurrence(*leaves, lengths=lengths)
    ref = recurrence_reference(x, gate, first, lengths, dy, dlast)
    assert_within(h, *ref["h"], "h")
    assert_within(last, *ref["last"], "last")
    grads = torch.autograd.grad((h, last), leaves, (dy, dlast))
    for name, got in zip(("dx", "dgate", "dfirst"), grads):
        assert_within(got, *ref[name], name)


def test_float64_and_second_derivatives():
    x, w, b = (randn(*s, seed=i).double().requires_grad_() for i, s in enumerate([(3, 4), (2, 4), (2,)]))
    assert torch.autograd.gradcheck(lambda *a: linear_act(*a, activation="gelu"), (x, w, b))
    assert torch.autograd.gradgradcheck(lambda *a: linear_act(*a, activation="gelu"), (x, w, b))
    n, p = randn(3, 5).double().requires_grad_(), randn(5, seed=1).double().requires_grad_()
    assert torch.autograd.gradcheck(lambda *a: layer_norm(*a), (n, p))
    s, g = (randn(2, 4, 3, seed=i).double().requires_grad_() for i in range(2))
    h = randn(2, 3, seed=2).double().requires_grad_()
    assert torch.autograd.gradcheck(lambda *a: gated_recurrence(*a), (s, g, h))


def test_refusals():
    x = randn(2, 6, 8)
    with pytest.raises(ValueError, match="Invalid backend"):
        layer_norm(x, backend="cuda")
    for call in (lambda: layer_norm(x, backend="native"), lambda: linear_act(x, randn(3, 8), backend="native"),
                 lambda: gated_recurrence(x, x, backend="native")):
        with pytest.raises(RuntimeError, match="runs on ROCm GPUs"):
            call()
    with pytest.raises(RuntimeError, match="weight must match the input's channels"):
        layer_norm(x, randn(7))
    with pytest.raises(RuntimeError, match="same dtype"):
        layer_norm(x.bfloat16(), randn(8), randn(8).bfloat16())
    with pytest.raises(RuntimeError, match=r"weight of \[outputs, inputs\]"):
        linear_act(x, randn(3, 7))
    with pytest.raises(RuntimeError, match="bias must match"):
        linear_act(x, randn(3, 8), randn(4))
    with pytest.raises(RuntimeError, match="residual must match"):
        linear_act(x, randn(3, 8), None, randn(2, 6, 4))
    with pytest.raises(ValueError, match="Invalid activation"):
        linear_act(x, randn(3, 8), activation="tanh")
    with pytest.raises(RuntimeError, match="gate must match"):
        gated_recurrence(x, x[:, :2])
    with pytest.raises(RuntimeError, match=r"\[batch, tokens, channels\]"):
        gated_recurrence(x[0], x[0])
    with pytest.raises(RuntimeError, match="initial_state must be float32"):
        gated_recurrence(x, x, randn(2, 7))
    with pytest.raises(RuntimeError, match="lengths must be int32 or int64"):
        gated_recurrence(x, x, lengths=torch.ones(2))
    with pytest.raises(ValueError, match="positive"):
        torch_convnd.LayerNorm(0)
    with pytest.raises(ValueError, match="Invalid activation"):
        torch_convnd.LinearAct(3, 3, activation="swish")


def test_fake_kernels():
    ops = torch.ops.torch_convnd
    with FakeTensorMode():
        x = torch.empty(3, 70, 16, device="cuda", dtype=torch.bfloat16)
        w, m = x.new_empty(16), x.new_empty(24, 16)
        y, statistics = ops.layer_norm(x, w, None, 1e-5, True)
        assert y.shape == x.shape and statistics.shape == (2, 210) and statistics.dtype == torch.float32
        dx, dw, db = ops.layer_norm_backward(y, x, w, None, statistics, [True, True, True])
        assert dx.shape == x.shape and dw.shape == (16,) and db is None
        y, slope = ops.linear_act(x, m, None, None, "gelu", True)
        assert y.shape == slope.shape == (3, 70, 24) and slope.dtype == torch.int16
        dx, dw, db = ops.linear_act_backward(y, x, m, slope, "gelu", [True, False, True])
        assert dx.shape == x.shape and dw is None and db.shape == (24,)
        h, last, carries = ops.gated_recurrence(x, x, None, None, True)
        assert h.shape == x.shape and last.shape == (3, 16) and last.dtype == torch.float32
        assert carries.shape == (3, 2, 16)
        dx, dg, df = ops.gated_recurrence_backward(h, last, x, x, None, carries, True)
        assert dx.shape == dg.shape == x.shape and df.shape == (3, 16)


@pytest.fixture(scope="module")
def lib():
    if not HIP_LIBRARY.exists():
        pytest.skip("native libraries not built (python __graft_entry__.py)")
    return _capi.bind(ctypes.CDLL(str(HIP_LIBRARY)))


def expect(lib, status, code, text):
    assert status == code
    assert text in lib.convnd_hip_last_error().decode()


def test_c_abi_checks(lib):
    """Calls that are refused before any device work."""
    bf16, f32, f64, f16 = _capi.BFLOAT16, _capi.FLOAT32, _capi.FLOAT64, _capi.FLOAT16
    bad, small = _capi.INVALID_ARGUMENT, _capi.WORKSPACE_TOO_SMALL
    one = ctypes.c_void_p(16)

    def norm(dtype=bf16, params=bf16, x=one, rows=4, channels=8, stride=8, mean=None, rstd=None):
        return lib.convnd_hip_layer_norm(dtype, params, x, stride, None, None, one, mean, rstd, rows, channels, 1e-5, None)

    expect(lib, norm(dtype=f64), bad, "float16, bfloat16 and float32")
    expect(lib, norm(params=f16), bad, "input's dtype or float32")
    expect(lib, norm(channels=0), bad, "channels")
    expect(lib, norm(rows=-1), bad, "rows")
    expect(lib, norm(stride=-8), bad, "overflow")
    expect(lib, norm(rows=2**62, stride=2**10), bad, "overflow")
    expect(lib, norm(mean=one), bad, "both statistics")
    expect(lib, norm(x=None), bad, "must not be null")
    assert norm(rows=0) == _capi.SUCCESS
    size = lib.convnd_hip_layer_norm_backward_workspace_size(bf16, 100, 8)
    assert size > 0
    expect(lib, lib.convnd_hip_layer_norm_backward(bf16, bf16, one, 8, one, 8, None, one, one, one, one, None, 100, 8,
                                                   one, size - 1, None), small, str(size))

    def linear(dtype=bf16, x=one, workspace=None, size=0, **fields):
        p = _capi.LinearProblem(rows=100, inputs=64, outputs=32, input_stride=64, residual_stride=32, grad_stride=32)
        for name, value in fields.items():
            setattr(p, name, value)
        return p, lib.convnd_hip_linear(dtype, ctypes.byref(p), x, one, None, None, one, None, workspace, size, None)

    expect(lib, linear(dtype=f64)[1], bad, "float16, bfloat16 and float32")
    expect(lib, linear(rows=-1)[1], bad, "rows")
    expect(lib, linear(inputs=0)[1], bad, "inputs")
    expect(lib, linear(inputs=2**21, input_stride=2**21)[1], bad, "2^21")
    expect(lib, linear(input_stride=63)[1], bad, "apart")
    expect(lib, linear(activation=9)[1], bad, "activation")
    expect(lib, linear(rows=2**31)[1], bad, "rows")
    expect(lib, linear(x=None)[1], bad, "must not be null")
    assert linear(rows=0)[1] == _capi.SUCCESS
    p, _ = linear(rows=0)
    p.rows, p.inputs, p.input_stride = 100, 63, 63  # odd 16-bit rows: padded copies
    size = lib.convnd_hip_linear_workspace_size(bf16, ctypes.byref(p), one, one)
    assert size >= 132 * 64 * 2
    assert lib.convnd_hip_linear_workspace_size(f32, ctypes.byref(p), one, one) < size
    expect(lib, lib.convnd_hip_linear(bf16, ctypes.byref(p), one, one, None, None, one, None, None, 0, None),
           small, str(size))
    size = lib.convnd_hip_linear_backward_workspace_size(bf16, ctypes.byref(p), one, one, one, 1, 1, 1)
    expect(lib, lib.convnd_hip_linear_backward(bf16, ctypes.byref(p), one, one, one, None, one, one, one, one,
                                               size - 1, None), small, str(size))
    p.activation = 2
    expect(lib, lib.convnd_hip_linear_backward(bf16, ctypes.byref(p), one, one, one, None, one, one, one, one, size,
                                               None), bad, "slope must not be null")

    def recurrence(dtype=bf16, x=one, size=0, **fields):
        p = _capi.RecurrenceProblem(batch=1, tokens=5000, channels=8, input_batch=40000, input_token=8,
                                    gate_batch=40000, gate_token=8)
        for name, value in fields.items():
            setattr(p, name, value)
        return lib.convnd_hip_recurrence(dtype, ctypes.byref(p), x, one, None, None, one, one, None, None, size, None)

    expect(lib, recurrence(dtype=f64), bad, "float16, bfloat16 and float32")
    expect(lib, recurrence(batch=-1), bad, "batch")
    expect(lib, recurrence(channels=0), bad, "channels")
    expect(lib, recurrence(input_token=7), bad, "apart")
    expect(lib, recurrence(gate_token=2**21), bad, "2^21")
    expect(lib, recurrence(x=None), bad, "must not be null")
    expect(lib, recurrence(), small, "workspace")
    assert recurrence(batch=0) == _capi.SUCCESS
    assert [lib.convnd_hip_recurrence_carries(n) for n in (-1, 0, 1, 64, 65)] == [0, 0, 1, 1, 2]


def block(**kw):
    torch.manual_seed(3)
    return torch_convnd.GatedConvBlock(12, kernel_size=3, expansion=2, dtype=torch.float64, **kw)


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
        torch.testing.assert_close(other, whole, rtol=1e-6, atol=1e-6)
        for a, b in zip(end, state):
            torch.testing.assert_close(a, b, rtol=1e-6, atol=1e-6)


def test_block_with_lengths():
    """Padded sequences give each one's own outputs and state."""
    model = block()
    x = randn(3, 8, 12).double()
    lengths = torch.tensor([8, 1, 5])
    padded, (window, hidden) = model(x, None, lengths)
    for i, n in enumerate(lengths.tolist()):
        alone, state = model(x[i : i + 1, :n])
        torch.testing.assert_close(padded[i : i + 1, :n], alone, rtol=1e-6, atol=1e-6)
        torch.testing.assert_close(window[i : i + 1], state[0], rtol=1e-6, atol=1e-6)
        torch.testing.assert_close(hidden[i : i + 1], state[1], rtol=1e-6, atol=1e-6)


def test_block_is_causal_and_refuses_other_shapes():
    model = block()
    x = randn(1, 6, 12).double()
    changed = x.clone()
    changed[:, 4:] += 1
    assert torch.equal(model(x)[0][:, :4], model(changed)[0][:, :4])
    with pytest.raises(ValueError, match="expected an input"):
        model(x[0])


def test_example_learns():
    command = [sys.executable, str(ROOT / "examples" / "byte_model.py"), "--steps", "41", "--channels", "32",
               "--blocks", "1", "--batch", "4", "--length", "48", "--write", "8"]
    result = subprocess.run(command, capture_output=True, text=True, timeout=300, env=None)
    assert result.returncode == 0, result.stderr
    losses = [float(line.split()[-1]) for line in result.stdout.splitlines() if line.startswith("step")]
    assert losses[-1] < losses[0] - 1, result.stdout


def test_c_abi_refuses_unaligned_workspaces(lib):
    bf16, bad = _capi.BFLOAT16, _capi.INVALID_ARGUMENT
    one, odd = ctypes.c_void_p(16), ctypes.c_void_p(20)
    size = lib.convnd_hip_layer_norm_backward_workspace_size(bf16, 100, 8)
    expect(lib, lib.convnd_hip_layer_norm_backward(bf16, bf16, one, 8, one, 8, None, one, one, one, one, None, 100, 8,
                                                   odd, size, None), bad, "aligned to 16 bytes")
    p = _capi.LinearProblem(rows=100, inputs=63, outputs=32, input_stride=63, residual_stride=32, grad_stride=32)
    at = ctypes.byref(p)
    size = lib.convnd_hip_linear_workspace_size(bf16, at, one, one)
    expect(lib, lib.convnd_hip_linear(bf16, at, one, one, None, None, one, None, odd, size, None), bad,
           "aligned to 16 bytes")
    size = lib.convnd_hip_linear_backward_workspace_size(bf16, at, one, one, one, 1, 1, 1)
    expect(lib, lib.convnd_hip_linear_backward(bf16, at, one, one, one, None, one, one, one, odd, size, None), bad,
           "aligned to 16 bytes")


def test_c_abi_refuses_overlapping_residual_rows(lib):
    one = ctypes.c_void_p(16)
    for stride in (31, 0, -32):
        p = _capi.LinearProblem(rows=4, inputs=64, outputs=32, input_stride=64, residual_stride=stride, grad_stride=32)
        expect(lib, lib.convnd_hip_linear(_capi.BFLOAT16, ctypes.byref(p), one, one, None, one, one, None, None, 0, None),
               _capi.INVALID_ARGUMENT, "apart")
