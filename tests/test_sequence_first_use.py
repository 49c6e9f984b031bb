"""Gradients of the sequence operators where nothing has loaded the native library yet: a graph
compiled as a program's first use, and a direct call of an operator. Each test runs a process of its
own, since loading cannot be undone."""

import subprocess
import sys
from pathlib import Path

import pytest

PACKAGE_ROOT = Path(__file__).resolve().parent.parent / "torch-convnd_amd"

HEAD = f"""
import sys
sys.path.insert(0, {str(PACKAGE_ROOT)!r})
import torch
import torch_convnd
from torch_convnd import _build
ops = torch.ops.torch_convnd
"""

# The fake kernels stand for any device, so the derivatives can be traced without one.
TRACED = HEAD + """
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

def leaf(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, requires_grad=True)

def grads(outputs, leaves, cotangents):
    got = torch.autograd.grad(outputs, leaves, cotangents)
    for g, t in zip(got, leaves):
        assert g.shape == t.shape and g.dtype == t.dtype, (g, t)
    return got

def targets(function, *args):
    return [str(n.target) for n in make_fx(function)(*args).graph.nodes if n.op == "call_function"]

with FakeTensorMode():
    for keep in (True, False):
        x, w, b = leaf(3, 70, 16), leaf(16), leaf(16)
        y, statistics = ops.layer_norm(x, w, b, 1e-5, keep)
        assert not statistics.requires_grad
        grads(y, (x, w, b), torch.empty_like(y))
        y, _ = ops.layer_norm(x, None, leaf(16, dtype=torch.float32), 1e-5, keep)
        grads(y, (x,), torch.empty_like(y))
        m, c, r = leaf(24, 16), leaf(24), leaf(3, 70, 24)
        for kind in ("gelu", "none"):
            y, slope = ops.linear_act(x, m, c, r, kind, keep)
            assert not slope.requires_grad
            grads(y, (x, m, c, r), torch.empty_like(y))
            y, _ = ops.linear_act(x, m, None, r, kind, keep)
            grads(y, (m, r), torch.empty_like(y))
        gate, first = leaf(3, 70, 16), leaf(3, 16, dtype=torch.float32)
        lengths = torch.empty(3, dtype=torch.int32)
        h, last, carries = ops.gated_recurrence(x, gate, first, lengths, keep)
        assert not carries.requires_grad
        grads((h, last), (x, gate, first), (torch.empty_like(h), torch.empty_like(last)))
        h, last, _ = ops.gated_recurrence(x, gate, None, None, keep)
        grads(last, (x, gate), torch.empty_like(last))
        for output, name in ((h, "gated_recurrence"), (y, "linear_act")):
            try:
                torch.autograd.grad(output.float().sum(), x, create_graph=True)
            except RuntimeError as error:
                assert f"{name} is differentiable once" in str(error), error
            else:
                raise AssertionError(name)

    def step(x, w, m, gate):
        y = ops.linear_act(ops.layer_norm(x, w, None, 1e-5, True)[0], m, None, None, "gelu", True)[0]
        h, last, _ = ops.gated_recurrence(y, gate, None, None, True)
        return torch.autograd.grad((h, last), (x, w, m, gate), (torch.ones_like(h), torch.ones_like(last)))

    found = targets(step, x, w, m, leaf(3, 70, 24))
    for name in ("layer_norm", "linear_act", "gated_recurrence"):
        for form in (name, name + "_backward"):
            assert found.count(f"torch_convnd.{form}.default") == 1, (form, found)
assert not _build._LOADED
print("traced")
"""

FIRST_USE = HEAD + """
from torch import nn

class Layers(nn.Module):
    def __init__(self):
        super().__init__()
        factory = {"device": "cuda", "dtype": torch.bfloat16}
        self.norm = torch_convnd.LayerNorm(64, **factory)
        self.project = torch_convnd.LinearAct(64, 192, activation="gelu", **factory)
        self.out = torch_convnd.LinearAct(96, 64, **factory)

    def forward(self, x, first, residual):
        update, gate = self.project(self.norm(x)).chunk(2, dim=2)
        h, last = torch_convnd.gated_recurrence(update, gate, first)
        return self.out(h, residual), last

torch.manual_seed(0)
model = Layers()
x, residual, dy = (torch.randn(3, 70, 64, device="cuda").bfloat16() for _ in range(3))
first, dlast = (torch.randn(3, 96, device="cuda") for _ in range(2))
leaves = [x.requires_grad_(), first.requires_grad_(), residual.requires_grad_(), *model.parameters()]
outputs = torch.compile(model, backend="aot_eager", fullgraph=True)(x, first, residual)
got = torch.autograd.grad(outputs, leaves, (dy, dlast))
assert _build._LOADED
eager = model(x, first, residual)
for a, b in zip((*outputs, *got), (*eager, *torch.autograd.grad(eager, leaves, (dy, dlast)))):
    assert torch.equal(a, b)
print("compiled")
"""

DIRECT = HEAD + """
x = torch.randn(40, 64, device="cuda").bfloat16().requires_grad_()
w = torch.randn(32, 64, device="cuda").bfloat16().requires_grad_()
dy = torch.randn(40, 32, device="cuda").bfloat16()
assert not _build._LOADED
y, _ = ops.linear_act(x, w, None, None, "gelu_tanh", False)
assert _build._LOADED
got = torch.autograd.grad(y, (x, w), dy)
again = torch_convnd.linear_act(x, w, activation="gelu_tanh")
for a, b in zip((y, *got), (again, *torch.autograd.grad(again, (x, w), dy))):
    assert torch.equal(a, b)
print("called")
"""


def run(code, said):
    result = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=110)
    assert result.returncode == 0 and said in result.stdout, result.stdout + result.stderr


def test_derivatives_are_traced_before_loading():
    run(TRACED, "traced")


@pytest.mark.gpu
def test_compiled_as_first_use():
    run(FIRST_USE, "compiled")


@pytest.mark.gpu
def test_operator_called_first():
    run(DIRECT, "called")
