"""Gradients of the delta rule and the gated linear layer where nothing has loaded the native library yet: graphs
traced and compiled as a program's first use. Each test runs a process of its own, since loading cannot be undone."""

import pytest

from test_sequence_first_use import HEAD, run

# The fake kernels stand for any device, so the derivatives can be traced without one.
TRACED = HEAD + """
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

def leaf(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, requires_grad=True)

def grads(outputs, leaves, cotangents):
    for g, t in zip(torch.autograd.grad(outputs, leaves, cotangents), leaves):
        assert g.shape == t.shape and g.dtype == t.dtype, (g, t)

def once(output, x, name):
    try:
        torch.autograd.grad(output.float().sum(), x, create_graph=True)
    except RuntimeError as error:
        assert f"{name} is differentiable once" in str(error), error
    else:
        raise AssertionError(name)

with FakeTensorMode():
    q, k, v = leaf(3, 70, 2, 16), leaf(3, 70, 2, 16), leaf(3, 70, 4, 20)
    decay, beta = (leaf(3, 70, 4, dtype=torch.float32) for _ in range(2))
    first, lengths = leaf(3, 4, 16, 20, dtype=torch.float32), torch.empty(3, dtype=torch.int32)
    x, w, b = leaf(3, 70, 16), leaf(24, 16), leaf(24)
    for keep in (True, False):
        o, last, saved = ops.gated_delta_rule(q, k, v, decay, beta, first, lengths, 0.25, True, keep)
        assert not saved.requires_grad
        leaves = (q, k, v, decay, beta, first)
        grads((o, last), leaves, (torch.empty_like(o), torch.empty_like(last)))
        o, last, _ = ops.gated_delta_rule(q, k, v, decay, beta, None, None, 0.25, False, keep)
        grads(last, leaves[:5], torch.empty_like(last))
        o, _, _ = ops.gated_delta_rule(q, k, v, decay, beta, None, None, 0.25, False, keep)
        grads(o, (q, v), torch.empty_like(o))
        once(o if keep else ops.gated_delta_rule(q, k, v, decay, beta, None, None, 0.25, False, keep)[0], q,
             "gated_delta_rule")
        y, kept = ops.gated_linear(x, w, b, "silu", keep)
        assert not kept.requires_grad
        grads(y, (x, w, b), torch.empty_like(y))
        y, _ = ops.gated_linear(x, w, None, "relu", keep)
        grads(y, (w,), torch.empty_like(y))
        once(ops.gated_linear(x, w, b, "gelu", keep)[0], x, "gated_linear")

    def step(x, w, q, k, decay, beta):
        y = ops.gated_linear(x, w, None, "silu", True)[0]
        o, last, _ = ops.gated_delta_rule(q, k, y.unflatten(2, (4, 3)), decay, beta, None, None, 1.0, True, True)
        return torch.autograd.grad((o, last), (x, w, q, k, decay, beta), (torch.ones_like(o), torch.ones_like(last)))

    found = [str(n.target) for n in make_fx(step)(x, w, q, k, decay, beta).graph.nodes if n.op == "call_function"]
    for name in ("gated_delta_rule", "gated_linear"):
        for form in (name, name + "_backward"):
            assert found.count(f"torch_convnd.{form}.default") == 1, (form, found)
assert not _build._LOADED
print("traced")
"""

COMPILED = HEAD + """
torch.manual_seed(0)
model = torch_convnd.GatedDeltaBlock(64, 2, device="cuda", dtype=torch.bfloat16)
x, dy = (torch.randn(3, 70, 64, device="cuda").bfloat16() for _ in range(2))
window, hidden = model.initial_state(x)
dlast = torch.randn_like(hidden)
leaves = [x.requires_grad_(), hidden.requires_grad_(), *model.parameters()]

def call(x, window, hidden):
    y, (_, last) = model(x, (window, hidden))
    return y, last

outputs = torch.compile(call, backend="aot_eager", fullgraph=True)(x, window, hidden)
got = torch.autograd.grad(outputs, leaves, (dy, dlast))
assert _build._LOADED
eager = call(x, window, hidden)
for a, b in zip((*outputs, *got), (*eager, *torch.autograd.grad(eager, leaves, (dy, dlast)))):
    assert torch.equal(a, b)
print("compiled")
"""

# Kernels with more LDS than they get unasked, whose first launch is under capture.
CAPTURED = HEAD + """
torch_convnd.load_native()
torch.manual_seed(0)
q, k, v, dy = (torch.randn(2, 130, 3, 128, device="cuda").bfloat16() for _ in range(4))
decay, beta = -torch.rand(2, 130, 3, device="cuda"), torch.rand(2, 130, 3, device="cuda")
x, w = torch.randn(300, 64, device="cuda").bfloat16(), torch.randn(96, 64, device="cuda").bfloat16()
g = torch.randn(300, 48, device="cuda").bfloat16()

def call():
    o, last, saved = ops.gated_delta_rule(q, k, v, decay, beta, None, None, 0.1, True, True)
    grads = ops.gated_delta_rule_backward(dy, None, q, k, v, decay, beta, None, saved, 0.1, True, False)
    y, kept = ops.gated_linear(x, w, None, "silu", True)
    more = ops.gated_linear_backward(g, x, w, kept, "silu", [True, True, True])
    return o, last, *grads[:5], y, *more

torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.no_grad():
    with torch.cuda.graph(graph):
        captured = call()
    for seed in (1, 2, 3):
        for t in (q, k, v, dy, x, g):
            t.copy_(torch.randn(t.shape, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, call()):
            assert torch.equal(a, b)
print("captured")
"""


def test_derivatives_are_traced_before_loading():
    run(TRACED, "traced")


@pytest.mark.gpu
def test_compiled_as_first_use():
    run(COMPILED, "compiled")


@pytest.mark.gpu
def test_captured_as_first_use():
    run(CAPTURED, "captured")
