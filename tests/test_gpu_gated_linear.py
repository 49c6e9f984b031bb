"""gated_linear on the gfx950 kernels against its 64-bit definition: few rows and tiles, ragged and unaligned
operands, split K, activations, biases, strides, refusals, streams and graphs."""

import pytest
import torch

from gated_linear_helpers import gated_reference
from sequence_helpers import assert_within
from torch_convnd import gated_linear

pytestmark = pytest.mark.gpu
KINDS = ["silu", "relu", "gelu", "gelu_tanh"]


def make(m, k, n, dtype, seed=0):
    """x, weight, bias and the cotangent of `n` outputs."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=g).to(dtype)
    w = (1.5 * torch.randn(2 * n, k, generator=g) / k**0.5).to(dtype)
    b = (0.5 * torch.randn(2 * n, generator=g)).to(dtype)
    dy = torch.randn(m, n, generator=g).to(dtype)
    return [t.cuda() for t in (x, w, b, dy)]


def assert_rounded(actual, value, noise, what):
    """assert_within where the value is in the type's range; past its largest number the rounding is infinity
    (or that number, where the value is within its noise of it)."""
    largest = torch.finfo(actual.dtype).max
    got, past = actual.detach().double().cpu(), value.abs() + noise > largest
    assert (got[past].sign() == value[past].sign()).all() and (got[past].abs() >= largest * 0.99).all(), what
    beyond = value.abs() - noise > largest * (1 + torch.finfo(actual.dtype).eps)
    assert got[beyond].isinf().all(), what
    assert_within(actual.cpu().masked_fill(past, 0), value.masked_fill(past, 0), noise, what)


def check(x, w, b, dy, kind="silu"):
    leaves = [t.detach().requires_grad_() for t in (x, w, b) if t is not None]
    y = gated_linear(*leaves, activation=kind, backend="native")
    grads = torch.autograd.grad(y, leaves, dy)
    ref = gated_reference(x, w, b, kind, dy)
    n = w.shape[0] // 2
    assert y.dtype == x.dtype and y.is_contiguous() and y.shape == (*x.shape[:-1], n)
    assert_rounded(y.reshape(-1, n), *ref["y"], "y")
    assert_rounded(grads[0].reshape(-1, x.shape[-1]), *ref["dx"], "dx")
    assert_rounded(grads[1], *ref["dw"], "dw")
    if b is not None:
        assert_rounded(grads[2], *ref["db"], "db")
    with torch.no_grad():
        assert torch.equal(gated_linear(*leaves, activation=kind), y)
    return y.detach(), grads


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m", [1, 3, 16, 17, 33, 64, 65, 130, 300])
@pytest.mark.parametrize(("k", "n"), [(1, 1), (8, 8), (33, 17), (64, 128), (200, 36), (136, 333)])
def test_sizes(m, k, n, dtype):
    check(*make(m, k, n, dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("m", [5, 150])
def test_epilogues(m, bias, kind, dtype):
    x, w, b, dy = make(m, 96, 80, dtype)
    check(x, w, b if bias else None, dy, kind)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize(("m", "k", "n"), [(96, 4096, 32), (2000, 64, 24), (130, 64, 2500), (1030, 257, 259)])
def test_long_sums(m, k, n, dtype):
    """Few tiles and a long K in each of the three products: K is split over workgroups."""
    check(*make(m, k, n, dtype), "gelu_tanh")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_many_tiles(dtype):
    """More tiles than the chip takes at a time, of each size, ragged on both sides."""
    x, w, _, dy = make(4104, 72, 1029, dtype)
    check(x, w, None, dy)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m", [6, 140])
def test_strides(m, dtype):
    x, w, b, dy = make(m, 64, 48, dtype)
    wide = torch.randn(m, 200, device="cuda").to(dtype)
    wide[:, 3:67] = x
    check(wide[:, 3:67], w, b, dy)  # rows off the vector boundary
    check(wide[:, 3:67].view(2, m // 2, 64), w, b, dy.view(2, -1, 48))
    check(x, w.t().contiguous().t(), b, dy)
    check(x[:1].expand(m, 64), w, b, dy[:1].expand(m, 48))
    odd = torch.randn(m * 64 + 1, device="cuda").to(dtype)[1:].view(m, 64)
    check(odd, w, None, dy)


def test_rows_and_outputs_do_not_mix():
    x, w, b, dy = make(200, 100, 70, torch.bfloat16)
    clean = gated_linear(x, w, b)
    x[150, 99] = float("nan")
    w[33, 0] = float("nan")
    w[70 + 41, 5] = float("nan")
    y = gated_linear(x, w, b)
    rows = [i for i in range(200) if i != 150]
    columns = [i for i in range(70) if i not in (33, 41)]
    assert torch.equal(y[rows][:, columns], clean[rows][:, columns])
    assert y[150].isnan().all() and y[:, [33, 41]].isnan().all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_large_sums(kind, dtype):
    """Gates far out on either side, where the activation is its argument or next to nothing."""
    x, w, b, dy = make(70, 32, 40, dtype)
    check(8 * x, 8 * w, b, dy, kind)


@pytest.mark.parametrize("shape", [(0, 24), (2, 0, 24)])
def test_no_rows(shape):
    x = torch.empty(shape, device="cuda", requires_grad=True)
    w = torch.randn(40, 24, device="cuda", requires_grad=True)
    b = torch.randn(40, device="cuda", requires_grad=True)
    y = gated_linear(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
    assert y.shape == (*shape[:-1], 20) and dx.shape == shape
    assert not dw.any() and not db.any()


@pytest.mark.parametrize("wanted", [(0,), (1,), (2,), (0, 2), (1, 2), (0, 1)])
@pytest.mark.parametrize("n", [56, 33])
def test_some_gradients(wanted, n):
    x, w, b, dy = make(140, 72, n, torch.bfloat16)
    leaves = [t.requires_grad_(i in wanted) for i, t in enumerate((x, w, b))]
    y = gated_linear(*leaves)
    grads = torch.autograd.grad(y, [leaves[i] for i in wanted], dy)
    ref = gated_reference(x, w, b, "silu", dy)
    for i, got in zip(wanted, grads):
        assert_within(got, *ref[("dx", "dw", "db")[i]], str(i))


def test_gradient_against_differences():
    x, w, b, dy = make(70, 24, 20, torch.float32)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    g = torch.Generator(device="cuda").manual_seed(5)
    step = 2.0**-6
    for kind in ("silu", "gelu", "gelu_tanh"):
        grads = torch.autograd.grad(gated_linear(*leaves, activation=kind), leaves, dy)
        for i, grad in enumerate(grads):
            direction = torch.randn(grad.shape, device="cuda", generator=g)
            value = []
            for sign in (1, -1):
                moved = [t.detach().double().cpu() for t in leaves]
                moved[i] += sign * step * direction.double().cpu()
                value.append((gated_reference(*moved, kind)["y"][0] * dy.double().cpu()).sum())
            slope = (value[0] - value[1]) / (2 * step)
            scale = (grad.double() * direction).abs().sum().item() + dy.abs().sum().item()
            assert abs(slope - (grad.double() * direction).sum().item()) <= scale * (16 * step**2 + 2.0**-16)


def test_same_bits_on_another_stream():
    x, w, b, dy = make(300, 128, 96, torch.bfloat16)
    expected = check(x, w, b, dy)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = check(x, w, b, dy)
    torch.cuda.current_stream().wait_stream(stream)
    for a, c in zip((got[0], *got[1]), (expected[0], *expected[1])):
        assert torch.equal(a, c)


@pytest.mark.parametrize("m", [4, 300])
def test_graph_replays(m):
    held = make(m, 130, 66, torch.bfloat16)

    def step():
        leaves = [t.detach().requires_grad_() for t in held[:3]]
        y = gated_linear(*leaves, activation="gelu")
        return (y.detach(), *torch.autograd.grad(y, leaves, held[3]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (1, 2, 3):
        for t, new in zip(held, make(m, 130, 66, torch.bfloat16, seed=seed)):
            t.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, step()):
            assert torch.equal(a, b)


def test_autocast():
    x, w, b, dy = make(40, 64, 48, torch.float32)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    with torch.autocast("cuda", torch.bfloat16):
        y = gated_linear(*leaves)
    assert y.dtype == torch.bfloat16
    grads = torch.autograd.grad(y, leaves, dy.bfloat16())
    ref = gated_reference(x.bfloat16(), w.bfloat16(), b.bfloat16(), "silu", dy.bfloat16())
    assert_within(y, *ref["y"], "y")
    for name, got in zip(("dx", "dw", "db"), grads):
        assert got.dtype == torch.float32
        assert_within(got.bfloat16(), *ref[name], name)


def test_refusals():
    x, w, b, dy = make(6, 16, 8, torch.bfloat16)

    def refused(match, *inputs, kind=RuntimeError, **options):
        with pytest.raises(kind, match=match):
            gated_linear(*inputs, **options)

    refused("Invalid activation", x, w, kind=ValueError, activation="tanh")
    refused("Invalid activation", x, w, kind=ValueError, activation=None)
    refused("supports float16, bfloat16 and float32", x.double(), w.double(), backend="native")
    refused("expects an input", x, w[:, :8])
    refused("expects an input", x, w[:15])
    refused("expects an input", x, w[0])
    refused("same device and dtype", x, w.half())
    refused("same device and dtype", x, w.cpu())
    refused("bias must match", x, w, b[:8])
    refused("bias must match", x, w, b.float())
    y = gated_linear(x.requires_grad_(), w)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(y.float().sum(), x, create_graph=True)
