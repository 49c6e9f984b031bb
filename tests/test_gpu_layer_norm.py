"""layer_norm on the gfx950 kernels against its 64-bit definition: channel counts around every
thread arrangement's edge, types, strides, missing parameters, refusals, streams and graphs."""

import pytest
import torch

import torch_convnd
from sequence_helpers import assert_within, norm_reference
from torch_convnd import layer_norm

pytestmark = pytest.mark.gpu
EPS = 1e-5


def make(rows, c, dtype, params=None, offset=0.5, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, c, generator=g) + offset * torch.randn(c, generator=g)).to(dtype)
    w = (1 + 0.2 * torch.randn(c, generator=g)).to(params or dtype)
    b = (0.2 * torch.randn(c, generator=g)).to(params or dtype)
    dy = torch.randn(rows, c, generator=g).to(dtype)
    return [t.cuda() for t in (x, w, b, dy)]


def check(x, w, b, dy, eps=EPS):
    leaves = [t.detach().requires_grad_() for t in (x, w, b) if t is not None]
    it = iter(leaves)
    xl = next(it)
    wl = None if w is None else next(it)
    bl = None if b is None else next(it)
    y = layer_norm(xl, wl, bl, eps, backend="native")
    grads = list(torch.autograd.grad(y, leaves, dy))
    ref = norm_reference(x, w, b, eps, dy)
    flat = lambda t: t.reshape(-1, x.shape[-1])  # noqa: E731
    assert y.dtype == x.dtype and y.is_contiguous()
    assert_within(flat(y), *ref["y"], "y")
    assert_within(flat(grads.pop(0)), *ref["dx"], "dx")
    for name, p in (("dw", w), ("db", b)):
        if p is not None:
            got = grads.pop(0)
            assert got.dtype == p.dtype
            assert_within(got, *ref[name], name)
    with torch.no_grad():
        assert torch.equal(layer_norm(xl, wl, bl, eps), y)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows", [1, 5, 1100])
@pytest.mark.parametrize("c", [1, 7, 33, 64, 65, 130, 257, 512, 769, 1024, 1300, 2048, 2051])
def test_sizes(rows, c, dtype):
    check(*make(rows, c, dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize(("rows", "c"), [(3, 4097), (1030, 4100), (2, 8192), (5, 16385), (3, 33001), (700, 20000)])
def test_long_rows(rows, c, dtype):
    check(*make(rows, c, dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("c", [40, 1001, 5000])
def test_float32_parameters(c, dtype):
    check(*make(9, c, dtype, params=torch.float32))


@pytest.mark.parametrize("missing", ["weight", "bias", "both"])
def test_missing_parameters(missing):
    x, w, b, dy = make(11, 200, torch.bfloat16)
    check(x, None if missing != "bias" else w, None if missing != "weight" else b, dy)


def test_large_offset():
    """A mean a thousand times the spread: the variance is taken about the mean."""
    x, w, b, dy = make(6, 640, torch.float32)
    check(x + 1000, w, b, dy)


def test_constant_rows():
    x, w, b, dy = make(4, 96, torch.float32)
    x[1] = 3.0
    x[2] = 0.0
    y = layer_norm(x, w, b, EPS)
    assert torch.equal(y[1], b) and torch.equal(y[2], b)


def test_strides():
    x, w, b, dy = make(24, 300, torch.bfloat16)
    wide = torch.randn(24, 700, device="cuda").to(torch.bfloat16)
    wide[:, 101:401] = x
    check(wide[:, 101:401], w, b, dy)  # odd offset: no row starts on a vector boundary
    check(x.view(2, 3, 4, 300), w, b, dy.view(2, 3, 4, 300))
    check(wide.view(2, 12, 700)[:, :, 101:401], w, b, dy.view(2, 12, 300))
    check(x.view(4, 6, 300).transpose(0, 1), w, b, dy.view(6, 4, 300))  # irregular: a copy
    check(x, w, b, torch.ones((), device="cuda", dtype=x.dtype).expand(24, 300))
    every = torch.randn(24, 600, device="cuda").to(torch.bfloat16)[:, ::2]
    check(every, w, b, dy)


def test_channels_last_activation():
    x, w, b, dy = make(2 * 3 * 4 * 5, 32, torch.float16)
    stored = x.view(2, 3, 4, 5, 32)
    activation = stored.movedim(-1, 1)  # [N, C, *spatial] stored channels-last
    y = layer_norm(activation.movedim(1, -1), w, b, EPS)
    assert_within(y.reshape(-1, 32), *norm_reference(x, w, b, EPS)["y"], "y")


@pytest.mark.parametrize("shape", [(0, 16), (3, 0, 16)])
def test_no_rows(shape):
    x = torch.empty(shape, device="cuda", requires_grad=True)
    w = torch.ones(16, device="cuda", requires_grad=True)
    y = layer_norm(x, w, None, EPS)
    dx, dw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
    assert y.shape == shape and dx.shape == shape and torch.equal(dw, torch.zeros_like(w))


def test_nonfinite_rows_stay_apart():
    x, w, b, _ = make(8, 512, torch.bfloat16)
    clean = layer_norm(x, w, b, EPS)
    x[3, 17] = float("inf")
    x[5, 500] = float("nan")
    y = layer_norm(x, w, b, EPS)
    for row in (0, 1, 2, 4, 6, 7):
        assert torch.equal(y[row], clean[row])
    assert y[3].isnan().any() and y[5].isnan().all()


def test_gradient_against_differences():
    """float32 differences of the operator itself along random directions."""
    x, w, b, dy = (t.double() for t in make(3, 48, torch.float32))
    leaves = [t.float().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(layer_norm(*leaves, EPS), leaves, dy.float())
    g = torch.Generator(device="cuda").manual_seed(5)
    step = 2.0**-6
    for i, grad in enumerate(grads):
        direction = torch.randn(grad.shape, device="cuda", generator=g)
        value = []
        for sign in (1, -1):
            moved = [t.detach().clone() for t in leaves]
            moved[i] += sign * step * direction
            value.append((layer_norm(*moved, EPS).double() * dy).sum())
        slope = (value[0] - value[1]) / (2 * step)
        # Third-order term of the difference (step^2) and float32 sums over the step.
        scale = (grad.double() * direction).abs().sum() + dy.abs().sum()
        assert abs(slope - (grad.double() * direction).sum()) <= scale * (4 * step**2 + 64 * 2.0**-24 / step)


def test_other_stream():
    x, w, b, dy = make(64, 640, torch.bfloat16)
    expected = layer_norm(x, w, b, EPS)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        y = layer_norm(x, w, b, EPS)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(y, expected)


def test_graph_replays():
    x, w, b, dy = make(1500, 384, torch.bfloat16)
    leaves = [t.requires_grad_() for t in (x, w, b)]

    def step():
        y = layer_norm(*leaves, EPS)
        return (y, *torch.autograd.grad(y, leaves, dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (1, 2, 3):
        fresh = make(1500, 384, torch.bfloat16, seed=seed)
        with torch.no_grad():
            for t, f in zip((*leaves, dy), fresh):
                t.copy_(f)
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(captured, step()):
            assert torch.equal(got, want)


def test_refusals():
    x, w, b, _ = make(4, 32, torch.bfloat16)
    with pytest.raises(RuntimeError, match="supports float16, bfloat16 and float32"):
        layer_norm(x.double(), None, None, backend="native")
    with pytest.raises(RuntimeError, match="weight must match the input's channels"):
        layer_norm(x, w[:16], b)
    with pytest.raises(RuntimeError, match="bias must match the input's channels"):
        layer_norm(x, w, b.cpu())
    with pytest.raises(RuntimeError, match="weight must match the input's channels"):
        layer_norm(x, w.half(), b)
    with pytest.raises(RuntimeError, match="same dtype"):
        layer_norm(x, w.float(), b)
    with pytest.raises(RuntimeError, match="channels in its last dimension"):
        layer_norm(torch.empty(3, 0, device="cuda"))
    with pytest.raises(ValueError, match="Invalid backend"):
        layer_norm(x, w, b, backend="cuda")
    y = layer_norm(x.requires_grad_(), w, b)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(y.float().sum(), x, create_graph=True)
    assert torch_convnd.layer_norm(x.double(), backend="torch").dtype == torch.float64
