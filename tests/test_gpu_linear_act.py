"""linear_act on the gfx950 kernels against its 64-bit definition: few rows and tiles, every product
with ragged and unaligned operands, split K, activations, residuals, refusals, streams and graphs."""

import pytest
import torch

from sequence_helpers import EPS32, activation_reference, assert_within, linear_reference
from torch_convnd import linear_act

pytestmark = pytest.mark.gpu
KINDS = [None, "relu", "gelu", "gelu_tanh"]


def make(m, k, n, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=g).to(dtype)
    w = (torch.randn(n, k, generator=g) / k**0.5).to(dtype)
    b = (0.5 * torch.randn(n, generator=g)).to(dtype)
    r = torch.randn(m, n, generator=g).to(dtype)
    dy = torch.randn(m, n, generator=g).to(dtype)
    return [t.cuda() for t in (x, w, b, r, dy)]


def check(x, w, b, r, dy, kind):
    leaves = [t.detach().requires_grad_() for t in (x, w, b, r) if t is not None]
    it = iter(leaves)
    xl, wl, bl, rl = (None if t is None else next(it) for t in (x, w, b, r))
    y = linear_act(xl, wl, bl, rl, activation=kind, backend="native")
    grads = iter(torch.autograd.grad(y, leaves, dy))
    ref = linear_reference(x, w, b, r, kind, dy)
    assert y.dtype == x.dtype and y.is_contiguous() and y.shape == (*x.shape[:-1], w.shape[0])
    assert_within(y.reshape(-1, w.shape[0]), *ref["y"], "y")
    assert_within(next(grads).reshape(-1, w.shape[1]), *ref["dx"], "dx")
    assert_within(next(grads), *ref["dw"], "dw")
    if b is not None:
        assert_within(next(grads), *ref["db"], "db")
    if r is not None:
        assert torch.equal(next(grads), dy)
    with torch.no_grad():
        assert torch.equal(linear_act(xl, wl, bl, rl, activation=kind), y)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m", [1, 3, 16, 17, 33, 64, 65, 130, 300])
@pytest.mark.parametrize(("k", "n"), [(1, 1), (8, 16), (33, 17), (64, 128), (200, 72), (136, 333)])
def test_sizes(m, k, n, dtype):
    check(*make(m, k, n, dtype), "gelu")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("parts", ["none", "bias", "residual", "both"])
@pytest.mark.parametrize("m", [5, 150])
def test_epilogues(m, parts, kind, dtype):
    x, w, b, r, dy = make(m, 96, 80, dtype)
    check(x, w, b if parts in ("bias", "both") else None, r if parts in ("residual", "both") else None, dy, kind)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize(("m", "k", "n"), [(96, 4096, 64), (2000, 64, 48), (130, 64, 5000), (1030, 257, 515)])
def test_long_sums(m, k, n, dtype):
    """Few tiles and a long K in each of the three products: K is split over workgroups."""
    check(*make(m, k, n, dtype), "gelu_tanh")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_many_tiles(dtype):
    """More tiles than the chip takes at a time, ragged on both sides."""
    x, w, b, r, dy = make(4104, 72, 2056, dtype)
    check(x, w, b, None, dy, "relu")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m", [6, 140])
def test_strides(m, dtype):
    x, w, b, r, dy = make(m, 64, 48, dtype)
    wide = torch.randn(m, 200, device="cuda").to(dtype)
    wide[:, 3:67], wide[:, 100:148] = x, r
    check(wide[:, 3:67], w, b, wide[:, 100:148], dy, "gelu")  # rows off the vector boundary
    check(wide[:, 3:67].view(2, m // 2, 64), w, b, r.view(2, -1, 48), dy.view(2, -1, 48), "gelu")
    check(x, w.t().contiguous().t(), b, r, dy, None)
    check(x[:1].expand(m, 64), w, b, r[:1].expand(m, 48), dy[:1].expand(m, 48), "gelu")
    odd = torch.randn(m * 64 + 1, device="cuda").to(dtype)[1:].view(m, 64)
    check(odd, w, None, None, dy, None)  # storage off the vector boundary


def test_rows_do_not_mix():
    """Non-finite rows, columns and padding stay out of every other result."""
    x, w, b, r, dy = make(200, 100, 70, torch.bfloat16)
    clean = linear_act(x, w, b, r, activation="gelu")
    x2, w2 = x.clone(), w.clone()
    x2[150, 99] = float("nan")
    w2[33, 0] = float("inf")
    y = linear_act(x2, w2, b, r, activation="gelu")
    rows = [i for i in range(200) if i != 150]
    columns = [i for i in range(70) if i != 33]
    assert torch.equal(y[rows][:, columns], clean[rows][:, columns])
    assert y[150].isnan().all()


@pytest.mark.parametrize("shape", [(0, 24), (2, 0, 24)])
def test_no_rows(shape):
    x = torch.empty(shape, device="cuda", requires_grad=True)
    w = torch.randn(40, 24, device="cuda", requires_grad=True)
    b = torch.randn(40, device="cuda", requires_grad=True)
    y = linear_act(x, w, b, activation="gelu")
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
    assert y.shape == (*shape[:-1], 40) and dx.shape == shape
    assert not dw.any() and not db.any()


@pytest.mark.parametrize("wanted", [(0,), (1,), (2,), (0, 2), (1, 2)])
def test_some_gradients(wanted):
    x, w, b, r, dy = make(140, 72, 56, torch.bfloat16)
    leaves = [t.requires_grad_(i in wanted) for i, t in enumerate((x, w, b))]
    y = linear_act(*leaves, activation="gelu")
    grads = torch.autograd.grad(y, [leaves[i] for i in wanted], dy)
    ref = linear_reference(x, w, b, None, "gelu", dy)
    for i, got in zip(wanted, grads):
        assert_within(got, *ref[("dx", "dw", "db")[i]], str(i))


def test_gradient_against_differences():
    x, w, b, r, dy = make(70, 24, 20, torch.float32)
    leaves = [t.requires_grad_() for t in (x, w, b, r)]
    g = torch.Generator(device="cuda").manual_seed(5)
    step = 2.0**-6
    for kind in ("gelu", "gelu_tanh", None):
        grads = torch.autograd.grad(linear_act(*leaves, activation=kind), leaves, dy)
        for i, grad in enumerate(grads):
            direction = torch.randn(grad.shape, device="cuda", generator=g)
            value = []
            for sign in (1, -1):
                moved = [t.detach().clone() for t in leaves]
                moved[i] += sign * step * direction
                value.append((linear_act(*moved, activation=kind).double() * dy.double()).sum())
            slope = (value[0] - value[1]) / (2 * step)
            scale = (grad.double() * direction).abs().sum() + dy.abs().sum()
            assert abs(slope - (grad.double() * direction).sum()) <= scale * (4 * step**2 + 64 * 2.0**-24 / step)


def test_same_bits_on_another_stream():
    x, w, b, r, dy = make(96, 4096, 64, torch.bfloat16)
    expected = linear_act(x, w, b, r, activation="gelu")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        y = linear_act(x, w, b, r, activation="gelu")
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(y, expected)


@pytest.mark.parametrize("m", [4, 300])
def test_graph_replays(m):
    inputs = make(m, 200, 136, torch.bfloat16)
    x, w, b, r, dy = inputs
    leaves = [t.requires_grad_() for t in (x, w, b, r)]

    def step():
        y = linear_act(*leaves, activation="gelu")
        return (y, *torch.autograd.grad(y, leaves[:3], dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (1, 2, 3):
        with torch.no_grad():
            for t, f in zip(inputs, make(m, 200, 136, torch.bfloat16, seed=seed)):
                t.copy_(f)
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(captured, step()):
            assert torch.equal(got, want)


def test_autocast():
    x, w, b, r, dy = make(70, 64, 48, torch.float32)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = linear_act(x, w, b, r, activation="gelu")
    assert torch.equal(y, linear_act(*(t.bfloat16() for t in (x, w, b, r)), activation="gelu"))


def test_refusals():
    x, w, b, r, _ = make(6, 16, 8, torch.bfloat16)
    with pytest.raises(RuntimeError, match="supports float16, bfloat16 and float32"):
        linear_act(x.double(), w.double(), backend="native")
    with pytest.raises(RuntimeError, match=r"weight of \[outputs, inputs\]"):
        linear_act(x[:, :8], w)
    with pytest.raises(RuntimeError, match="same device and dtype"):
        linear_act(x, w.half())
    with pytest.raises(RuntimeError, match="same device and dtype"):
        linear_act(x, w.cpu())
    with pytest.raises(RuntimeError, match="bias must match"):
        linear_act(x, w, b[:4])
    with pytest.raises(RuntimeError, match="bias must match"):
        linear_act(x, w, b.float())
    with pytest.raises(RuntimeError, match="residual must match"):
        linear_act(x, w, b, r[:3])
    with pytest.raises(ValueError, match="Invalid activation"):
        linear_act(x, w, activation="silu")
    y = linear_act(x.requires_grad_(), w)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(y.float().sum(), x, create_graph=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("kind", ["gelu", "gelu_tanh"])
@pytest.mark.parametrize("m", [7, 90, 600])
def test_nan_stays_in_its_row(m, kind, dtype):
    """A NaN's slope reaches the gradients of its row and of the weight, and no other row."""
    x, w, b, r, dy = make(m, 40, 72, dtype)
    bad = m // 2
    clean = linear_reference(x, w, b, r, kind, dy)
    x[bad, 3] = float("nan")
    leaves = [t.requires_grad_() for t in (x, w)]
    y = linear_act(*leaves, b, r, activation=kind, backend="native")
    dx, dw = torch.autograd.grad(y, leaves, dy)
    assert y[bad].isnan().all() and dx[bad].isnan().all() and dw.isnan().all()
    rest = torch.arange(m) != bad
    assert_within(y[rest.cuda()], *(t[rest] for t in clean["y"]), "y")
    assert_within(dx[rest.cuda()], *(t[rest] for t in clean["dx"]), "dx")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", ["relu", "gelu", "gelu_tanh"])
def test_kept_slopes(kind, dtype):
    """What the forward keeps in 16 bits: every slope to half a step of 1 / 28672, 0 and 1 exactly."""
    z = torch.cat([torch.linspace(-12, 12, 4001), torch.tensor([-3e4, -60.0, 0.0, 60.0, 3e4])]).to(dtype).cuda()
    w = torch.ones(1, 1, device="cuda", dtype=dtype)
    _, kept = torch.ops.torch_convnd.linear_act(z[:, None], w, None, None, kind, True)
    assert kept.dtype == torch.int16
    z64 = z.double().cpu()
    _, slope = activation_reference(z64, kind)
    error = (kept.cpu().double().squeeze(1) / 28672 - slope).abs()
    # The evaluation adds 16 roundings of |z| + 1 where the slope changes, none where it is flat.
    assert (error <= 0.5 / 28672 + 16 * EPS32 * (z64.abs().clamp(max=16) + 1)).all(), error.max()
    assert (kept[z >= 12] == 28672).all() and (kept[z <= -12] == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [1024, 1003])
def test_outputs_beyond_the_caches(n, dtype):
    """Outputs of over 96 MB are stored past the caches: rows all over them, and the row ends."""
    m = 52001
    x, w, b, r, _ = make(m, 24, n, dtype)
    rows = torch.cat([torch.arange(0, m, 1999), torch.arange(m - 70, m)]).cuda()
    with torch.no_grad():
        y = linear_act(x, w, b, r, activation="gelu")
        again = linear_act(x, w, b, r, activation="gelu")
    assert torch.equal(y, again)
    assert_within(y[rows], *linear_reference(x[rows], w, b, r[rows], "gelu")["y"], "y")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize(("m", "k", "n"), [(5, 16385, 40), (16, 8200, 33), (20, 8192, 72), (31, 4097, 17), (33, 4099, 50)])
def test_few_long_rows(m, k, n, dtype):
    """A few rows, on either side of the lengths from which tiles take them with K in parts."""
    check(*make(m, k, n, dtype), "gelu_tanh")
