"""linear_act on its large tiles against the 64-bit definition: 128 and 256 tiles of several stages, with K
whole and in parts, in the forward, each gradient alone and both at once, at ragged sizes. Each case
asserts the plan it is there for. Results are compared at a sample of rows (outputs, the input's gradient)
and of outputs (the weight's and the bias's), which needs a part of the 64-bit products only."""

import pytest
import torch

from sequence_helpers import assert_within, linear_reference
from torch_convnd import _build, _capi, linear_act, load_native

pytestmark = pytest.mark.gpu
FORWARD, INPUT, WEIGHT, BOTH = range(4)
HALF = (torch.bfloat16, torch.float16)
SINGLE = (torch.float32,)

# what, types, tile, K in parts, rows, inputs, outputs
CASES = [
    (FORWARD, HALF, 128, False, 267, 299, 10099),
    (FORWARD, HALF, 128, True, 200, 2253, 4185),
    (FORWARD, HALF, 256, False, 1257, 301, 10023),
    (FORWARD, HALF, 256, False, 8192, 1024, 4096),
    (FORWARD, HALF, 256, True, 5523, 7707, 139),
    (INPUT, HALF, 128, False, 269, 9933, 301),
    (INPUT, HALF, 128, True, 211, 4201, 2275),
    (INPUT, HALF, 256, False, 5865, 2059, 299),
    (INPUT, HALF, 256, True, 5773, 179, 7699),
    (WEIGHT, HALF, 128, False, 267, 267, 10099),
    (WEIGHT, HALF, 128, True, 6925, 201, 1397),
    (WEIGHT, HALF, 256, False, 299, 1255, 9865),
    (WEIGHT, HALF, 256, True, 11719, 6535, 131),
    (BOTH, HALF, 128, False, 287, 4887, 261),
    (BOTH, HALF, 128, True, 2487, 197, 1765),
    (BOTH, HALF, 256, False, 269, 12293, 561),
    (BOTH, HALF, 256, True, 6471, 133, 4391),
    (BOTH, HALF, 256, True, 8192, 1024, 4096),
    (FORWARD, SINGLE, 128, False, 391, 343, 7013),
    (FORWARD, SINGLE, 128, True, 1833, 1045, 553),
    (INPUT, SINGLE, 128, False, 5677, 545, 341),
    (INPUT, SINGLE, 128, True, 577, 1641, 1049),
    (WEIGHT, SINGLE, 128, False, 343, 9913, 287),
    (WEIGHT, SINGLE, 128, True, 1029, 2151, 461),
    (BOTH, SINGLE, 128, False, 333, 4521, 333),
    (BOTH, SINGLE, 128, True, 1045, 465, 983),
]


def make(m, k, n, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    return [t.to(dtype) for t in (randn(m, k), randn(n, k) / k**0.5, 0.5 * randn(n), randn(m, n), randn(m, n))]


def sample(n):
    """Some two hundred of n: the first and last tile's, and spread ones."""
    picked = torch.cat([torch.arange(min(n, 40)), torch.arange(0, n, max(1, n // 97)), torch.arange(max(0, n - 70), n)])
    return picked.unique().cuda()


@pytest.mark.parametrize(
    ("what", "dtype", "tile", "split", "m", "k", "n"),
    [(what, dtype, *rest) for what, types, *rest in CASES for dtype in types],
)
def test_large_tiles(what, dtype, tile, split, m, k, n):
    load_native()
    plan = _capi.linear_plan(_build.hip_library(), m, k, n, dtype, what)
    parts = (plan["input_splits"], plan["weight_splits"]) if what == BOTH else (plan["splits"],)
    assert plan["tile"] == tile and (max(parts) > 1) == split, plan
    x, w, b, r, dy = make(m, k, n, dtype)
    rows, outputs = sample(m), sample(n)
    kind = "gelu_tanh"
    if what == FORWARD:
        with torch.no_grad():
            y = linear_act(x, w, b, r, activation=kind, backend="native")
            again = linear_act(x, w, b, r, activation=kind, backend="native")
        assert torch.equal(y, again)
        assert_within(y[rows], *linear_reference(x[rows], w, b, r[rows], kind)["y"], "y")
        return
    leaves = [t.requires_grad_() for t in ((x,) if what == INPUT else (w, b) if what == WEIGHT else (x, w, b))]
    y = linear_act(x, w, b, r, activation=kind, backend="native")
    got = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    for one, other in zip(got, torch.autograd.grad(y, leaves, dy)):
        assert torch.equal(one, other)
    if what != WEIGHT:
        assert_within(got[0][rows], *linear_reference(x[rows], w, b, None, kind, dy[rows])["dx"], "dx")
    if what != INPUT:
        ref = linear_reference(x, w[outputs], b[outputs], None, kind, dy[:, outputs])
        assert_within(got[-2][outputs], *ref["dw"], "dw")
        assert_within(got[-1][outputs], *ref["db"], "db")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_do_not_mix_in_large_tiles(dtype):
    """A NaN row of x and an infinite row of W stay in their row and column, through the ragged ends too."""
    m, k, n = (1257, 301, 10023) if dtype == torch.bfloat16 else (391, 343, 7013)
    load_native()
    assert _capi.linear_plan(_build.hip_library(), m, k, n, dtype, FORWARD)["tile"] >= 128
    x, w, b, r, _ = make(m, k, n, dtype)
    with torch.no_grad():
        clean = linear_act(x, w, b, r, activation="gelu")
        x[m - 2, k - 1] = float("nan")
        w[n - 3, 0] = float("inf")
        y = linear_act(x, w, b, r, activation="gelu")
    rows, columns = torch.arange(m) != m - 2, torch.arange(n) != n - 3
    assert torch.equal(y[rows][:, columns], clean[rows][:, columns]) and y[m - 2].isnan().all()
