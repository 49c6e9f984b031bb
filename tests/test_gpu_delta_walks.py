"""gated_delta_rule in the forms that need many heads or many tokens: walks of 64 columns a workgroup (more than 128
walks), and segments of the tokens in 16 bits, each against the 64-bit definition with states and lengths."""

import pytest
import torch

from delta_helpers import make_delta
from test_gpu_delta_rule import TYPES, check
from torch_convnd import _build, _capi, gated_delta_rule, load_native

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize(
    "shape", [(5, 90, 16, 32, 64, 40), (3, 75, 48, 48, 128, 100), (2, 70, 11, 33, 40, 130), (9, 33, 8, 16, 100, 64)]
)
def test_walks_of_64_columns(shape, dtype):
    batch, tokens, _, heads, _, value_size = shape
    assert batch * heads * -(-value_size // 64) > 128
    data = make_delta(*shape, dtype)
    data[3][:, tokens // 2] = -float("inf")
    lengths = torch.tensor([tokens, tokens // 3, 0, tokens - 1, 1, 64, 32, tokens, 5][:batch])
    got = check(data, lengths)
    *inputs, first, _, dlast = (t.cuda() for t in data)
    if batch > 2:
        assert torch.equal(got[1][2], first[2]) and torch.equal(got[7][2], dlast[2])
    check(data, state=False, normalize=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(2, 4200, 1, 2, 128, 40), (1, 4200, 2, 4, 64, 70)])
def test_segments_of_several_heads(shape, dtype):
    """Eight segments and more, a sequence that ends in a middle one, a packed document that starts in another."""
    load_native()
    plan = _capi.delta_plan(_build.hip_library(), *shape, dtype, saving=True)
    assert plan["segments"] >= 8
    data = make_delta(*shape, dtype)
    data[3][:, 1500] = -float("inf")
    check(data, torch.tensor([4200, 2000][: shape[0]]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("held", [float("inf"), float("nan")])
def test_what_is_not_finite_stays_in_its_column(held, dtype):
    """Earlier chunks, other columns, heads and sequences are as they were; its own column holds no number from its
    token on."""
    data = make_delta(2, 150, 1, 2, 32, 48, dtype)
    *inputs, first, _, _ = (t.cuda() for t in data)
    with torch.no_grad():
        o, last = gated_delta_rule(*inputs, first)
        inputs[2][0, 70, 1, 5] = held
        p, after = gated_delta_rule(*inputs, first)
    assert not p[0, 71:, 1, 5].isfinite().any() and not after[0, 1, :, 5].isfinite().any()
    chunk = 64 if dtype != torch.float32 else 32
    p[0, 70 // chunk * chunk :, 1, 5] = o[0, 70 // chunk * chunk :, 1, 5]
    after[0, 1, :, 5] = last[0, 1, :, 5]
    assert torch.equal(o, p) and torch.equal(last, after)
