"""gated_linear where a product's other half is infinite: a relu that is shut passes nothing on to its gate."""

import pytest
import torch

from test_gpu_gated_linear import make
from torch_convnd import gated_linear

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m", [3, 150, 1100])
def test_a_shut_gate_beside_an_infinity(m, dtype):
    x, w, b, dy = make(m, 64, 40, dtype)
    x[:, 0] = 1
    w[40 + 3, 0] = float("inf")  # output 3's factor beside its gate
    b[3] = -100  # shut in every row
    b[43] = 0
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(gated_linear(*leaves, activation="relu", backend="native"), leaves, dy)
    leaves = [t.detach().float().cpu().requires_grad_() for t in (x, w, b)]
    expected = torch.autograd.grad(gated_linear(*leaves, activation="relu"), leaves, dy.float().cpu())
    assert not expected[1][3].any() and not expected[2][3].any()
    assert not grads[1][3].any() and not grads[2][3].any()
    for grad, e in zip(grads, expected):
        assert torch.equal(grad.isnan().cpu(), e.isnan())
