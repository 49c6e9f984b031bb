"""The delta rule where tensors have more than 2^31 elements: a head at their end against the same head alone."""

import pytest
import torch

from torch_convnd import gated_delta_rule

pytestmark = pytest.mark.gpu


def test_elements_past_32_bits():
    tokens, heads, size = 33000, 512, 128  # 2^31.01 values
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k = (torch.randn(1, tokens, 1, size, device="cuda", generator=g).bfloat16() for _ in range(2))
    v, dy = (torch.randn(1, tokens, heads, size, device="cuda", dtype=torch.bfloat16, generator=g) for _ in range(2))
    decay = -0.2 * torch.rand(1, tokens, heads, device="cuda", generator=g)
    beta = torch.rand(1, tokens, heads, device="cuda", generator=g)

    def train(v, decay, beta, dy):
        leaves = [t.detach().requires_grad_() for t in (v, decay, beta)]
        o, last = gated_delta_rule(q, k, *leaves, normalize=True)
        return o.detach(), last.detach(), *torch.autograd.grad(o, leaves, dy)

    whole = train(v, decay, beta, dy)
    alone = train(v[:, :, -1:], decay[..., -1:], beta[..., -1:], dy[:, :, -1:])
    for i, (a, b) in enumerate(zip(whole, alone)):
        a = (a[:, -1:] if i == 1 else a[:, :, -1:]).float()
        # Other plans sum in another order: outputs differ by their rounding (2^-8 each), gradients of decay and beta
        # by those of the one-term operands as well (five on each side).
        assert (a - b.float()).norm() <= (2 * 2.0**-8 if i < 3 else 12 * 2.0**-8) * b.float().norm(), i
        assert (a[:, -1] - b.float()[:, -1]).norm() <= 24 * 2.0**-8 * b.float()[:, -1].norm(), i
