"""The delta rule where tensors have more than 2^31 elements: gradients that sum over all value heads, of queries, keys
and first states, against those of the same heads a few at a time."""

import pytest
import torch

from torch_convnd import gated_delta_rule

pytestmark = pytest.mark.gpu


def test_sums_over_heads_past_32_bits():
    tokens, heads, size, part = 33000, 512, 128, 64  # 2^31.01 values
    g = torch.Generator(device="cuda").manual_seed(2)
    q, k = (torch.randn(1, tokens, 1, size, device="cuda", generator=g).bfloat16() for _ in range(2))
    v, dy = (torch.randn(1, tokens, heads, size, device="cuda", dtype=torch.bfloat16, generator=g) for _ in range(2))
    decay = -0.2 * torch.rand(1, tokens, heads, device="cuda", generator=g)
    beta = torch.rand(1, tokens, heads, device="cuda", generator=g)
    first = 0.3 * torch.randn(1, heads, size, size, device="cuda", generator=g)
    dlast = torch.randn(1, heads, size, size, device="cuda", generator=g)

    def train(at):
        leaves = [t.detach().requires_grad_() for t in (q, k, first[:, at])]
        o, last = gated_delta_rule(*leaves[:2], v[:, :, at], decay[..., at], beta[..., at], leaves[2], normalize=True)
        grads = torch.autograd.grad((o, last), leaves, (dy[:, :, at], dlast[:, at]))
        return o.detach(), last.detach(), grads

    o, last, (dq, dk, dfirst) = train(slice(0, heads))
    sums = [torch.zeros(q.shape, device="cuda") for _ in range(2)]
    for begin in range(0, heads, part):
        at = slice(begin, begin + part)
        some, end, grads = train(at)
        for total, grad in zip(sums, grads):
            total += grad
        # Both sums' order and walks differ: an output's rounding on each side; states in float32 and two terms.
        assert (o[:, :, at].float() - some.float()).norm() <= 2 * 2.0**-8 * some.float().norm(), begin
        for a, b in ((last[:, at], end), (dfirst[:, at], grads[2])):
            assert (a - b).norm() <= 2.0**-12 * b.norm(), begin
    # Of eight sums each rounded by itself: their squares add up as the sums' own do (independent heads), so one
    # rounding of the whole and the five of the one-term operands, on each side.
    for name, a, b in (("dq", dq, sums[0]), ("dk", dk, sums[1])):
        off = (a.float() - b).norm(dim=-1) / (b.norm(dim=-1) + b.norm() / tokens**0.5)
        assert off.max() <= 12 * 2.0**-8, name
        assert (a.float() - b).norm() <= 12 * 2.0**-8 * b.norm(), name
