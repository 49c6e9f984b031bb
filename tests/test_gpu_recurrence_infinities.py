"""An infinite state over tokens whose gates' product passes below float32's range: token by token it
stays infinite, and so it has to where the tokens are joined as maps, in every kernel of the
gated recurrence and in both directions."""

import pytest
import torch

from torch_convnd import gated_recurrence

pytestmark = pytest.mark.gpu


def walk(x, gate, state, dy, dlast):
    """h, the last state, dx and dfirst token by token in float32, as the definition reads."""
    keep, take = torch.sigmoid(gate), torch.sigmoid(-gate)
    h = []
    for t in range(x.shape[1]):
        state = keep[:, t] * state + take[:, t] * x[:, t]
        h.append(state)
    back, dx = dlast, [None] * x.shape[1]
    for t in reversed(range(x.shape[1])):
        total = back + dy[:, t]
        dx[t], back = take[:, t] * total, keep[:, t] * total
    return torch.stack(h, 1), state, torch.stack(dx, 1), back


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize(
    ("batch", "tokens", "c"),
    [(3, 8, 40), (3, 300, 40), (2, 300, 2050), (40, 400, 2048), (300, 150, 130), (2, 1500, 33), (1, 9000, 130)],
)
def test_infinite_states_stay_infinite(batch, tokens, c, dtype):
    g = torch.Generator().manual_seed(tokens)
    x, dy = (torch.randn(batch, tokens, c, generator=g).to(dtype).cuda() for _ in range(2))
    gate = (torch.randn(batch, tokens, c, generator=g) - 8).to(dtype).cuda()  # each token keeps about 3e-4
    gate[:, tokens // 2, 1::5] = -float("inf")  # a closed gate: zero times infinity is NaN there
    first, dlast = (torch.randn(batch, c, generator=g).cuda() for _ in range(2))
    first[:, ::3], first[:, 1::3] = float("inf"), -float("inf")
    dlast[:, ::2] = float("inf")
    x[-1, tokens // 3, 2::3] = float("inf")
    leaves = [x.requires_grad_(), gate, first.requires_grad_()]
    h, last = gated_recurrence(*leaves, backend="native")
    dx, dfirst = torch.autograd.grad((h, last), (x, first), (dy, dlast))
    with torch.no_grad():
        wants = walk(x.float(), gate.float(), first, dy.float(), dlast)
    for name, got, want in zip(("h", "last", "dx", "dfirst"), (h, last, dx, dfirst), wants):
        got = got.detach()
        assert torch.equal(got.isnan(), want.isnan()), name
        assert torch.equal(got.isposinf(), want.isposinf()), name
        assert torch.equal(got.isneginf(), want.isneginf()), name
