"""What the state of a block holds on to between calls."""

import pytest
import torch

from torch_convnd import GatedConvBlock


@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("tokens", [1, 3, 4, 64])
@pytest.mark.parametrize("kernel_size", [1, 4])
@pytest.mark.parametrize("batch", [1, 3])
def test_state_does_not_hold_the_prompt(batch, kernel_size, tokens, ragged):
    torch.manual_seed(0)
    model = GatedConvBlock(12, kernel_size=kernel_size, expansion=2)
    x = torch.randn(batch, tokens, 12)
    lengths = torch.full((batch,), tokens) if ragged else None
    with torch.no_grad():
        _, (window, hidden) = model(x, None, lengths)
        padded = torch.cat((x.new_zeros(batch, kernel_size - 1, 12), model.norm_tokens(x)), dim=1)
    assert torch.equal(window, padded[:, tokens:])
    # A step's window is a view of itself and the one token: at most as much again as it needs.
    assert window.untyped_storage().nbytes() <= 2 * window.numel() * window.element_size()
    assert hidden.untyped_storage().nbytes() == hidden.numel() * hidden.element_size()
