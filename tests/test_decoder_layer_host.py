"""FusedDecoderLayer's plumbing, without a GPU."""
import torch
from torch import nn

from nano_ktrans_amd import FusedDecoderLayer


class Double(nn.Module):
    """An attention half of the caller's own, as it was before weights could be given."""

    def forward(self, hidden_states, batch):
        return 2 * hidden_states + batch


class Weighing(nn.Module):
    def forward(self, hidden_states, batch, weights=None):
        if weights is not None:
            weights += 1
        return 2 * hidden_states + batch


def test_attention_halves_without_weights_still_fit():
    x = torch.arange(6.0).view(2, 3)
    assert torch.equal(FusedDecoderLayer(Double(), nn.Identity())(x, 1.0), 2 * x + 1)


def test_weights_reach_the_attention_half():
    x, w = torch.arange(6.0).view(2, 3), torch.zeros(4)
    layer = FusedDecoderLayer(Weighing(), nn.Identity())
    assert torch.equal(layer(x, 1.0, w), 2 * x + 1) and bool((w == 1).all())
    assert torch.equal(layer(x, 1.0, weights=w), 2 * x + 1) and bool((w == 2).all())
    layer(x, 1.0)
    assert bool((w == 2).all())
