"""Positions with several axes: what callers may pass for the axes.  Against write with the same numbers in a list."""
import numpy as np
import pytest
import torch

from attn_cases import DEV, generator, make_attention, randn
from nano_ktrans_amd import rope_axes, rope_table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", [tuple, np.array, lambda x: np.array(x, dtype=np.int32), lambda x: np.array(x, dtype=np.uint8),
                                  torch.tensor, lambda x: [np.int64(i) for i in x]])
def test_axes_of_any_integers(gpu_device, kind):
    g = generator(11)
    attn, twin = (make_attention(8, 2, 128, "bf16", 64, 2) for _ in range(2))
    axes, rope = rope_axes([24, 20, 20], interleaved=True), rope_table(500, 128, device=DEV)
    q, k, v = randn(g, 70, 8, 128), randn(g, 70, 2, 128), randn(g, 70, 2, 128)
    positions, slots = torch.randint(0, 500, (3, 70), generator=g, device=DEV), torch.arange(70, device=DEV)
    want = twin.write(q, k, v, positions, slots, rope, axes=axes)
    assert torch.equal(attn.write(q, k, v, positions, slots, rope, axes=kind(axes)), want)
    assert torch.equal(attn.k_cache, twin.k_cache)


@pytest.mark.parametrize("axes", [[0.0] * 64, np.zeros(64), [0] * 63 + [1.5], np.zeros((64, 1), dtype=np.int64), ["0"] * 64])
def test_axes_that_are_none(gpu_device, axes):
    g = generator(12)
    attn = make_attention(8, 2, 128, "bf16", 64, 2)
    with pytest.raises((ValueError, TypeError)):
        attn.write(randn(g, 3, 8, 128), randn(g, 3, 2, 128), randn(g, 3, 2, 128),
                   torch.zeros(3, 3, dtype=torch.int64, device=DEV), torch.arange(3, device=DEV),
                   rope_table(50, 128, device=DEV), axes=axes)
    torch.cuda.synchronize()
    assert not bool(attn.k_cache.any())
