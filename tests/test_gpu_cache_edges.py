"""The paged cache's calls on the GPU where a batch is padded, indexes lie outside the cache, or a call is large."""
import sys

import pytest
import torch

from attn_cases import DEV, U, dense, generator, make_attention, poison, randn, rotated
from nano_ktrans_amd import rope_table
from nano_ktrans_amd import _native as N
from test_gpu_cache import check_stored

pytestmark = pytest.mark.gpu


def announce(msg):
    sys.__stderr__.write(f"[gpu-case] {msg}\n")
    sys.__stderr__.flush()


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
@pytest.mark.parametrize("tokens", [9, 1100])
def test_padding_positions_are_no_error(gpu_device, fmt, tokens):
    """A padded batch as ``slots`` takes it: tokens at negative positions are not stored, their queries are zero,
    and nothing is reported; a position outside the rotation table of a token that has a slot still is."""
    announce(f"padding positions {fmt} T={tokens}")
    attn = make_attention(4, 2, 128, fmt, 64, 40)
    poison(attn)
    g = generator(4)
    table = torch.randperm(40, generator=g, device=DEV).view(2, 20).to(torch.int32)
    seqs = torch.arange(tokens, device=DEV) % 2
    positions = torch.arange(tokens, device=DEV) // 2 + 60
    padding = torch.zeros(tokens, dtype=torch.bool, device=DEV)
    padding[[1, tokens // 2, tokens - 2, tokens - 1]] = True
    positions[padding] = -1
    positions[1] = -77
    q, k, v = (randn(g, tokens, h, 128) for h in (4, 2, 2))
    rope = rope_table(700, 128, 1e4, DEV)
    slots = attn.slots(table, seqs, positions)
    out = attn.write(q, k, v, positions, slots, rope)
    attn.check_status()
    assert bool((out[padding] == 0).all())
    on = ~padding
    rows = rope[positions[on]]
    want, spread = rotated(q[on], None, 0, rows)
    assert bool(((out[on].double() - want).abs() <= U * want.abs() + 2.0 ** -20 * spread * (1 + U)).all())
    want_k, spread_k = rotated(k[on], None, 0, rows)
    check_stored(attn, slots[on], want_k, spread_k, v.double()[on])
    every = torch.arange(40 * 64, device=DEV)
    stored = ~torch.isnan(dense(attn, every)[0]).flatten(1).any(dim=1)
    assert torch.equal(every[stored], slots[on].sort().values)
    slots[1] = 5
    attn.write(q, k, v, positions, slots, rope)
    assert attn.status() == {name: name == "bad_position" for name in N.ATTN_STATUS}
