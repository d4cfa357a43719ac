"""Attention over the paged cache on the GPU at the ends of its values' and indexes' ranges, against the plain
64-bit implementation in attn_cases.py (which has the tolerances)."""
import sys

import pytest
import torch

from attn_cases import DEV, generator, make_problem, randn, split_rows

pytestmark = pytest.mark.gpu


def announce(msg):
    sys.__stderr__.write(f"[gpu-case] {msg}\n")
    sys.__stderr__.flush()


def starts_of(counts):
    return torch.tensor(split_rows(counts), dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("counts", [None, [9, 40]])
def test_64_bit_indexes_do_not_wrap(gpu_device, counts):
    """Integers of 64 bits that 32 bits do not hold are out of range, not what their lower half says."""
    announce(f"64-bit indexes, rows {counts}")
    p = make_problem([200, 200], heads=8, kv_heads=2, dim=128, fmt="bf16", page=64, seed=16)
    n = counts or [1, 1]
    starts = starts_of(counts) if counts else None
    q = randn(generator(17), sum(n), 8, 128)
    good = p.attn.forward(q, p.table, p.lens, starts)
    for by in (1 << 32, -(1 << 32), 1 << 40):
        table = p.table.long()
        table[0, 1] += by
        got = p.attn.forward(q, table, p.lens, starts)
        st = p.attn.status()
        assert st["bad_page"] and not st["bad_length"], by
        assert torch.equal(got[n[0]:], good[n[0]:]) and not torch.equal(got[:n[0]], good[:n[0]])
        p.attn._status.zero_()
        lens = p.lens.long()
        lens[0] += by
        got = p.attn.forward(q, p.table, lens, starts)
        assert p.attn.status()["bad_length"], by
        assert torch.equal(got[n[0]:], good[n[0]:]) and not torch.equal(got[:n[0]], good[:n[0]])
        p.attn._status.zero_()
