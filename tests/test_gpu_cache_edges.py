"""The paged cache's calls on the GPU where a batch is padded, indexes lie outside the cache, or a call is large."""
import sys

import pytest
import torch

from attn_cases import DEV, U, dense, generator, make_attention, make_problem, poison, randn, rotated
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


def test_slots_report_pages_that_no_sequence_has(gpu_device):
    """A token whose page-table entry is not a page of the cache gets no slot of it (``write`` stores nothing) and
    is reported; padding, and entries that no token needs, are not.  In a captured graph as well."""
    announce("slots of unallocated pages")
    attn = make_attention(2, 1, 64, "bf16", 64, 9)
    poison(attn)
    table = torch.tensor([[7, 2, -1], [0, -1, 9]], dtype=torch.int32, device=DEV)
    seqs = torch.tensor([0, 0, 1, 1, 0], device=DEV)
    fine = torch.tensor([3, 64, 63, -1, -130], device=DEV)
    attn.slots(table, seqs, fine)
    attn.check_status()
    g = generator(2)
    q, k, v = randn(g, 5, 2, 64), randn(g, 5, 1, 64), randn(g, 5, 1, 64)
    rope = rope_table(256, 64, 1e4, DEV)
    positions = fine.clone()
    positions[3] = 70
    slots = attn.slots(table, seqs, positions)
    attn.write(q, k, v, positions, slots, rope)
    assert attn.status() == {name: name == "bad_page" for name in N.ATTN_STATUS}
    with pytest.raises(N.NativeError, match="bad_page"):
        attn.check_status()
    attn.check_status()
    every = torch.arange(9 * 64, device=DEV)
    stored = ~torch.isnan(dense(attn, every)[0]).flatten(1).any(dim=1)
    assert every[stored].tolist() == [63, 2 * 64, 7 * 64 + 3]
    for at in (130, -2):
        positions[3] = at  # a page past the cache; padding
        attn.slots(table, seqs, positions)
        assert attn.status()["bad_page"] == (at > 0)
        attn._status.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = attn.slots(table, seqs, positions)
    for at, bad in ((70, True), (5, False), (-1, False), (69, True)):
        positions[3] = at
        graph.replay()
        assert attn.status()["bad_page"] == bad, at
        attn._status.zero_()
        assert torch.equal(held, attn.slots(table, seqs, positions))
        attn._status.zero_()


def test_keep_takes_64_bit_indexes_for_what_they_are(gpu_device):
    """Kept indexes, counts, contexts and pages that 32 bits do not hold are out of range and reported, not what
    their lower half says."""
    announce("keep: 64-bit indexes")
    for which, bit in (("table", "bad_page"), ("context", "bad_kept"), ("kept", "bad_kept"), ("counts", "bad_kept")):
        p = make_problem([100, 100], heads=4, kv_heads=2, dim=64, fmt="int8", page=64, seed=1, width=2)
        args = {"table": p.table.long(), "context": torch.tensor([20, 20], device=DEV),
                "kept": torch.tensor([[1, 3], [2, 5]], device=DEV), "counts": torch.tensor([2, 2], device=DEV)}
        args[which][(0,) * args[which].dim()] += 1 << 32
        p.attn.keep(args["table"], args["context"], args["kept"], args["counts"])
        st = p.attn.status()
        assert st == {name: name == bit for name in N.ATTN_STATUS}, which
        # the second sequence is not affected; of the first, what is out of range is not moved
        moved = [{} if which in ("table", "context") else {1: 3} if which == "kept" else {0: 1, 1: 3}, {0: 2, 1: 5}]
        for b, m in enumerate(moved):
            at = torch.arange(100, device=DEV)
            index = at.clone()
            for to, src in m.items():
                index[20 + to] = 20 + src
            k, v = dense(p.attn, p.attn.slots(p.table, torch.full_like(at, b), at))
            assert torch.equal(k, p.k[b][index]) and torch.equal(v, p.v[b][index]), (which, b)
