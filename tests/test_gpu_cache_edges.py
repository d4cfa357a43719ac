"""The paged cache's calls on the GPU where a batch is padded, indexes lie outside the cache, or a call is large."""
import sys

import pytest
import torch

from attn_cases import DEV, U, dense, generator, make_attention, make_problem, poison, put, randn, rotated
from nano_ktrans_amd import rope_table
from nano_ktrans_amd import _native as N
from test_gpu_cache import check_stored, random_slots

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


SHAPES = [(32, 4, 128, 64), (16, 16, 128, 256), (14, 2, 64, 64), (5, 1, 64, 128), (1, 1, 128, 64), (6, 3, 128, 128),
          (2, 1, 64, 64)]


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
@pytest.mark.parametrize("heads,kv_heads,dim,page", SHAPES)
@pytest.mark.parametrize("tokens,run,norm", [(1024, True, False), (1025, True, True), (1100, False, False), (1337, True, False)])
def test_write_of_many_tokens(gpu_device, heads, kv_heads, dim, page, fmt, tokens, run, norm):
    """On both sides of the size from which a launch takes wide windows and four heads at a time (whose number
    need not be a multiple of four): runs of slots from an odd offset, broken by padding and by swapped tokens, and
    scattered slots; a last window of any size."""
    announce(f"write {heads}/{kv_heads}/{dim} page {page} {fmt} T={tokens} run={run} norm={norm}")
    g = generator(tokens + heads)
    attn = make_attention(heads, kv_heads, dim, fmt, page, 1536 // page + 1)
    poison(attn)
    qkv = randn(g, tokens, (heads + 2 * kv_heads) * dim)
    q, k, v = (x.unflatten(1, (-1, dim)) for x in qkv.split([heads * dim, kv_heads * dim, kv_heads * dim], dim=1))
    slots = (page - 5) + torch.arange(tokens, device=DEV) if run else random_slots(g, attn, tokens)
    slots[[100, 101, 700]] = slots[[101, 100, 640]]
    slots[[3, 640, tokens - 1]] = -1
    slots[tokens - 2] = -7
    rope = rope_table(131072, dim, 1e6, DEV)
    positions = torch.randint(0, 131072, (tokens,), generator=g, device=DEV)
    weights = {"q_norm": 1 + 0.1 * randn(g, dim), "k_norm": 1 + 0.1 * randn(g, dim)} if norm else {}
    before = [x.clone() for x in (attn.k_cache, attn.v_cache)]
    out = attn.write(q, k, v, positions, slots, rope, **weights)
    assert not any(attn.status().values())
    rows = rope[positions]
    want, spread = rotated(q, weights.get("q_norm"), 1e-6, rows)
    assert bool(((out.double() - want).abs() <= U * want.abs() + 2.0 ** -20 * spread * (1 + U)).all())
    want, spread = rotated(k, weights.get("k_norm"), 1e-6, rows)
    on = slots >= 0
    check_stored(attn, slots[on], want[on], spread[on], v.double()[on])
    every = torch.arange(attn.num_pages * page, device=DEV)
    other = every[~torch.isin(every, slots[on])]
    at, r, unit = torch.div(other, page, rounding_mode="floor"), other % page, attn.v_cache.shape[4]
    as_int = torch.int16 if fmt == "bf16" else torch.int8
    assert torch.equal(attn.k_cache[at, :, r].view(as_int), before[0][at, :, r].view(as_int))
    vi = torch.div(r, unit, rounding_mode="floor"), r % unit
    assert torch.equal(attn.v_cache[at, :, vi[0], :, vi[1]].view(as_int), before[1][at, :, vi[0], :, vi[1]].view(as_int))
    # in place: the same bits; and in calls of a few tokens each: the same cache
    held = [x.clone() for x in (attn.k_cache, attn.v_cache)]
    q2 = q.contiguous()
    assert torch.equal(attn.write(q2, k.contiguous(), v.contiguous(), positions, slots, rope, out=q2, **weights), out)
    poison(attn)
    for i in range(0, tokens, 333):
        part = slice(i, i + 333)
        few = attn.write(q[part], k[part], v[part], positions[part], slots[part], rope, **weights)
        assert torch.equal(few, out[part])
    for x, y in zip((attn.k_cache, attn.v_cache), held):
        assert torch.equal(x.view(as_int), y.view(as_int))


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
@pytest.mark.parametrize("heads,kv_heads,dim,page", SHAPES)
@pytest.mark.parametrize("n,run", [(1024, True), (1025, True), (1100, False), (1337, True)])
def test_read_of_many_slots(gpu_device, heads, kv_heads, dim, page, fmt, n, run):
    """On both sides of the size from which a launch takes wide windows: runs and scattered slots, repeated ones,
    and negative ones (zeros)."""
    announce(f"read {kv_heads}/{dim} page {page} {fmt} n={n} run={run}")
    g = generator(n)
    attn = make_attention(heads, kv_heads, dim, fmt, page, 1536 // page + 1)
    total = attn.num_pages * page
    put(attn, torch.arange(total, device=DEV), randn(g, total, kv_heads, dim).float(), randn(g, total, kv_heads, dim).float())
    slots = (3 + torch.arange(n, device=DEV)) if run else random_slots(g, attn, n)
    slots[[5, 700, n - 1]] = -1
    slots[[9, 800]] = slots[[2, 12]]
    want = dense(attn, slots.clamp(min=0))
    for a, b in zip(attn.read(slots), want):
        b = torch.where((slots >= 0).view(-1, 1, 1), b, 0.0)
        assert torch.equal(a, b.to(torch.float32).to(torch.bfloat16))  # (as in the small calls' test)
    assert not any(attn.status().values())


def test_keep_of_padding_sequences_is_no_error(gpu_device):
    """A sequence that keeps nothing may have any context (a padded batch's length less its rows is negative); one
    that keeps something of a negative context is reported and not moved."""
    announce("keep: padding sequences")
    p = make_problem([100, 100], heads=4, kv_heads=2, dim=64, fmt="bf16", page=64, seed=1, width=2)
    kept = torch.tensor([[1, 3], [2, 5]], dtype=torch.int32, device=DEV)
    for counts, bad in (([0, 2], False), ([1, 2], True)):
        p.attn.keep(p.table, torch.tensor([-4, 20], device=DEV), kept, torch.tensor(counts, device=DEV))
        assert p.attn.status() == {name: bad and name == "bad_kept" for name in N.ATTN_STATUS}
        for b, m in enumerate(({}, {0: 2, 1: 5})):
            at = torch.arange(100, device=DEV)
            index = at.clone()
            for to, src in m.items():
                index[20 + to] = 20 + src
            slots = p.attn.slots(p.table, torch.full_like(at, b), at)
            k, v = dense(p.attn, slots)
            assert torch.equal(k, p.k[b][index]) and torch.equal(v, p.v[b][index]), b
            put(p.attn, slots, p.k[b].float(), p.v[b].float())
