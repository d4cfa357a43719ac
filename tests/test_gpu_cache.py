"""The paged cache on the GPU: head norms, rotation and the write, reading back, and keeping drafted tokens,
against the plain 64-bit implementation in attn_cases.py."""
import sys

import pytest
import torch

from attn_cases import DEV, U, dense, generator, make_attention, make_problem, poison, put, randn, rotated
from nano_ktrans_amd import rope_table
from nano_ktrans_amd import _native as N

pytestmark = pytest.mark.gpu


def announce(msg):
    sys.__stderr__.write(f"[gpu-case] {msg}\n")
    sys.__stderr__.flush()


def random_slots(g, attn, n):
    return torch.randperm(attn.num_pages * attn.page_size, generator=g, device=DEV)[:n]


def check_stored(attn, slots, want_k, spread_k, want_v):
    """The cache's rows at the slots against float64 rows (attn_cases.py has the tolerances)."""
    k, v = dense(attn, slots)
    for got, want, err in ((k, want_k, 2.0 ** -20 * spread_k), (v, want_v, torch.zeros_like(want_v))):
        if attn.cache_format == "bf16":
            bound = U * want.abs() + err * (1 + U)
        else:
            step = want.abs().amax(dim=-1, keepdim=True) / 127
            bound = step * (0.5 + 2.0 ** -15) + err
        assert bool(((got - want).abs() <= bound + 2.0 ** -130).all())


SHAPES = [(32, 4, 128, 64), (32, 8, 128, 128), (16, 16, 128, 256), (14, 2, 64, 64), (5, 1, 64, 128), (1, 1, 128, 64)]


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
@pytest.mark.parametrize("heads,kv_heads,dim,page", SHAPES)
@pytest.mark.parametrize("tokens,run,norm", [(1, False, True), (7, False, False), (64, True, True), (333, True, False),
                                             (200, False, True)])
def test_write(gpu_device, heads, kv_heads, dim, page, fmt, tokens, run, norm):
    """Consecutive slots (from an odd offset, so that pieces of the value layout are cut on both sides) and
    scattered ones; q, k and v as parts of one projection's output; padding tokens; far positions."""
    announce(f"write {heads}/{kv_heads}/{dim} page {page} {fmt} T={tokens} run={run} norm={norm}")
    g = generator(tokens * 7 + heads)
    attn = make_attention(heads, kv_heads, dim, fmt, page, 12)
    poison(attn)
    qkv = randn(g, tokens, (heads + 2 * kv_heads) * dim)
    q, k, v = (x.unflatten(1, (-1, dim)) for x in qkv.split([heads * dim, kv_heads * dim, kv_heads * dim], dim=1))
    slots = (page - 5) + torch.arange(tokens, device=DEV) if run else random_slots(g, attn, tokens)
    if tokens > 6:
        slots[3] = -1
        slots[tokens - 1] = -7
    rope = rope_table(131072, dim, 1e6, DEV)
    positions = torch.randint(0, 131072, (tokens,), generator=g, device=DEV)
    positions[0] = 131071
    weights = {"q_norm": 1 + 0.1 * randn(g, dim), "k_norm": 1 + 0.1 * randn(g, dim)} if norm else {}
    before = [x.clone() for x in (attn.k_cache, attn.v_cache)]
    out = attn.write(q, k, v, positions, slots, rope, **weights)
    assert not any(attn.status().values())
    rows = rope[positions]
    want_q, spread = rotated(q, weights.get("q_norm"), 1e-6, rows)
    assert bool(((out.double() - want_q).abs() <= U * want_q.abs() + 2.0 ** -20 * spread * (1 + U)).all())
    want_k, spread_k = rotated(k, weights.get("k_norm"), 1e-6, rows)
    on = slots >= 0
    check_stored(attn, slots[on], want_k[on], spread_k[on], v.double()[on])
    # nothing else was touched
    every = torch.arange(attn.num_pages * page, device=DEV)
    other = every[~torch.isin(every, slots[on])]
    at, r, unit = torch.div(other, page, rounding_mode="floor"), other % page, attn.v_cache.shape[4]
    as_int = torch.int16 if fmt == "bf16" else torch.int8
    assert torch.equal(attn.k_cache[at, :, r].view(as_int), before[0][at, :, r].view(as_int))
    vi = torch.div(r, unit, rounding_mode="floor"), r % unit
    assert torch.equal(attn.v_cache[at, :, vi[0], :, vi[1]].view(as_int), before[1][at, :, vi[0], :, vi[1]].view(as_int))
    # in place, and from contiguous copies: the same bits
    q2 = q.contiguous()
    same = attn.write(q2, k.contiguous(), v.contiguous(), positions.int(), slots, rope, out=q2, **weights)
    assert same.data_ptr() == q2.data_ptr() and torch.equal(same, out)


def test_write_takes_unaligned_views(gpu_device):
    """Rows 2 bytes off and odd token strides are copied first, not read wrongly."""
    announce("write from odd strides and addresses")
    g = generator(3)
    attn = make_attention(4, 2, 64, "bf16", 64, 4)
    rope = rope_table(64, 64, 1e4, DEV)
    flat = randn(g, 9, 8 * 64 + 1)
    views = flat[:, 1:257].unflatten(1, (4, 64)), flat[:, 257:385].unflatten(1, (2, 64)), flat[:, 385:].unflatten(1, (2, 64))
    pos, slots = torch.arange(9, device=DEV), torch.arange(9, device=DEV) + 30
    got = attn.write(*views, pos, slots, rope)
    k, v = attn.read(slots)
    want = attn.write(*(x.contiguous() for x in views), pos, slots, rope)
    assert torch.equal(got, want)
    assert torch.equal(v, views[2]) and all(torch.equal(a, b) for a, b in zip(attn.read(slots), (k, v)))


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
def test_write_special_rows(gpu_device, fmt):
    """Rows of zeros, of one large value, of tiny values, with an infinity and with a NaN: each row on its own."""
    announce(f"write special rows {fmt}")
    attn = make_attention(2, 1, 64, fmt, 64, 2)
    rope = rope_table(8, 64, 1e4, DEV)
    g = generator(11)
    rows = randn(g, 8, 1, 64)
    rows[0] = 0
    rows[1] = 0
    rows[1, 0, 5] = 3e38
    rows[2] *= 1e-30
    rows[3, 0, 7] = float("inf")
    rows[4, 0, 9] = float("nan")
    rows[5] = -rows[5].abs()
    zero = torch.zeros(8, dtype=torch.int64, device=DEV)  # position 0: no rotation
    slots = torch.arange(8, device=DEV)
    attn.write(torch.zeros(8, 2, 64, dtype=torch.bfloat16, device=DEV), rows, rows, zero, slots, rope)
    for got in attn.read(slots):
        for i in (0, 1, 2, 5, 6, 7):
            want = rows[i].double()
            step = want.abs().amax() / 127 if fmt == "int8" else 0.0
            assert bool(((got[i].double() - want).abs() <= step * (0.5 + 2.0 ** -15) + U * (want.abs() + step)).all()), i
        if fmt == "bf16":
            # (a key's infinity also meets the sine of 0: its pair is NaN)
            assert not bool(torch.isfinite(got[3, 0, 7])) and not bool(torch.isfinite(got[4, 0, 9]))
            assert int(torch.isfinite(got[3]).sum()) >= 62 and int(torch.isfinite(got[4]).sum()) >= 62
        else:
            assert bool(torch.isnan(got[3]).all()) and bool(torch.isnan(got[4]).all())


@pytest.mark.parametrize("largest", [127 * 2.0 ** -133, 2.0 ** -126, 1.2e-38, 3e-37, 1e-20])
def test_write_tiny_rows_to_int8(gpu_device, largest):
    """Rows whose scale, or its reciprocal, is outside fp32's normal range.  The scale is max / 127 to fp32's
    denormal step, 2^-149, so codes up to 127 are off by that many of them beside the half step."""
    announce(f"write tiny rows {largest}")
    attn = make_attention(2, 1, 64, "int8", 64, 1)
    rows = (torch.linspace(-1, 1, 64, dtype=torch.float64) * largest).to(torch.bfloat16).view(1, 1, 64).to(DEV)
    slots = torch.arange(1, device=DEV)
    attn.write(torch.zeros(1, 2, 64, dtype=torch.bfloat16, device=DEV), rows, rows, torch.zeros_like(slots), slots,
               rope_table(1, 64, 1e4, DEV))
    want = rows[0].double()
    for got in dense(attn, slots):
        step = want.abs().amax() / 127
        assert bool(((got[0] - want).abs() <= step * (0.5 + 2.0 ** -15) + 2.0 ** -142).all())


def test_write_reports_bad_slots_and_positions(gpu_device):
    announce("write: bad slots and positions")
    attn = make_attention(4, 2, 128, "int8", 64, 3)
    poison(attn)
    g = generator(5)
    q, k, v = randn(g, 6, 4, 128), randn(g, 6, 2, 128), randn(g, 6, 2, 128)
    rope = rope_table(100, 128, 1e4, DEV)
    pos = torch.tensor([1, 2, 3, 100, -1, 99], device=DEV)
    slots = torch.tensor([0, 3 * 64, 1 << 40, 7, 8, 191], device=DEV)
    out = attn.write(q, k, v, pos, slots, rope)
    st = attn.status()
    assert st["bad_slot"] and st["bad_position"] and not st["bad_page"]
    with pytest.raises(N.NativeError, match="bad_slot"):
        attn.check_status()
    attn.check_status()
    assert bool((out[3:5] == 0).all())
    ok = torch.tensor([0, 5], device=DEV)
    want, spread = rotated(k, None, 0, rope[pos.clamp(0, 99)])
    check_stored(attn, slots[ok], want[ok], spread[ok], v.double()[ok])
    stored = torch.isfinite(attn.k_scales[:, 0].reshape(-1)).nonzero().flatten().tolist()
    assert stored == [0, 191] and torch.isfinite(attn.v_scales[:, 1].reshape(-1)).nonzero().flatten().tolist() == [0, 191]


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(32, 4, 128, 64), (16, 16, 128, 256), (5, 1, 64, 128)])
@pytest.mark.parametrize("n,run", [(1, False), (15, True), (64, True), (700, True), (129, False)])
def test_read(gpu_device, heads, kv_heads, dim, page, fmt, n, run):
    """Runs and scattered slots, repeated ones, and negative ones (zeros)."""
    announce(f"read {kv_heads}/{dim} page {page} {fmt} n={n} run={run}")
    g = generator(n)
    attn = make_attention(heads, kv_heads, dim, fmt, page, 12)
    every = torch.arange(12 * page, device=DEV)
    put(attn, every, randn(g, 12 * page, kv_heads, dim).float(), randn(g, 12 * page, kv_heads, dim).float())
    slots = (3 + torch.arange(n, device=DEV)) if run else random_slots(g, attn, n)
    if n > 20:
        slots[5] = -1
        slots[9] = slots[2]
        slots[11] = slots[12]
    got = attn.read(slots)
    want = dense(attn, slots.clamp(min=0))
    for a, b in zip(got, want):
        b = torch.where((slots >= 0).view(-1, 1, 1), b, 0.0)
        assert torch.equal(a, b.to(torch.float32).to(torch.bfloat16))  # one product in fp32 (24 bits hold it), one rounding
    assert not any(attn.status().values())
    bad = slots.clone()
    bad[0] = 12 * page
    assert bool((attn.read(bad)[0][0] == 0).all()) and attn.status()["bad_slot"]


def test_slots(gpu_device):
    """Padding positions, and positions and sequences that the page table does not have."""
    attn = make_attention(2, 1, 64, "bf16", 64, 9)
    table = torch.tensor([[7, 2], [0, -1]], dtype=torch.int32, device=DEV)
    seqs = torch.tensor([0, 0, 1, 1, 0, 1, 2, -1], device=DEV)
    positions = torch.tensor([3, 64, 63, 70, 128, -1, 0, 0], dtype=torch.int32, device=DEV)
    past = 9 * 64
    want = [7 * 64 + 3, 2 * 64, 63, -64 + 6, past, -1, past, past]
    assert attn.slots(table, seqs, positions).tolist() == want
    assert attn.slots(table[:, :0], seqs, positions).tolist() == [past] * 5 + [-1, past, past]


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
@pytest.mark.parametrize("page", [64, 256])
def test_keep(gpu_device, fmt, page):
    """Drafts of several sizes, of which some, all or none are kept; contexts that end inside a page; a draft
    that crosses pages; everything else stays as it was."""
    announce(f"keep {fmt} page {page}")
    drafts, contexts = [12, 70, 5, 64, 1, 40], [page - 3, 130, 0, 2 * page, 77, page - 20]
    kept = [[0, 3, 4, 9], list(range(1, 70)), [], list(range(64)), [0], [7, 8, 39]]
    lengths = [c + n for c, n in zip(contexts, drafts)]
    p = make_problem(lengths, heads=8, kv_heads=2, dim=128, fmt=fmt, page=page, seed=page, width=5)
    width = max(len(x) for x in kept)
    rows = torch.full((6, width), 1 << 20, dtype=torch.int32)
    for b, x in enumerate(kept):
        rows[b, :len(x)] = torch.tensor(x, dtype=torch.int32)
    counts = torch.tensor([len(x) for x in kept], dtype=torch.int64, device=DEV)
    p.attn.keep(p.table, torch.tensor(contexts, device=DEV), rows.to(DEV), counts)
    assert not any(p.attn.status().values())
    for b, (c, x) in enumerate(zip(contexts, kept)):
        at = torch.arange(lengths[b], device=DEV)
        k, v = dense(p.attn, p.attn.slots(p.table, torch.full_like(at, b), at))
        index = at.clone()
        index[c:c + len(x)] = c + torch.tensor(x, dtype=torch.int64, device=DEV)
        assert torch.equal(k, p.k[b][index]) and torch.equal(v, p.v[b][index]), b


def test_keep_reports_what_it_leaves_out(gpu_device):
    announce("keep: bad kept indices, counts and pages")
    p = make_problem([100, 100, 100, 100], heads=4, kv_heads=2, dim=64, fmt="int8", page=64, seed=1, width=2)
    table = p.table.clone()
    table[2, 1] = -3
    table[3, 1] = p.attn.num_pages
    kept = torch.tensor([[1, 0, 200, 5], [0, 2, 3, 4], [0, 35, 50, 60], [1, 2, 3, 45]], dtype=torch.int32, device=DEV)
    counts = torch.tensor([4, 9, 4, 4], dtype=torch.int32, device=DEV)
    context = torch.tensor([20, 20, 20, 20], dtype=torch.int32, device=DEV)
    p.attn.keep(table, context, kept, counts)
    st = p.attn.status()
    assert st["bad_kept"] and st["bad_page"] and not st["bad_slot"]
    moved = [{0: 1, 3: 5}, {1: 2, 2: 3, 3: 4}, {1: 35}, {0: 1, 1: 2, 2: 3}]  # 35 + 20 < 64: the page before
    for b, m in enumerate(moved):
        at = torch.arange(100, device=DEV)
        index = at.clone()
        for to, src in m.items():
            index[20 + to] = 20 + src
        k, v = dense(p.attn, p.attn.slots(p.table, torch.full_like(at, b), at))
        assert torch.equal(k, p.k[b][index]) and torch.equal(v, p.v[b][index]), b


def test_write_and_read_past_32_bit_offsets(gpu_device):
    """A cache of more than 4 GiB per tensor: the first, the last and some middle pages."""
    announce("cache past 4 GiB")
    g = generator(9)
    attn = make_attention(8, 8, 128, "bf16", 256, 10000)  # 5.2 GB of keys, as much of values
    slots = torch.cat([torch.arange(40, device=DEV) + at for at in (0, 8191 * 256 + 250, 8192 * 256 + 100,
                                                                     10000 * 256 - 40)])
    n = slots.numel()
    k, v = randn(g, n, 8, 128), randn(g, n, 8, 128)
    attn.write(randn(g, n, 8, 128), k, v, torch.zeros(n, dtype=torch.int64, device=DEV), slots,
               rope_table(4, 128, 1e4, DEV))
    got = attn.read(slots)
    assert torch.equal(got[0], k) and torch.equal(got[1], v)  # position 0 turns by nothing


def test_refusals(gpu_device):
    attn = make_attention(8, 2, 128, "bf16", 64, 4)
    g = generator(1)
    q, k, v = randn(g, 3, 8, 128), randn(g, 3, 2, 128), randn(g, 3, 2, 128)
    pos = torch.zeros(3, dtype=torch.int64, device=DEV)
    rope = rope_table(8, 128, 1e4, DEV)
    good = dict(q=q, k=k, v=v, positions=pos, slots=pos, rope=rope)
    for bad in (dict(q=q.float()), dict(q=q[:, :4]), dict(k=k[:2]), dict(v=v.cpu()), dict(positions=pos.float()),
                dict(slots=pos[:2]), dict(rope=rope.double()), dict(rope=rope[:, :64]), dict(q_norm=pos),
                dict(out=q.float()), dict(out=q[:2]), dict(rope=rope.cpu())):
        with pytest.raises(ValueError):
            attn.write(**{**good, **bad})
    for bad in (torch.zeros(3, device=DEV), torch.zeros(2, 2, dtype=torch.int64, device=DEV), pos.cpu()):
        with pytest.raises(ValueError):
            attn.read(bad)
    table = torch.zeros(2, 2, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError):
        attn.keep(table, pos, table, pos[:2])
    with pytest.raises(ValueError):
        attn.keep(table, pos[:2], pos[:2], pos[:2])
    with pytest.raises(ValueError, match="cache_format"):
        make_attention(8, 2, 128, "int4", 64, 4)
    with pytest.raises(N.NativeError, match="head_dim"):
        make_attention(8, 2, 96, "bf16", 64, 4)
    # nothing to do is no error
    assert attn.write(q[:0], k[:0], v[:0], pos[:0], pos[:0], rope).shape == (0, 8, 128)
    assert attn.read(pos[:0])[0].shape == (0, 2, 128)
    attn.keep(table[:0], pos[:0], table[:0], pos[:0])


def test_another_stream_and_a_captured_graph(gpu_device):
    """Write and read captured together, replayed on new inputs, with eager work between the replays; and on
    another stream than the default one."""
    announce("cache calls in a graph")
    g = generator(21)
    attn = make_attention(8, 2, 128, "int8", 64, 8)
    rope = rope_table(512, 128, 1e4, DEV)
    T = 24
    q, k, v = randn(g, T, 8, 128), randn(g, T, 2, 128), randn(g, T, 2, 128)
    pos, slots = torch.arange(T, device=DEV), torch.arange(T, device=DEV) + 50
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = attn.write(q, k, v, pos, slots, rope), *attn.read(slots)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = attn.write(q, k, v, pos, slots, rope), *attn.read(slots)
    for i in range(4):
        fresh = [randn(g, *x.shape) for x in (q, k, v)]
        for x, y in zip((q, k, v), fresh):
            x.copy_(y)
        slots.copy_(torch.arange(T, device=DEV) + 3 * i)
        other = attn.write(*fresh, pos, slots + 200, rope), *attn.read(slots + 200)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, other)), i
    assert all(torch.isfinite(x).all() for x in first)
