"""Attention over the paged cache on the GPU, against the plain 64-bit implementation in attn_cases.py: single
tokens, prompts, chunks and drafted trees, at the lengths, masks and pages where it can go wrong."""
import sys

import pytest
import torch

from attn_cases import (DEV, causal, check_attention, check_rows, dense, generator, make_attention, make_problem, put,
                        randn, reference, split_rows, tree_sees)
from nano_ktrans_amd import tree_mask_from_parents

pytestmark = pytest.mark.gpu

SHAPES = [(32, 4, 128, 64), (32, 8, 128, 128), (16, 16, 128, 256), (14, 2, 64, 64), (48, 1, 64, 128), (3, 3, 64, 64)]


def announce(msg):
    sys.__stderr__.write(f"[gpu-case] {msg}\n")
    sys.__stderr__.flush()


def starts_of(counts):
    return torch.tensor(split_rows(counts), dtype=torch.int32, device=DEV)


def random_trees(g, counts):
    parents = []
    for n in counts:
        r = torch.randint(1, 7, (max(n, 1),), generator=g, device=DEV).tolist()
        parents.append([max(-1, j - r[j]) for j in range(n)])
    return tree_mask_from_parents(parents, DEV)


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
@pytest.mark.parametrize("heads,kv_heads,dim,page", SHAPES)
def test_single_tokens(gpu_device, heads, kv_heads, dim, page, fmt):
    """One row per sequence; lengths from 0 and 1 to several pages, around the ends of pages and tiles."""
    announce(f"decode {heads}/{kv_heads}/{dim} page {page} {fmt}")
    lengths = [1, 0, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 300, 511, 1025]
    p = make_problem(lengths, heads=heads, kv_heads=kv_heads, dim=dim, fmt=fmt, page=page, seed=heads)
    q = randn(generator(1), len(lengths), heads, dim)
    check_attention(p, None, q, p.attn.forward(q, p.table, p.lens))
    # tighter bounds on the lengths choose another launch; other integer types are taken too
    check_attention(p, None, q, p.attn.forward(q, p.table.long(), p.lens.long(), max_seq_len=1025))
    check_attention(p, None, q, p.attn.forward(q, p.table, p.lens, starts_of([1] * len(lengths)), max_queries=1))
    assert not any(p.attn.status().values())


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
@pytest.mark.parametrize("heads,kv_heads,lengths", [(32, 4, [20011]), (16, 16, [9000, 1, 4097]), (32, 8, [6000] * 3 + [70])])
def test_single_tokens_long(gpu_device, heads, kv_heads, lengths, fmt):
    """Contexts that are split over workgroups and joined; short ones beside them."""
    announce(f"decode long {heads}/{kv_heads} {lengths} {fmt}")
    p = make_problem(lengths, heads=heads, kv_heads=kv_heads, dim=128, fmt=fmt, page=128, seed=3)
    q = randn(generator(2), len(lengths), heads, 128)
    got = p.attn.forward(q, p.table, p.lens)
    check_attention(p, None, q, got)
    assert torch.equal(got, p.attn.forward(q, p.table, p.lens))


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
@pytest.mark.parametrize("heads,kv_heads,dim,page", SHAPES)
@pytest.mark.parametrize("counts,contexts", [
    ([1, 2, 3], [0, 62, 200]),                  # a few rows per sequence
    ([17, 0, 64, 5], [0, 9, 0, 130]),           # one without rows
    ([130, 33], [0, 95]),
    ([257], [70]),
])
def test_prompts_and_chunks(gpu_device, heads, kv_heads, dim, page, fmt, counts, contexts):
    announce(f"causal {heads}/{kv_heads}/{dim} page {page} {fmt} rows {counts} contexts {contexts}")
    lengths = [n + c for n, c in zip(counts, contexts)]
    p = make_problem(lengths, heads=heads, kv_heads=kv_heads, dim=dim, fmt=fmt, page=page, seed=sum(counts))
    q = randn(generator(4), sum(counts), heads, dim)
    got = p.attn.forward(q, p.table, p.lens, starts_of(counts))
    check_attention(p, counts, q, got)
    tight = p.attn.forward(q, p.table, p.lens, starts_of(counts), max_queries=max(counts), max_seq_len=max(lengths))
    check_attention(p, counts, q, tight)
    assert not any(p.attn.status().values())


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
@pytest.mark.parametrize("counts,contexts", [([1500], [0]), ([700, 40], [1300, 3000]), ([48], [20000])])
def test_long_prompts(gpu_device, fmt, counts, contexts):
    announce(f"causal long {fmt} rows {counts} contexts {contexts}")
    lengths = [n + c for n, c in zip(counts, contexts)]
    p = make_problem(lengths, heads=8, kv_heads=2, dim=128, fmt=fmt, page=64, seed=5)
    q = randn(generator(5), sum(counts), 8, 128)
    got = p.attn.forward(q, p.table, p.lens, starts_of(counts), max_queries=max(counts), max_seq_len=max(lengths))
    check_attention(p, counts, q, got)


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
@pytest.mark.parametrize("heads,kv_heads,dim,page", SHAPES)
@pytest.mark.parametrize("counts,contexts", [([1, 5, 12], [30, 0, 700]), ([64, 65, 3], [64, 61, 10]), ([150], [90])])
def test_trees(gpu_device, heads, kv_heads, dim, page, fmt, counts, contexts):
    announce(f"tree {heads}/{kv_heads}/{dim} page {page} {fmt} rows {counts} contexts {contexts}")
    lengths = [n + c for n, c in zip(counts, contexts)]
    p = make_problem(lengths, heads=heads, kv_heads=kv_heads, dim=dim, fmt=fmt, page=page, seed=sum(counts) + 1)
    g = generator(6)
    q, mask = randn(g, sum(counts), heads, dim), random_trees(g, counts)
    got = p.attn.forward_tree(q, mask, p.table, p.lens, starts_of(counts), max_queries=max(counts))
    check_attention(p, counts, q, got, mask)
    assert torch.equal(got, p.attn.forward_tree(q, mask, p.table, p.lens, starts_of(counts), max_queries=max(counts)))
    # a chain is causal attention
    chain = tree_mask_from_parents([list(range(-1, n - 1)) for n in counts], DEV)
    check_attention(p, counts, q, p.attn.forward_tree(q, chain, p.table, p.lens, starts_of(counts)))


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lengths", [[5, 31, 33, 64, 65, 100, 129, 4], [9, 700, 64, 2049, 90, 127, 6, 40],
                                     [6100, 5, 3000, 20]])
def test_few_rows(gpu_device, fmt, dim, lengths):
    """17 to 64 rows per sequence (and sequences of none, and with more rows than tokens beside them): drafts
    and causal rows, alone and in parts."""
    counts = [5, 16, 1, 8, 13, 0, 7, 3][:len(lengths)]
    announce(f"few rows {fmt} dim {dim} rows {counts} of {lengths}")
    p = make_problem(lengths, heads=8, kv_heads=2, dim=dim, fmt=fmt, page=64, seed=sum(lengths))
    g = generator(len(lengths))
    q = randn(g, sum(counts), 8, dim)
    mask = random_trees(g, counts)
    for most in (16, None):  # 64 rows bound the launch, then the whole batch's
        check_attention(p, counts, q, p.attn.forward(q, p.table, p.lens, starts_of(counts), max_queries=most))
        check_attention(p, counts, q, p.attn.forward_tree(q, mask, p.table, p.lens, starts_of(counts), max_queries=most),
                        mask)
    assert not any(p.attn.status().values())


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
def test_tree_rows_that_see_nothing(gpu_device, fmt):
    """Masks with empty rows and no context (zeros), without the row's own bit, with bits past the draft,
    and masks shorter than the draft."""
    announce(f"tree: empty rows {fmt}")
    counts, lengths = [4, 70, 3], [4, 70, 90]
    p = make_problem(lengths, heads=8, kv_heads=2, dim=128, fmt=fmt, page=64, seed=2)
    q = randn(generator(7), 77, 8, 128)
    mask = torch.zeros(77, 2, dtype=torch.int64, device=DEV)
    mask[1, 0] = 0b1000
    mask[2, 0] = -1
    mask[2, 1] = -1
    mask[4 + 5, 1] = 0b100000
    mask[4 + 6, 1] = 0b1111000000
    mask[4 + 69, 0] = -1 << 63
    got = p.attn.forward_tree(q, mask, p.table, p.lens, starts_of(counts))
    check_attention(p, counts, q, got, mask)
    assert bool((got[0] == 0).all()) and bool((got[3] == 0).all()) and bool((got[4:9] == 0).all())
    assert bool((got[1] != 0).any()) and bool((got[74:] != 0).any())
    short = mask[:, :1].contiguous()
    check_attention(p, counts, q, p.attn.forward_tree(q, short, p.table, p.lens, starts_of(counts)), short)
    one = torch.tensor([0b1, 0], dtype=torch.int64, device=DEV).view(2, 1)  # one drafted token per sequence
    two = make_problem([1, 1], heads=8, kv_heads=2, dim=128, fmt=fmt, page=64, seed=2)
    got = two.attn.forward_tree(q[:2], one, two.table, two.lens)
    check_attention(two, None, q[:2], got, one)
    assert bool((got[1] == 0).all())


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
@pytest.mark.parametrize("counts", [[1, 1], [16, 5], [20, 5], [90, 130]])
def test_unseen_tokens_do_not_reach_a_row(gpu_device, fmt, counts):
    """NaN and infinities in later tokens (causal) and in unseen branches (trees): the rows that do not see
    them keep their bits; the rows that do are NaN or infinite as the formula's."""
    announce(f"unseen NaN and infinities {fmt} rows {counts}")
    lengths = [counts[0] + 37, counts[1] + 130]
    p = make_problem(lengths, heads=8, kv_heads=2, dim=128, fmt=fmt, page=64, seed=8)
    g = generator(9)
    q = randn(g, sum(counts), 8, 128)
    starts = starts_of(counts)
    clean = p.attn.forward(q, p.table, p.lens, starts)
    mask = random_trees(g, counts)
    clean_tree = p.attn.forward_tree(q, mask, p.table, p.lens, starts)
    for b, (n, length) in enumerate(zip(counts, lengths)):
        at = torch.tensor([length - 1, length - 1 - n // 2], device=DEV)
        slots = p.attn.slots(p.table, torch.full_like(at, b), at)
        page, r, unit = torch.div(slots, 64, rounding_mode="floor"), slots % 64, p.attn.v_cache.shape[4]
        if fmt == "bf16":
            p.attn.v_cache[page[0], 0, r[0] // unit, 3, r[0] % unit] = float("nan")
            p.attn.v_cache[page[1], :, r[1] // unit, 70, r[1] % unit] = float("inf")
            p.attn.k_cache[page[0], 1, r[0], 5] = float("inf")
        else:
            p.attn.v_scales[page[0], 0, r[0]] = float("nan")
            p.attn.v_scales[page[1], :, r[1]] = float("inf")
            p.attn.k_scales[page[0], 1, r[0]] = float("nan")
        every = torch.arange(length, device=DEV)
        p.k[b], p.v[b] = dense(p.attn, p.attn.slots(p.table, torch.full_like(every, b), every))
    for clean_out, m in ((clean, None), (clean_tree, mask)):
        got = p.attn.forward(q, p.table, p.lens, starts) if m is None else \
            p.attn.forward_tree(q, m, p.table, p.lens, starts)
        at = split_rows(counts)
        for b, (n, length) in enumerate(zip(counts, lengths)):
            rows = slice(at[b], at[b + 1])
            sees = causal(n, length) if m is None else tree_sees(m[rows], n, length)
            hit = sees[:, length - 1] | sees[:, length - 1 - n // 2]
            assert torch.equal(got[rows][~hit], clean_out[rows][~hit]), f"sequence {b}: an unseen token came through"
            touched = ~torch.isfinite(got[rows]).flatten(1).all(dim=1)
            assert torch.equal(touched, hit), f"sequence {b}"
            if fmt == "bf16":  # only dimension 3 of head group 0, dimension 70, and head group 1's infinite scores
                off = ~torch.isfinite(got[rows][:, :4])
                off[:, :, [3, 70]] = False
                assert not bool(off.any())


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
def test_large_scores(gpu_device, fmt):
    """Scores of hundreds: a softmax whose maximum moves by far along the tokens, ascending and descending."""
    announce(f"large scores {fmt}")
    lengths = [700, 700]
    p = make_problem(lengths, heads=8, kv_heads=2, dim=128, fmt=fmt, page=64, seed=12)
    ramp = torch.linspace(0.1, 6.0, 700, device=DEV)
    g = generator(13)
    base = randn(g, 1, 2, 128).float()
    for b, r in enumerate((ramp, ramp.flip(0))):
        at = torch.arange(700, device=DEV)
        slots = p.attn.slots(p.table, torch.full_like(at, b), at)
        put(p.attn, slots, base * r.view(-1, 1, 1), randn(g, 700, 2, 128).float())
        p.k[b], p.v[b] = dense(p.attn, slots)
    q = torch.cat([base.repeat_interleave(4, dim=1)] * 4).to(torch.bfloat16) * 8
    got = p.attn.forward(q, p.table, p.lens, starts_of([2, 2]))
    # the same rows in the launch for more of them: each form within the bounds below of the same values
    other = p.attn.forward(torch.cat([q[:1].expand(8, -1, -1), q[:2], q[2:3].expand(6, -1, -1), q[2:]]), p.table, p.lens,
                           starts_of([10, 8]))
    # scores up to 8 * 6 * |base|^2 / sqrt(128) ~ 550 with one sign: an fp32 score is off by 2^-24 * 136 * 550
    # (2^-7.8 would come out of a sum of 128 such roundings; they add as a walk: 2^-24 * 12 * 550 * 4 < 2^-9)
    for b in range(2):
        want, A = reference(q[2 * b:2 * b + 2], p.k[b], p.v[b], causal(2, 700), p.attn.scale)
        for x in (got[2 * b:2 * b + 2], other[[8, 9] if b == 0 else [16, 17]]):
            assert bool(((x.double() - want).abs() <= (2 * 2.0 ** -8 + 2.0 ** -7) * A).all())


def test_rows_behind_the_last_sequence_stay(gpu_device):
    """A padded batch: rows of q behind the last sequence keep what out held."""
    announce("padded batch")
    p = make_problem([80, 9], heads=8, kv_heads=2, dim=128, fmt="bf16", page=64, seed=14)
    q = randn(generator(15), 40, 8, 128)
    for counts in ([3, 2], [30, 9], [1, 1]):
        out = torch.full_like(q, 7.0)
        got = p.attn.forward(q, p.table, p.lens, starts_of(counts), out=out)
        assert got.data_ptr() == out.data_ptr()
        check_attention(p, counts, q, got)
        assert bool((out[sum(counts):] == 7.0).all())
        mask = tree_mask_from_parents([list(range(-1, n - 1)) for n in counts + [40 - sum(counts)]], DEV)
        out = torch.full_like(q, 7.0)
        check_attention(p, counts, q, p.attn.forward_tree(q, mask, p.table, p.lens, starts_of(counts), out=out))
        assert bool((out[sum(counts):] == 7.0).all())


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
@pytest.mark.parametrize("counts,lengths", [(None, [700, 0, 3000]), ([4, 1], [2500, 9]), ([130, 0, 45], [900, 4, 2000])])
def test_in_place_of_the_queries(gpu_device, fmt, counts, lengths):
    """out = q: the same bits, with and without splits, rows behind the last sequence as they were."""
    announce(f"in place {fmt} rows {counts} of {lengths}")
    p = make_problem(lengths, heads=8, kv_heads=2, dim=64, fmt=fmt, page=64, seed=8)
    behind = 0 if counts is None else 5
    q = randn(generator(9), sum(counts or [1] * len(lengths)) + behind, 8, 64)
    starts = None if counts is None else torch.tensor(split_rows(counts), dtype=torch.int32, device=DEV)
    most = None if counts is None else max(counts)
    want = p.attn.forward(q, p.table, p.lens, starts, max_queries=most, out=q.clone())
    got = q.clone()
    p.attn.forward(got, p.table, p.lens, starts, max_queries=most, out=got)
    assert torch.equal(got, want)
    if counts is not None:
        assert torch.equal(got[sum(counts):], q[sum(counts):]) and not torch.equal(got, q)
        mask = torch.full((q.shape[0], 3), -1, dtype=torch.int64, device=DEV)
        want = p.attn.forward_tree(q, mask, p.table, p.lens, starts, max_queries=most, out=q.clone())
        p.attn.forward_tree(q, mask, p.table, p.lens, starts, max_queries=most, out=q)
        assert torch.equal(q, want)


@pytest.mark.parametrize("counts", [None, [9, 40]])
def test_bad_pages_and_lengths_are_reported(gpu_device, counts):
    """Pages outside the cache are not seen; lengths past the table are cut, negative ones nothing; rows past
    max_queries stay.  The other sequences of the batch are not affected."""
    announce(f"bad pages and lengths, rows {counts}")
    p = make_problem([200, 200], heads=8, kv_heads=2, dim=128, fmt="bf16", page=64, seed=16)
    n = counts or [1, 1]
    starts = starts_of(counts) if counts else None
    q = randn(generator(17), sum(n), 8, 128)
    good = p.attn.forward(q, p.table, p.lens, starts)
    for bad_page in (-1, p.attn.num_pages, 2 ** 31 - 1):
        table = p.table.clone()
        table[0, 1] = bad_page
        got = p.attn.forward(q, table, p.lens, starts)
        st = p.attn.status()
        assert st["bad_page"] and not st["bad_length"]
        p.attn._status.zero_()
        sees = causal(n[0], 200)
        sees[:, 64:128] = False
        want, A = reference(q[:n[0]], p.k[0], p.v[0], sees, p.attn.scale)
        check_rows(got[:n[0]], want, A)
        assert torch.equal(got[n[0]:], good[n[0]:])
    lens = torch.tensor([-5, 200], dtype=torch.int32, device=DEV)
    got = p.attn.forward(q, p.table, lens, starts)
    assert p.attn.status()["bad_length"] and bool((got[:n[0]] == 0).all()) and torch.equal(got[n[0]:], good[n[0]:])
    p.attn._status.zero_()
    lens[0] = 4 * 64 + n[0]  # past the table: every token of it, of a context that long
    got = p.attn.forward(q, p.table, lens, starts)
    assert p.attn.status()["bad_length"] and torch.equal(got[n[0]:], good[n[0]:])
    p.attn._status.zero_()
    got = p.attn.forward(q, p.table, p.lens, starts, max_seq_len=150)
    assert p.attn.status()["bad_length"]
    if counts:
        p.attn._status.zero_()
        out = torch.full_like(q, 3.0)
        p.attn.forward(q, p.table, p.lens, starts, max_queries=8, out=out)
        assert p.attn.status()["bad_length"]
        check_rows(out[:8], *[x[:8] for x in reference(q[:9], p.k[0], p.v[0], causal(9, 200), p.attn.scale)])


def test_past_32_bit_offsets(gpu_device):
    """Sequences whose pages lie behind 4 GiB of a cache tensor."""
    announce("attention past 4 GiB")
    g = generator(19)
    attn = make_attention(8, 8, 128, "bf16", 256, 10000)
    table = torch.tensor([[9999, 0, 8192], [4097, 8191, 5]], dtype=torch.int32, device=DEV)
    lengths = [700, 513]
    ks, vs = [], []
    for b, n in enumerate(lengths):
        slots = attn.slots(table, torch.full((n,), b, device=DEV), torch.arange(n, device=DEV))
        put(attn, slots, randn(g, n, 8, 128).float(), randn(g, n, 8, 128).float())
        k, v = dense(attn, slots)
        ks.append(k)
        vs.append(v)
    lens = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    for counts in ([1, 1], [200, 60]):
        q = randn(g, sum(counts), 8, 128)
        got = attn.forward(q, table, lens, starts_of(counts), max_queries=max(counts))
        at = split_rows(counts)
        for b in range(2):
            rows = slice(at[b], at[b + 1])
            check_rows(got[rows], *reference(q[rows], ks[b], vs[b], causal(counts[b], lengths[b]), attn.scale))


@pytest.mark.parametrize("scale", [0.02, 1.0])
def test_other_scales(gpu_device, scale):
    announce(f"scale {scale}")
    p = make_problem([300, 77], heads=8, kv_heads=2, dim=64, fmt="bf16", page=64, seed=18, spread=0.3)
    p.attn.scale = scale
    q = randn(generator(18), 45, 8, 64)
    for counts in ([1, 1], [40, 5]):
        check_attention(p, counts, q[:sum(counts)], p.attn.forward(q[:sum(counts)], p.table, p.lens, starts_of(counts)))


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
def test_scores_far_below_zero(gpu_device, fmt):
    """Every score of a row is far below zero: the maximum has to come down to it."""
    announce(f"scores far below zero {fmt}")
    lengths = [1000, 70]
    p = make_problem(lengths, heads=8, kv_heads=2, dim=128, fmt=fmt, page=64, seed=19)
    g = generator(20)
    base = 4 * randn(g, 1, 2, 128).float()
    for b, n in enumerate(lengths):
        at = torch.arange(n, device=DEV)
        slots = p.attn.slots(p.table, torch.full_like(at, b), at)
        put(p.attn, slots, base + 0.1 * randn(g, n, 2, 128).float(), randn(g, n, 2, 128).float())
        p.k[b], p.v[b] = dense(p.attn, slots)
    for counts in ([1, 1], [5, 40]):
        q = (-4 * base.repeat_interleave(4, dim=1) / 4).expand(sum(counts), -1, -1).to(torch.bfloat16).contiguous()
        got = p.attn.forward(q, p.table, p.lens, starts_of(counts))
        at = split_rows(counts)
        for b in range(2):
            rows = slice(at[b], at[b + 1])
            want, A = reference(q[rows], p.k[b], p.v[b], causal(counts[b], lengths[b]), p.attn.scale)
            # scores of about -16 |base|^2 / sqrt(128) = -180: fp32 off by 2^-24 * 136 * 180 at most, 2^-9.4
            assert bool(((got[rows].double() - want).abs() <= (2 * 2.0 ** -8 + 2.0 ** -7) * A).all())


def test_rows_do_not_depend_on_the_batch(gpu_device):
    """The same sequence alone, among others and in other rows gives the same bits (fixed launch bounds)."""
    announce("batch independence")
    p = make_problem([900, 333, 64], heads=16, kv_heads=4, dim=128, fmt="int8", page=64, seed=20)
    q = randn(generator(21), 3, 16, 128)
    every = p.attn.forward(q, p.table, p.lens)
    order = torch.tensor([2, 0, 1], device=DEV)
    assert torch.equal(p.attn.forward(q[order], p.table[order], p.lens[order]), every[order])


def test_captured_graph_with_growing_lengths(gpu_device):
    """A decode step captured once and replayed while lengths grow on the device, with eager calls of other
    shapes between the replays."""
    announce("decode step in a graph")
    lengths = [3000, 100, 1, 64]
    p = make_problem([n + 8 for n in lengths], heads=32, kv_heads=4, dim=128, fmt="bf16", page=64, seed=22)
    g = generator(23)
    q = randn(g, 4, 32, 128)
    lens = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    p.attn.forward(q, p.table, lens)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = p.attn.forward(q, p.table, lens)
    for i in range(5):
        lens += 1
        q.copy_(randn(g, 4, 32, 128))
        rows = randn(g, 300, 32, 128)
        p.attn.forward(rows, p.table[:1], lens[:1], starts_of([300]))  # eager, its own workspace
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, p.attn.forward(q, p.table, lens)), i
        for b in range(4):
            n = lengths[b] + i + 1
            check_rows(out[b:b + 1], *reference(q[b:b + 1], p.k[b][:n], p.v[b][:n], causal(1, n), p.attn.scale))


def test_two_graphs_and_two_streams_at_once(gpu_device):
    """Calls that overlap share nothing: two graphs replayed on two streams, and eager calls beside them."""
    announce("two graphs at once")
    p = make_problem([5000, 4000], heads=32, kv_heads=4, dim=128, fmt="int8", page=64, seed=24)
    g = generator(25)
    qs = [randn(g, 2, 32, 128), randn(g, 40, 32, 128)]
    starts = [None, starts_of([30, 10])]
    want = [p.attn.forward(q, p.table, p.lens, s).clone() for q, s in zip(qs, starts)]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for q, s in zip(qs, starts):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(p.attn.forward(q, p.table, p.lens, s))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for x in outs:
            x.zero_()
        torch.cuda.synchronize()
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        eager = p.attn.forward(qs[0], p.table, p.lens)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(eager, want[0])


def test_forward_refusals(gpu_device):
    attn = make_attention(8, 2, 128, "bf16", 64, 4)
    g = generator(1)
    q = randn(g, 3, 8, 128)
    table = torch.zeros(3, 2, dtype=torch.int32, device=DEV)
    lens = torch.ones(3, dtype=torch.int32, device=DEV)
    mask = torch.zeros(3, 1, dtype=torch.int64, device=DEV)
    good = dict(q=q, page_table=table, seq_lens=lens)
    for bad in (dict(q=q.half()), dict(q=q.cpu()), dict(q=q[:, :4]), dict(q=q[:2]), dict(page_table=table[0]),
                dict(page_table=table.float()), dict(page_table=table.cpu()), dict(seq_lens=lens[:2]),
                dict(query_starts=lens), dict(out=q.float()), dict(out=q[:2])):
        with pytest.raises(ValueError):
            attn.forward(**{**good, **bad})
        with pytest.raises(ValueError):
            attn.forward_tree(tree_mask=mask, **{**good, **bad})
    for bad in (mask.int(), mask[0], mask[:2], mask.cpu()):
        with pytest.raises(ValueError):
            attn.forward_tree(q, bad, table, lens)
    with pytest.raises(RuntimeError):
        attn.forward_tree(q, mask[:, :0], table, lens)
    for scale in (0.0, -1.0, float("nan")):
        with pytest.raises(ValueError, match="scale"):
            make_attention(8, 2, 128, "bf16", 64, 4, scale=scale)
    # rows one element off 16 bytes, and transposed ones, are copied
    p = make_problem([70, 3, 9], heads=8, kv_heads=2, dim=128, fmt="bf16", page=64, seed=30)
    want = p.attn.forward(q, p.table, p.lens)
    off = torch.cat([q.new_zeros(1), q.flatten()])[1:].view_as(q)
    turned = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(p.attn.forward(off, p.table, p.lens), want)
    assert torch.equal(p.attn.forward(turned, p.table, p.lens), want)
    assert torch.equal(p.attn.forward(q.flatten(1), p.table, p.lens), want)
    # nothing to do: no rows, no sequences, no pages
    assert attn.forward(q[:0], table[:0], lens[:0]).shape == (0, 8, 128)
    assert attn.forward(q[:0], table, lens, torch.zeros(4, dtype=torch.int32, device=DEV)).shape == (0, 8, 128)
    none = torch.zeros(3, dtype=torch.int32, device=DEV)
    assert bool((attn.forward(q, table[:, :0], none) == 0).all())
