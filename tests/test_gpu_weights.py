"""Attention that sums what each cached token got (forward_weights), against the plain 64-bit implementation.

Tolerance.  A row's weight p is off by 2^-9.9 of itself at most (attn_cases.py: its own score's error and the
sum's; no rounding to bf16 enters the sums), fp32 sums of R positive terms and one last addition to what was
there by (R + 8) 2^-24 of the sum.  So |got - want| <= (2^-9.9 + (R + 8) 2^-24) added + 2^-24 |want|."""
import math
import sys

import pytest
import torch

from attn_cases import DEV, causal, check_attention, check_rows, dense, generator, make_problem, put, randn, reference, split_rows
from nano_ktrans_amd import _native as N

pytestmark = pytest.mark.gpu


def announce(msg):
    sys.__stderr__.write(f"[gpu-case] {msg}\n")
    sys.__stderr__.flush()


def starts_of(counts):
    return torch.tensor(split_rows(counts), dtype=torch.int32, device=DEV)


def start_weights(g, B, HK, width):
    """What earlier calls left: some of it zero."""
    w = torch.rand(B, HK, width, generator=g, device=DEV) * 3
    return w * (torch.rand(B, HK, width, generator=g, device=DEV) > 0.3)


def added_weights(q, k, sees, scale, last):
    """float64 [HK, L]: what the last rows of one sequence give its tokens."""
    n, H, _ = q.shape
    HK = k.shape[1]
    out = torch.zeros(HK, k.shape[0], dtype=torch.float64, device=q.device)
    if n == 0 or k.shape[0] == 0:
        return out
    empty = ~sees.any(dim=1)
    for h in range(H):
        s = (q[:, h].double() @ k[:, h // (H // HK)].T) * scale
        s = torch.where(sees, s, -math.inf)
        s = torch.where(empty.unsqueeze(1), 0.0, s)
        p = torch.where(sees & ~empty.unsqueeze(1), torch.softmax(s, dim=1), 0.0)
        out[h // (H // HK)] += p[max(0, n - last):].sum(dim=0)
    return out


def check_weights(p, counts, q, before, after, last=None):
    counts = counts or [1] * len(p.lengths)
    starts = split_rows(counts)
    for b, (n, length) in enumerate(zip(counts, p.lengths)):
        rows = q[starts[b]:starts[b + 1]]
        add = added_weights(rows, p.k[b], causal(n, length), p.attn.scale, n if last is None else last)
        got, was = after[b].double(), before[b].double()
        want = was[:, :length] + add
        R = n * q.shape[1] // p.attn.num_kv_heads
        bound = (2.0 ** -9.9 + (R + 8) * 2.0 ** -24) * add + 2.0 ** -24 * want.abs()
        off = (got[:, :length] - want).abs() - bound
        assert bool((off <= 0).all()), f"sequence {b} ({n} rows, {length} tokens): worst {float(off.max())} over its bound"
        assert torch.equal(after[b][:, length:], before[b][:, length:]), f"sequence {b}: weights behind its end changed"


SHAPES = [(32, 4, 128), (32, 8, 128), (16, 16, 128), (14, 2, 64), (5, 1, 64)]


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES)
@pytest.mark.parametrize("lengths", [[1], [517], [64, 1, 65, 0, 700, 2500]])
def test_decode(gpu_device, heads, kv_heads, dim, fmt, lengths):
    announce(f"weights decode {heads}/{kv_heads}/{dim} {fmt} {lengths}")
    p = make_problem(lengths, heads=heads, kv_heads=kv_heads, dim=dim, fmt=fmt, page=128, seed=1)
    g = generator(2)
    q = randn(g, len(lengths), heads, dim)
    before = start_weights(g, len(lengths), kv_heads, 3000)
    after = before.clone()
    got = p.attn.forward_weights(q, after, p.table, p.lens, max_seq_len=2600)
    check_attention(p, None, q, got)
    check_weights(p, None, q, before, after)
    p.attn.check_status()


@pytest.mark.parametrize("heads,kv_heads,dim,counts", [
    (32, 4, 128, [1, 1, 1]), (5, 1, 64, [1]), (32, 4, 128, [3, 8]), (5, 1, 64, [4]), (14, 2, 64, [40])])
def test_one_int8_token_is_its_value(gpu_device, heads, kv_heads, dim, counts):
    """A row that sees one token: weight x scale is rounded to bf16 for the product, but all of that is common to
    the row and taken out again.  What is left: the output's rounding, 2^-8 of it, and a few of fp32, under 2^-20."""
    announce(f"weights of one int8 token {heads}/{kv_heads}/{dim} {counts}")
    for seed in range(4):
        p = make_problem(counts, heads=heads, kv_heads=kv_heads, dim=dim, fmt="int8", page=64, seed=seed)
        q = randn(generator(seed + 9), sum(counts), heads, dim)
        weights = torch.zeros(len(counts), kv_heads, max(counts), device=DEV)
        starts = None if max(counts) == 1 else starts_of(counts)
        got = p.attn.forward_weights(q, weights, p.table, p.lens, starts, max_queries=max(counts), max_seq_len=max(counts))
        for b, first in enumerate(split_rows(counts)[:-1]):
            want = p.v[b][0].repeat_interleave(heads // kv_heads, dim=0).double()
            off = (got[first].double() - want).abs() - (2.0 ** -8 + 2.0 ** -20) * want.abs()
            assert bool((off <= 0).all()), f"sequence {b}: worst {float(off.max())} over its bound"


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES)
@pytest.mark.parametrize("counts,lengths", [([2, 1], [70, 1]), ([5, 16, 1], [40, 300, 90]), ([33, 64, 0, 7], [900, 64, 12, 8]),
                                            ([300, 129, 1], [300, 2000, 555]), ([12], [5])])
@pytest.mark.parametrize("last", [None, 1, 40])
def test_prompts(gpu_device, heads, kv_heads, dim, fmt, counts, lengths, last):
    """All forms of the attention kernels, parts of rows, rows before the cache's first token."""
    announce(f"weights prompts {heads}/{kv_heads}/{dim} {fmt} rows {counts} of {lengths} last {last}")
    p = make_problem(lengths, heads=heads, kv_heads=kv_heads, dim=dim, fmt=fmt, page=64, seed=3)
    g = generator(4)
    q = randn(g, sum(counts), heads, dim)
    before = start_weights(g, len(lengths), kv_heads, p.table.shape[1] * 64)
    after = before.clone()
    got = p.attn.forward_weights(q, after, p.table, p.lens, starts_of(counts), max_queries=max(counts), last=last)
    check_attention(p, counts, q, got)
    check_weights(p, counts, q, before, after, last)
    p.attn.check_status()


def test_long_prompt_and_strided_weights(gpu_device):
    """Enough rows for several parts of them; weights as part of a larger array, heads outside of sequences."""
    announce("weights long prompt")
    counts, lengths = [2100, 3], [2100, 4000]
    p = make_problem(lengths, heads=8, kv_heads=2, dim=128, fmt="bf16", page=256, seed=5)
    g = generator(6)
    q = randn(g, sum(counts), 8, 128)
    whole = torch.rand(2, 5, 5000, generator=g, device=DEV)
    before = whole.clone()
    after = whole[:, 1:3, 7:4300].transpose(0, 1)
    got = p.attn.forward_weights(q, after, p.table, p.lens, starts_of(counts), max_queries=2100, max_seq_len=4000)
    check_attention(p, counts, q, got)
    check_weights(p, counts, q, before[:, 1:3, 7:4300].transpose(0, 1), after)
    whole[:, 1:3, 7:4300] = before[:, 1:3, 7:4300]
    assert torch.equal(whole, before)


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
def test_few_rows_of_a_wide_bound(gpu_device, fmt):
    """A bound so wide that the scores of the rows are not kept (over 1 GiB): the keys are read again."""
    announce(f"weights of a wide bound {fmt}")
    lengths = [500, 3, 260] * 22
    p = make_problem(lengths, heads=32, kv_heads=4, dim=128, fmt=fmt, page=256, seed=20, width=2)
    table = torch.full((66, 548), -1, dtype=torch.int32, device=DEV)
    table[:, :2] = p.table
    g = generator(21)
    q = randn(g, 66, 32, 128)
    before = start_weights(g, 66, 4, 548 * 256)
    after = before.clone()
    got = p.attn.forward_weights(q, after, table, p.lens)
    check_attention(p, None, q, got)
    check_weights(p, None, q, before, after)
    narrow = before.clone()
    assert torch.equal(got, p.attn.forward_weights(q, narrow, table, p.lens, max_seq_len=512))
    assert float((narrow - after).abs().max()) <= 2.0 ** -14
    p.attn.check_status()


def test_calls_add_up_and_repeat(gpu_device):
    """A prompt in chunks gives what the whole prompt gives; the same call gives the same bits."""
    announce("weights in chunks")
    p = make_problem([600], heads=8, kv_heads=2, dim=64, fmt="bf16", page=64, seed=7)
    g = generator(8)
    q = randn(g, 600, 8, 64)
    sums = [torch.zeros(1, 2, 640, device=DEV) for _ in range(3)]
    for i in range(2):
        p.attn.forward_weights(q, sums[i], p.table, p.lens, starts_of([600]))
    assert torch.equal(sums[0], sums[1])
    for at, n in ((0, 1), (1, 63), (64, 236), (300, 300)):
        lens = torch.tensor([at + n], dtype=torch.int32, device=DEV)
        p.attn.forward_weights(q[at:at + n], sums[2], p.table, lens, starts_of([n]))
    check_weights(p, [600], q, torch.zeros_like(sums[0]), sums[0])
    check_weights(p, [600], q, torch.zeros_like(sums[0]), sums[2])


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
@pytest.mark.parametrize("counts", [[1, 1], [3, 4], [5, 16], [40, 70]])
@pytest.mark.parametrize("sign", [1, -1])
def test_large_scores(gpu_device, fmt, counts, sign):
    """Scores of 2^11 to 2^121 in size, one token's above all others' by a part of itself (as in
    test_gpu_attention_edges.py): a row's weight is 1 there and 0 elsewhere, never another power of two."""
    announce(f"weights of large scores {fmt} {counts} {sign}")
    lengths = [700, 300]
    p = make_problem(lengths, heads=8, kv_heads=2, dim=128, fmt=fmt, page=64, seed=9)
    g = generator(10)
    base = 1.0 - 2.0 * torch.randint(0, 2, (2, 128), generator=g, device=DEV).float()
    for power in (4, 15, 33, 55):
        q = (base * 2.0 ** power * sign).repeat_interleave(4, dim=0).to(torch.bfloat16)
        q = q.expand(sum(counts), -1, -1).contiguous()
        best = []
        for b, length in enumerate(lengths):
            size = torch.linspace(0.25, 0.75, length, device=DEV)[torch.randperm(length, generator=g, device=DEV)]
            size = torch.where(size == size.max(), 0.75, size.clamp(max=0.70))
            at = int(size.argmax())
            if at > length - counts[b]:  # (all rows see it)
                size[[0, at]] = size[[at, 0]]
                at = 0
            best.append(at)
            k = base.unsqueeze(0) * size.view(-1, 1, 1) * 2.0 ** power * sign
            if sign < 0:  # (all scores negative, the best nearest to zero)
                k = -base.unsqueeze(0) * (1.0 - size).view(-1, 1, 1) * 2.0 ** power * sign
            at_all = torch.arange(length, device=DEV)
            put(p.attn, p.attn.slots(p.table, torch.full_like(at_all, b), at_all), k,
                randn(g, length, 2, 128).float())
        w = torch.zeros(2, 2, p.table.shape[1] * 64, device=DEV)
        p.attn.forward_weights(q, w, p.table, p.lens, starts_of(counts), max_queries=max(counts))
        want = torch.zeros_like(w)
        for b, at in enumerate(best):
            want[b, :, at] = 4 * counts[b]
        assert torch.equal(w, want), f"power {power}"


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
@pytest.mark.parametrize("counts", [[1], [4], [16], [70]])
def test_nan_and_infinity(gpu_device, fmt, counts):
    """What no row sees reaches nothing, whatever lies there; a NaN in a value is none in its weight; a NaN key
    makes the weights of the rows that see it NaN and leaves the others."""
    announce(f"weights NaN {fmt} {counts}")
    n, length = counts[0], 200
    p = make_problem([length], heads=8, kv_heads=2, dim=128, fmt=fmt, page=64, seed=11)
    g = generator(12)
    q = randn(g, n, 8, 128)
    at = torch.arange(length, device=DEV)
    slots = p.attn.slots(p.table, torch.zeros_like(at), at)
    k, v = randn(g, length, 2, 128).float(), randn(g, length, 2, 128).float()
    put(p.attn, slots, k, v)
    p.k[0], p.v[0] = dense(p.attn, slots)
    page, r = int(slots[17]) // 64, int(slots[17]) % 64
    if fmt == "bf16":
        unit = 8
        p.attn.v_cache[page, 0, r // unit, 3, r % unit] = float("nan")
    else:
        p.attn.v_scales[page, 0, r] = float("nan")
    before = torch.zeros(1, 2, 256, device=DEV)
    after = before.clone()
    out = p.attn.forward_weights(q, after, p.table, p.lens, starts_of(counts))
    assert bool(torch.isnan(out[:, :4]).any()) and not bool(torch.isnan(out[:, 4:]).any())
    check_weights(p, counts, q, before, after)
    if n < 2:
        return
    # a NaN key at the last token but one: the rows before it do not see it
    page, r = int(slots[length - 2]) // 64, int(slots[length - 2]) % 64
    if fmt == "bf16":
        p.attn.k_cache[page, 0, r, 5] = float("nan")
    else:
        p.attn.k_scales[page, 0, r] = float("nan")
    after = before.clone()
    p.attn.forward_weights(q, after, p.table, p.lens, starts_of(counts))
    assert bool(torch.isnan(after[0, 0, :length]).all()) and not bool(torch.isnan(after[0, 1]).any())
    after = before.clone()
    short = torch.tensor([length - 2], dtype=torch.int32, device=DEV)
    p.attn.forward_weights(q[:n - 2], after, p.table, short, starts_of([n - 2]))
    assert not bool(torch.isnan(after).any())


def test_shared_pages_padding_and_bad_pages(gpu_device):
    """Two sequences on the same pages each get their own weights; rows behind the last sequence stay; a page
    outside the cache is reported and its tokens' weights stay."""
    announce("weights shared pages")
    p = make_problem([130, 130], heads=8, kv_heads=2, dim=128, fmt="bf16", page=64, seed=13)
    p.table[1] = p.table[0]
    p.k[1], p.v[1] = p.k[0], p.v[0]
    g = generator(14)
    q = randn(g, 9, 8, 128)
    before = start_weights(g, 2, 2, 192)
    after = before.clone()
    out = torch.full((9, 8, 128), 7.0, dtype=torch.bfloat16, device=DEV)
    p.attn.forward_weights(q, after, p.table, p.lens, starts_of([2, 4]), max_queries=5, out=out)
    check_attention(p, [2, 4], q, out)
    check_weights(p, [2, 4], q, before, after)
    assert bool((out[6:] == 7.0).all())
    p.attn.check_status()
    p.table[1, 1] = p.attn.num_pages
    after = before.clone()
    p.attn.forward_weights(q, after, p.table, p.lens, starts_of([2, 4]), max_queries=5)
    assert torch.equal(after[1, :, 64:128], before[1, :, 64:128])
    assert not torch.equal(after[1, :, :64], before[1, :, :64])
    assert p.attn.status()["bad_page"]


def test_graph_replays_and_streams(gpu_device):
    """A captured decode step adds to the weights at every replay, beside eager calls on another stream."""
    announce("weights in a graph")
    lengths = [900, 33, 400]
    p = make_problem(lengths, heads=32, kv_heads=4, dim=128, fmt="int8", page=64, seed=15)
    g = generator(16)
    q = randn(g, 3, 32, 128)
    w, eager = torch.zeros(3, 4, 960, device=DEV), torch.zeros(3, 4, 960, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        p.attn.forward_weights(q, w, p.table, p.lens, max_seq_len=900)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = p.attn.forward_weights(q, w, p.table, p.lens, max_seq_len=900)
    torch.cuda.current_stream().wait_stream(side)
    w.zero_()
    for _ in range(3):
        graph.replay()
        want = p.attn.forward_weights(q, eager, p.table, p.lens, max_seq_len=900)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(w, eager)
    q.copy_(randn(g, 3, 32, 128))
    graph.replay()
    want = p.attn.forward_weights(q, eager, p.table, p.lens, max_seq_len=900)
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(w, eager)


@pytest.mark.parametrize("make", [
    lambda w: w.half(), lambda w: w[:1], lambda w: w[:, :1], lambda w: w[0], lambda w: w[:, :, ::2], lambda w: w.cpu(),
    lambda w: w[:, :, :100], lambda w: w[:1].expand(2, -1, -1), lambda w: w[:, :1].expand(-1, 2, -1),
])
def test_refused_weights(gpu_device, make):
    p = make_problem([130, 100], heads=8, kv_heads=2, dim=128, fmt="bf16", page=64, seed=17)
    w = torch.zeros(2, 2, 192, device=DEV)
    with pytest.raises((ValueError, N.NativeError)):
        p.attn.forward_weights(randn(generator(1), 2, 8, 128), make(w), p.table, p.lens)
    with pytest.raises(ValueError):
        p.attn.forward_weights(randn(generator(1), 2, 8, 128), w, p.table, p.lens, last=0)
    q = randn(generator(1), 2, 8, 128)
    with pytest.raises(N.NativeError, match="overlaps q"):
        p.attn.forward_weights(q, w, p.table, p.lens, out=q)
    torch.cuda.synchronize()
    assert not bool(w.any())
