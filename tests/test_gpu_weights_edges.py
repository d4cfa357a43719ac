"""forward_weights: its outputs beside forward's, against the plain 64-bit implementation.  Tolerances beside the
tests."""
import pytest
import torch

from attn_cases import DEV, check_rows, causal, dense, generator, make_problem, put, randn, reference, split_rows
from nano_ktrans_amd import _native as N
from test_gpu_weights import added_weights, announce, check_weights, start_weights, starts_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv_heads,dim,counts", [
    (8, 2, 128, [40]), (8, 2, 128, [16]), (14, 2, 64, [40]), (14, 2, 64, [8]), (4, 4, 128, [300]), (32, 4, 128, [5, 3]),
    (32, 4, 128, [1]), (8, 2, 128, [4, 1]), (14, 2, 64, [2])])
def test_later_token_that_outweighs_the_rest(gpu_device, heads, kv_heads, dim, counts):
    """bf16.  A row's scores, in powers of two: 0 for token 0, 7 to 8 (by row) for a later token of the same wave, far
    less for all others; only the later token has a value.  A row's largest weight so far may lie 2^8 below 1 when
    that comes, so that its weight w is no power of two and rounding it for the product changes it by up to 2^-8 of
    itself.  Divided by a sum of the rounded weights that is gone: with r = 1 + e of each, the quotient is off by p0
    |e0 - e1|, p0 <= 2^-7 the weight of token 0, under 2^-14 of it.  A score is a sum of two terms under 2^4 in size,
    off by 2^-20 at most, which moves the quotient by p0 2^-20.  What is left is the output's rounding: (2^-8 + 2^-13)
    |want|."""
    announce(f"weights, later token {heads}/{kv_heads}/{dim} rows {counts}")
    late = 70 if max(counts) * heads // kv_heads > 16 else 130  # (few rows: a wave's steps are 128 tokens apart)
    lengths = [late + 30 + n for n in counts]
    p = make_problem(lengths, heads=heads, kv_heads=kv_heads, dim=dim, fmt="bf16", page=64, seed=31)
    g = generator(32)
    rows = sum(counts)
    # q has 1 at 0 and its row's power at 1; keys ask for -64 of the first or the whole of the second
    unit = p.attn.scale * 1.4426950408889634
    q = torch.zeros(rows, heads, dim, device=DEV)
    q[:, :, 0] = 1.0
    q[:, :, 1] = 7 + torch.rand(rows, heads, generator=g, device=DEV) * 0.98
    q = q.to(torch.bfloat16)
    for b, length in enumerate(lengths):
        k, v = torch.zeros(length, kv_heads, dim, device=DEV), torch.zeros(length, kv_heads, dim, device=DEV)
        k[:, :, 0] = -64.0 / unit
        k[0, :, 0] = k[late, :, 0] = 0.0
        k[late, :, 1] = 1.0 / unit
        v[late] = 1 + torch.rand(kv_heads, dim, generator=g, device=DEV)
        at = torch.arange(length, device=DEV)
        slots = p.attn.slots(p.table, torch.full_like(at, b), at)
        put(p.attn, slots, k, v)
        p.k[b], p.v[b] = dense(p.attn, slots)
    weights = torch.zeros(len(counts), kv_heads, p.table.shape[1] * 64, device=DEV)
    before = weights.clone()
    got = p.attn.forward_weights(q, weights, p.table, p.lens, starts_of(counts), max_queries=max(counts))
    starts = split_rows(counts)
    for b, (n, length) in enumerate(zip(counts, lengths)):
        mine = slice(starts[b], starts[b + 1])
        want, _ = reference(q[mine], p.k[b], p.v[b], causal(n, length), p.attn.scale)
        off = (got[mine].double() - want).abs() - (2.0 ** -8 + 2.0 ** -13) * want.abs()
        assert bool((off <= 0).all()), f"sequence {b}: worst {float(off.max())} over its bound"
    check_weights(p, counts, q, before, weights)


@pytest.mark.parametrize("heads,kv_heads,dim,counts,lengths", [
    (32, 4, 128, [600], [600]), (32, 8, 128, [129, 40], [2000, 700]), (14, 2, 64, [600], [600]), (8, 2, 128, [16, 9], [300, 64]),
    (14, 2, 64, [8, 9], [3000, 500]), (8, 2, 128, [2100], [2100])])
def test_bf16_outputs_are_as_exact_as_forwards(gpu_device, heads, kv_heads, dim, counts, lengths):
    """Tiles.  Rounding weight p_j to p_j (1 + e_j) for the product and dividing by the sum of what was rounded leaves
    the sum of p_j e_j (v_j - out) in a row's output: so it is in forward.  Here the tokens of each part of the
    sequence are evened by themselves, which leaves p_j e_j (v_j - out of the part), of no larger variance: a part's
    mean lies nearer to its values than the row's.  So the rms error is forward's at most, but for what a sample of at
    least 10^4 rows x heads x dimensions differs by, under 1 / 100.

    Rows that see up to 128 tokens, the least of a part, have one part (where a sequence has more than 64 rows x
    heads of a group; below that the halves of each 64 tokens are parts): the same quotient, with fp32 sums taken in
    another way, off by 2^-14 at most for the terms here.  An output lies on the other side of a border between two
    bf16 numbers in 2^-14 / 2^-8 of the cases: fewer than 1 in 32 differ, by one step."""
    announce(f"weights, outputs of forward {heads}/{kv_heads}/{dim} rows {counts} of {lengths}")
    p = make_problem(lengths, heads=heads, kv_heads=kv_heads, dim=dim, fmt="bf16", page=64, seed=33)
    q = 2 * randn(generator(34), sum(counts), heads, dim)
    weights = torch.zeros(len(counts), kv_heads, p.table.shape[1] * 64, device=DEV)
    args = (p.table, p.lens, starts_of(counts))
    other = p.attn.forward(q, *args, max_queries=max(counts))
    got = p.attn.forward_weights(q, weights, *args, max_queries=max(counts))
    starts = split_rows(counts)
    squares = [0.0, 0.0]
    for b, (n, length) in enumerate(zip(counts, lengths)):
        mine = slice(starts[b], starts[b + 1])
        want, _ = reference(q[mine], p.k[b], p.v[b], causal(n, length), p.attn.scale)
        for i, out in enumerate((got, other)):
            squares[i] += float((out[mine].double() - want).square().sum())
        few = torch.arange(length - n + 1, length + 1, device=DEV) <= (128 if max(counts) * heads // kv_heads > 64 else 0)
        x, y = got[mine][few], other[mine][few]
        differ = x != y
        assert int(differ.sum()) <= x.numel() / 32
        # (a step: 2^-7 of the power of two below; sums near zero have larger errors than their own size says)
        size = y.double().abs().clamp(min=2.0 ** -6)
        assert bool(((x.double() - y.double()).abs() <= 2.0 ** -7 * size).all())
    assert squares[0] <= 1.01 ** 2 * squares[1], f"rms {squares[0] ** 0.5} where forward has {squares[1] ** 0.5}"


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 4, 128), (14, 2, 64)])
@pytest.mark.parametrize("counts", [[1, 1, 1], [2, 1, 2], [8, 5, 0], [150, 1, 300]])
def test_lengths_that_are_cut(gpu_device, heads, kv_heads, dim, fmt, counts):
    """Lengths past max_seq_len, past a sequence's pages, negative: reported; the rows keep their positions and see (and give
    weight to) the tokens up to the cut.  Tolerances as in test_gpu_weights.py."""
    announce(f"weights, cut lengths {heads}/{kv_heads}/{dim} {fmt} rows {counts}")
    told, cut = [700, 450, -3], [600, 384, 0]
    p = make_problem([700, 384, 40], heads=heads, kv_heads=kv_heads, dim=dim, fmt=fmt, page=64, seed=35)
    p.table[1, 6:] = -1  # (the second sequence's pages end at 384: the rest is reported and not seen)
    lens = torch.tensor(told, dtype=torch.int32, device=DEV)
    g = generator(36)
    q = randn(g, sum(counts), heads, dim)
    before = start_weights(g, 3, kv_heads, 640)
    after = before.clone()
    got = p.attn.forward_weights(q, after, p.table, lens, starts_of(counts), max_queries=max(counts), max_seq_len=600)
    seen = p.attn.status()
    assert seen["bad_length"] and seen["bad_page"]
    starts = split_rows(counts)
    for b, n in enumerate(counts):
        mine = slice(starts[b], starts[b + 1])
        k, v = p.k[b][:cut[b]], p.v[b][:cut[b]]
        sees = causal(n, max(told[b], 0))[:, :cut[b]]
        want, A = reference(q[mine], k, v, sees, p.attn.scale)
        check_rows(got[mine], want, A)
        add = added_weights(q[mine], k, sees, p.attn.scale, n)
        was, now = before[b].double(), after[b].double()
        R = n * heads // kv_heads
        bound = (2.0 ** -9.9 + (R + 8) * 2.0 ** -24) * add + 2.0 ** -24 * (was[:, :cut[b]] + add)
        assert bool(((now[:, :cut[b]] - was[:, :cut[b]] - add).abs() <= bound).all())
        assert torch.equal(after[b][:, cut[b]:], before[b][:, cut[b]:])


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
@pytest.mark.parametrize("counts,most", [([5, 2], 2), ([40, 1], 16), ([300, 20], 70)])
def test_more_rows_than_the_bound(gpu_device, fmt, counts, most):
    """Rows past max_queries are reported, left as they were, and give nothing."""
    announce(f"weights, rows {counts} past {most} {fmt}")
    lengths = [400, 90]
    p = make_problem(lengths, heads=8, kv_heads=2, dim=128, fmt=fmt, page=64, seed=37)
    g = generator(38)
    q = randn(g, sum(counts), 8, 128)
    before = start_weights(g, 2, 2, 448)
    after = before.clone()
    out = torch.full((sum(counts), 8, 128), 7.0, dtype=torch.bfloat16, device=DEV)
    p.attn.forward_weights(q, after, p.table, p.lens, starts_of(counts), max_queries=most, out=out)
    with pytest.raises(N.NativeError, match="bad_length"):
        p.attn.check_status()
    starts = split_rows(counts)
    for b, (n, length) in enumerate(zip(counts, lengths)):
        done = min(n, most)
        mine = slice(starts[b], starts[b] + done)
        sees = causal(n, length)[:done]
        want, A = reference(q[mine], p.k[b], p.v[b], sees, p.attn.scale)
        check_rows(out[mine], want, A)
        assert bool((out[starts[b] + done:starts[b + 1]] == 7.0).all())
        add = added_weights(q[mine], p.k[b], sees, p.attn.scale, done)
        was, now = before[b].double()[:, :length], after[b].double()[:, :length]
        bound = (2.0 ** -9.9 + (done * 4 + 8) * 2.0 ** -24) * add + 2.0 ** -24 * (was + add)
        assert bool(((now - was - add).abs() <= bound).all())
        assert torch.equal(after[b][:, length:], before[b][:, length:])


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
def test_two_streams_at_once(gpu_device, fmt):
    """A captured decode step replayed on one stream, prompts on another and decode steps on a third, with nothing
    between them: each gives what it gives alone, bit for bit."""
    announce(f"weights on three streams {fmt}")
    lengths = [3000, 33, 2400]
    p = make_problem(lengths, heads=32, kv_heads=4, dim=128, fmt=fmt, page=64, seed=39)
    g = generator(40)
    q, rows, counts = randn(g, 3, 32, 128), randn(g, 730, 32, 128), [700, 20, 10]
    starts, width = starts_of(counts), p.table.shape[1] * 64

    def decode(w):
        return p.attn.forward_weights(q, w, p.table, p.lens, max_seq_len=3000)

    def prompt(w):
        return p.attn.forward_weights(rows, w, p.table, p.lens, starts, max_queries=700, max_seq_len=3000)

    alone = [torch.zeros(3, 4, width, device=DEV) for _ in range(2)]
    steps = [decode(alone[0]) for _ in range(6)]
    prompts = [prompt(alone[1]) for _ in range(6)]
    together = [torch.zeros_like(alone[0]) for _ in range(3)]
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[0]):
        captured = decode(together[0])
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(6):
        with torch.cuda.stream(streams[0]):
            graph.replay()
        with torch.cuda.stream(streams[1]):
            outs[0].append(prompt(together[1]))
        with torch.cuda.stream(streams[2]):
            outs[1].append(decode(together[2]))
    torch.cuda.synchronize()
    assert torch.equal(captured, steps[-1]) and torch.equal(together[0], alone[0])
    assert all(torch.equal(a, b) for a, b in zip(outs[0], prompts)) and torch.equal(together[1], alone[1])
    assert all(torch.equal(a, b) for a, b in zip(outs[1], steps)) and torch.equal(together[2], alone[0])
    p.attn.check_status()
