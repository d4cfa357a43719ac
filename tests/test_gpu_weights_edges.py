"""forward_weights: its outputs beside forward's, against the plain 64-bit implementation.  Tolerances beside the
tests."""
import pytest
import torch

from attn_cases import DEV, causal, dense, generator, make_problem, put, randn, reference, split_rows
from test_gpu_weights import announce, check_weights, starts_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv_heads,dim,counts", [
    (8, 2, 128, [40]), (8, 2, 128, [16]), (14, 2, 64, [40]), (14, 2, 64, [8]), (4, 4, 128, [300]), (32, 4, 128, [5, 3])])
def test_later_token_that_outweighs_the_rest(gpu_device, heads, kv_heads, dim, counts):
    """bf16, tiles.  A row's scores, in powers of two: 0 for token 0, 7 to 8 (by row) for token 70, far less for all
    others; only token 70 has a value.  A row's largest weight so far may lie 2^8 below 1 when token 70 comes, so
    that its weight w is no power of two and rounding it for the product changes it by up to 2^-8 of itself.  Divided
    by a sum of the rounded weights that is gone: with r = 1 + e of each, the quotient is off by p0 |e0 - e1|, p0 <=
    2^-7 the weight of token 0, under 2^-14 of it.  A score is a sum of two terms under 2^4 in size, off by 2^-20 at
    most, which moves the quotient by p0 2^-20.  What is left is the output's rounding: (2^-8 + 2^-13) |want|."""
    announce(f"weights, later token {heads}/{kv_heads}/{dim} rows {counts}")
    lengths = [100 + n for n in counts]
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
        k[0, :, 0] = k[70, :, 0] = 0.0
        k[70, :, 1] = 1.0 / unit
        v[70] = 1 + torch.rand(kv_heads, dim, generator=g, device=DEV)
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
