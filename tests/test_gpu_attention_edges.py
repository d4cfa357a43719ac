"""Attention over the paged cache on the GPU at the ends of its values' and indexes' ranges, against the plain
64-bit implementation in attn_cases.py (which has the tolerances)."""
import sys

import pytest
import torch

from attn_cases import DEV, check_attention, dense, generator, make_problem, put, randn, split_rows

pytestmark = pytest.mark.gpu

# rows per sequence of 8 / 2 heads: the row form, the 64-row form and the tile form
FORMS = [[1, 1], [3, 4], [5, 16], [40, 70]]


def announce(msg):
    sys.__stderr__.write(f"[gpu-case] {msg}\n")
    sys.__stderr__.flush()


def starts_of(counts):
    return torch.tensor(split_rows(counts), dtype=torch.int32, device=DEV)


def signs(g, *shape):
    return 1.0 - 2.0 * torch.randint(0, 2, shape, generator=g, device=DEV).float()


def store(p, b, k, v):
    """Keys and values [len, HK, D] (fp32) as sequence b's, and what the cache then holds of them."""
    at = torch.arange(p.lengths[b], device=DEV)
    slots = p.attn.slots(p.table, torch.full_like(at, b), at)
    put(p.attn, slots, k, v)
    p.k[b], p.v[b] = dense(p.attn, slots)


def attend(p, counts, q):
    return p.attn.forward(q, p.table, p.lens, starts_of(counts), max_queries=max(counts))


@pytest.mark.parametrize("counts", FORMS)
@pytest.mark.parametrize("lengths", [[80, 75], [700, 3000]])
def test_infinite_values_reach_the_rows_that_see_them(gpu_device, counts, lengths):
    """An infinity in a value, beside later tokens: the rows that see it are infinite there and nowhere else
    (not NaN), also where its own score lies far above all before it.  Such rows' weights are 0 and 1 (the
    next score is 2^-250 of it), so their scores' size adds no error."""
    announce(f"infinite values, rows {counts} of {lengths}")
    p = make_problem(lengths, heads=8, kv_heads=2, dim=128, fmt="bf16", page=64, seed=3)
    g = generator(5)
    base = signs(g, 2, 128)
    for b, (n, length) in enumerate(zip(counts, lengths)):
        for far in (False, True):
            k, v = 0.01 * randn(g, length, 2, 128).float(), randn(g, length, 2, 128).float()
            at = length - 1 - n // 2
            if far:
                k[at] = base
            v[at, 0, 3], v[at, 1, 70], v[at, 1, 71] = float("inf"), float("-inf"), float("inf")
            store(p, b, k, v)
            q = (16 * base).repeat_interleave(4, dim=0).to(torch.bfloat16).expand(sum(counts), -1, -1).contiguous()
            check_attention(p, counts, q, attend(p, counts, q))


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
@pytest.mark.parametrize("counts", FORMS)
@pytest.mark.parametrize("lengths", [[80, 75], [700, 3000]])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_past_24_bits(gpu_device, fmt, counts, lengths, sign):
    """Finite scores of 2^35 to 2^125, one token's above all others' by a part of itself: its value, whatever a
    product of such a score keeps of its lower bits.  (fp32 scores are off by 2^-16 of their terms' sum at most,
    the gaps are 2^-7 of the largest and more, so all weights but that token's are 0.)"""
    announce(f"large scores {fmt} rows {counts} of {lengths} sign {sign}")
    p = make_problem(lengths, heads=8, kv_heads=2, dim=128, fmt=fmt, page=64, seed=4)
    g = generator(6)
    base = signs(g, 2, 128)
    for power in (15, 33, 55):
        for b, (n, length) in enumerate(zip(counts, lengths)):
            c = torch.randint(2, 127, (length,), generator=g, device=DEV).float()
            c[length - n - b] = 128 if sign > 0 else 1  # (every row sees it)
            store(p, b, c.view(-1, 1, 1) * base * 2.0 ** power, randn(g, length, 2, 128).float())
        q = (sign * 2.0 ** power * base).repeat_interleave(4, dim=0).to(torch.bfloat16)
        q = q.expand(sum(counts), -1, -1).contiguous()
        check_attention(p, counts, q, attend(p, counts, q))


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
@pytest.mark.parametrize("counts", FORMS)
@pytest.mark.parametrize("lengths", [[80, 75], [700, 3000]])
def test_finite_scores_near_the_lowest_number(gpu_device, fmt, counts, lengths):
    """Every score of a row is finite and below -1.2e38 (times log2(e)): such a row is not one that sees
    nothing.  One token's score is a fifth above all others', so the row is its value."""
    announce(f"lowest scores {fmt} rows {counts} of {lengths}")
    p = make_problem(lengths, heads=8, kv_heads=2, dim=128, fmt=fmt, page=64, seed=4)
    p.attn.scale = 1.0
    g = generator(7)
    base = signs(g, 2, 128)
    for b, (n, length) in enumerate(zip(counts, lengths)):
        c = 1.25 + 0.125 * torch.randint(0, 11, (length,), generator=g, device=DEV).float()
        c[length - n - b] = 1  # (every row sees it)
        store(p, b, c.view(-1, 1, 1) * base * 2.0 ** 59, randn(g, length, 2, 128).float())
    q = (-2.0 ** 60 * base).repeat_interleave(4, dim=0).to(torch.bfloat16).expand(sum(counts), -1, -1).contiguous()
    check_attention(p, counts, q, attend(p, counts, q))


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
@pytest.mark.parametrize("counts", FORMS)
@pytest.mark.parametrize("power", [120, -120])
def test_values_near_the_largest_and_smallest_numbers(gpu_device, fmt, counts, power):
    """Values up to 2^120, whose weighted sum passes fp32's range if a weight is 2^7.5 and does not if weights
    are 1 at most (74 x 2^120): the scores rise by 2^7.5 behind the first 64 tokens, or 256 (each wave of the
    row form has then seen some).  And as small ones, which weights below 1 must not lose: 2^-120 leaves 2^-29
    of it to fp32's smallest step, 2^-21 under a weight of 2^-8, far below the weight's rounding."""
    announce(f"values of 2^{power} {fmt} rows {counts}")
    g = generator(8)
    base = signs(g, 2, 128)
    for low in (64, 256):
        length = low + 74
        p = make_problem([length, length], heads=8, kv_heads=2, dim=128, fmt=fmt, page=64, seed=4)
        for b in range(2):
            k = torch.zeros(length, 2, 128, device=DEV)
            k[low:] = 0.4609375 * base  # a score of 5.2 = 7.5 ln 2
            v = torch.rand(length, 2, 128, generator=g, device=DEV)
            v[:, :, ::2] *= signs(g, length, 2, 64)
            store(p, b, k, v * 2.0 ** power)
        q = base.repeat_interleave(4, dim=0).to(torch.bfloat16).expand(sum(counts), -1, -1).contiguous()
        got = attend(p, counts, q)
        if power < 0:
            # held against values 2^120 times as large (a power of two: exact), so that the bound's share for
            # values in the denormal range does not cover them
            p.v = [v * 2.0 ** 120 for v in p.v]
            got = got.double() * 2.0 ** 120
        check_attention(p, counts, q, got)


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
@pytest.mark.parametrize("counts", FORMS[1:])
@pytest.mark.parametrize("lengths", [[80, 75], [700, 3000]])
def test_large_values_reach_only_the_rows_that_see_them(gpu_device, fmt, counts, lengths):
    """A finite value of 2^121 in a sequence's last token: the rows before the last keep their bits."""
    announce(f"large unseen values {fmt} rows {counts} of {lengths}")
    p = make_problem(lengths, heads=8, kv_heads=2, dim=128, fmt=fmt, page=64, seed=9)
    g = generator(10)
    q = randn(g, sum(counts), 8, 128)
    before = attend(p, counts, q)
    for b, length in enumerate(lengths):
        # (the last token alone: an int8 row that is stored once more may get another scale)
        at = torch.arange(length, device=DEV)
        slots = p.attn.slots(p.table, torch.full_like(at, b), at)
        put(p.attn, slots[-1:], p.k[b][-1:].float(), 2.0 ** 121 * randn(g, 1, 2, 128).float())
        p.k[b], p.v[b] = dense(p.attn, slots)
    got = attend(p, counts, q)
    check_attention(p, counts, q, got)
    last = torch.tensor(split_rows(counts)[1:], device=DEV) - 1
    others = torch.ones(sum(counts), dtype=torch.bool, device=DEV)
    others[last] = False
    assert torch.equal(got[others], before[others]) and not torch.equal(got[last], before[last])


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
