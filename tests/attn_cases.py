"""Seeded attention problems and a plain 64-bit implementation of the attention half's operators.

Tolerances.  u = 2^-8: a rounding to bf16 is off by at most half a step, finfo(bf16).eps / 2 of the value.

Attention: a softmax weight p (int8 caches: times its value's scale) is rounded to bf16 once before it
multiplies v, so a row's output is off by at most u * A, A = sum_j p_j |v_j|; the output itself is rounded
once more, u * (|out| + u A).  Everything else is fp32: a score of D products is off by at most about
(D + 8) 2^-24 sum |scale q_d k_d|, which the cases keep under 2^-24 * 136 * 64 < 2^-10.9 (their scores'
absolute sums stay below 64), and a weight by twice that relatively (its own score and the sum's): under
2^-9.9 A.  So |got - want| <= u |want| + (u + u^2 + 2^-9.9) A, plus 2^-130 for values in the denormal range.

Rotated rows: fp32 arithmetic of about 10 operations, under 2^-20 of |x1| + |x2| (the two rotated values,
after the norm), and one rounding, u |want|.  int8: code = round(x / scale) of that fp32 value, so the
stored value is off by half a scale step and by what the fp32 value is; scale itself by 2^-22 relatively.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import List, Optional

import torch

U = 2.0 ** -8
DEV = "cuda"


def generator(seed: int) -> torch.Generator:
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def randn(g, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


@dataclass
class Problem:
    """A cache with sequences of the given lengths in it: random pages in random order."""
    attn: object
    table: torch.Tensor          # int32 [B, W]
    lens: torch.Tensor           # int32 [B]
    lengths: List[int]
    k: torch.Tensor              # float64 [B][len, HK, D] as stored
    v: torch.Tensor


def make_attention(heads, kv_heads, dim, fmt, page, num_pages, **kw):
    from nano_ktrans_amd import NativeAttention

    return NativeAttention(num_heads=heads, num_kv_heads=kv_heads, head_dim=dim, num_pages=num_pages, page_size=page,
                           cache_format=fmt, **kw)


def poison(attn) -> None:
    """Fill the cache with NaN (int8: with NaN scales), as memory that nothing was written to may hold."""
    if attn.cache_format == "bf16":
        attn.k_cache.fill_(float("nan"))
        attn.v_cache.fill_(float("nan"))
    else:
        attn.k_cache.fill_(-128)
        attn.v_cache.fill_(-128)
        attn.k_scales.fill_(float("nan"))
        attn.v_scales.fill_(float("nan"))


def dense(attn, slots: torch.Tensor):
    """float64 keys and values [n, HK, D] at the slots, by the documented layout (no library call)."""
    slots = slots.long()
    page, r = torch.div(slots, attn.page_size, rounding_mode="floor"), slots % attn.page_size
    unit = attn.v_cache.shape[4]
    k = attn.k_cache[page, :, r].double()
    v = attn.v_cache[page, :, torch.div(r, unit, rounding_mode="floor"), :, r % unit].double()
    if attn.k_scales is not None:
        k = k * attn.k_scales[page, :, r].double().unsqueeze(-1)
        v = v * attn.v_scales[page, :, r].double().unsqueeze(-1)
    return k, v


def put(attn, slots: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> None:
    """Store fp32 rows [n, HK, D] at the slots by the documented layout (no library call)."""
    slots = slots.long()
    page, r = torch.div(slots, attn.page_size, rounding_mode="floor"), slots % attn.page_size
    unit = attn.v_cache.shape[4]
    if attn.k_scales is not None:
        for x, scales, which in ((k, attn.k_scales, 0), (v, attn.v_scales, 1)):
            s = x.abs().amax(dim=-1) / 127
            s = torch.where(s == 0, 1.0, s)
            scales[page, :, r] = s
            x = torch.round(x / s.unsqueeze(-1)).clamp(-127, 127)
            k, v = (x, v) if which == 0 else (k, x)
    attn.k_cache[page, :, r] = k.to(attn.k_cache.dtype)
    attn.v_cache[page, :, torch.div(r, unit, rounding_mode="floor"), :, r % unit] = v.to(attn.v_cache.dtype)


def make_problem(lengths, *, heads, kv_heads, dim, fmt, page, seed=0, width=None, spread=1.0, num_pages=None):
    g = generator(seed)
    W = width or max(1, max((n + page - 1) // page for n in lengths))
    B = len(lengths)
    pages = num_pages or B * W + 2
    attn = make_attention(heads, kv_heads, dim, fmt, page, pages)
    poison(attn)
    table = torch.randperm(pages, generator=g, device=DEV)[:B * W].view(B, W).to(torch.int32)
    ks, vs = [], []
    for b, n in enumerate(lengths):
        slots = attn.slots(table, torch.full((n,), b, device=DEV), torch.arange(n, device=DEV))
        put(attn, slots, spread * randn(g, n, kv_heads, dim).float(), randn(g, n, kv_heads, dim).float())
        k, v = dense(attn, slots)
        ks.append(k)
        vs.append(v)
    return Problem(attn, table, torch.tensor(lengths, dtype=torch.int32, device=DEV), list(lengths), ks, vs)


def reference(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, sees: torch.Tensor, scale: float):
    """float64 attention of one sequence: q [n, H, D], k and v [L, HK, D], sees [n, L] bool.  Returns
    (out, A) [n, H, D]; a row that sees nothing is zero.  What a row does not see is left out, not
    multiplied by zero."""
    n, H, D = q.shape
    group = H // k.shape[1]
    out = torch.zeros(n, H, D, dtype=torch.float64, device=q.device)
    A = torch.zeros_like(out)
    if k.shape[0] == 0 or n == 0:
        return out, A
    empty = ~sees.any(dim=1)
    clean = not bool(torch.isnan(v).any() or torch.isinf(v).any())
    for h in range(H):
        s = (q[:, h].double() @ k[:, h // group].T) * scale
        s = torch.where(sees, s, -math.inf)
        s = torch.where(empty.unsqueeze(1), 0.0, s)
        p = torch.softmax(s, dim=1)
        p = torch.where(empty.unsqueeze(1), 0.0, p)
        vh = v[:, h // group]
        if clean:
            out[:, h], A[:, h] = p @ vh, p @ vh.abs()
        else:
            for i in range(n):
                at = sees[i]
                out[i, h] = (p[i, at].unsqueeze(1) * vh[at]).sum(0)
                A[i, h] = (p[i, at].unsqueeze(1) * vh[at].abs()).sum(0)
    return out, A


def causal(n: int, length: int) -> torch.Tensor:
    i = torch.arange(n, device=DEV).unsqueeze(1)
    j = torch.arange(length, device=DEV).unsqueeze(0)
    return j <= length - n + i


def tree_sees(mask: torch.Tensor, n: int, length: int) -> torch.Tensor:
    """sees [n, length] of one sequence's rows of a tree mask."""
    sees = torch.zeros(n, length, dtype=torch.bool, device=DEV)
    context = length - n
    sees[:, :max(0, context)] = True
    for j in range(max(0, -context), n):
        if j // 64 < mask.shape[1]:
            sees[:, context + j] = ((mask[:, j // 64] >> (j % 64)) & 1).bool()
    return sees


def check_rows(got: torch.Tensor, want: torch.Tensor, A: torch.Tensor, what: str = "") -> None:
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    fine = torch.isfinite(want) & torch.isfinite(A)
    assert torch.equal(got[~torch.isfinite(want) & ~torch.isnan(want)], want[~torch.isfinite(want) & ~torch.isnan(want)])
    bound = U * want.abs() + (U + U * U + 2.0 ** -9.9) * A + 2.0 ** -130
    off = torch.where(fine, (got - want).abs() - bound, -1.0)
    assert bool((off <= 0).all()), \
        f"{what}: {int((off > 0).sum())} of {off.numel()} values off, worst by {float(off.max())} over its bound"


def split_rows(counts):
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    return starts


def check_attention(p: Problem, counts: Optional[List[int]], q: torch.Tensor, got: torch.Tensor, mask=None):
    """All rows against the 64-bit reference; counts None: one row per sequence."""
    counts = counts or [1] * len(p.lengths)
    starts = split_rows(counts)
    for b, (n, length) in enumerate(zip(counts, p.lengths)):
        rows = slice(starts[b], starts[b + 1])
        sees = causal(n, length) if mask is None else tree_sees(mask[rows], n, length)
        want, A = reference(q[rows], p.k[b], p.v[b], sees, p.attn.scale)
        check_rows(got[rows], want, A, f"sequence {b} ({n} rows, {length} tokens)")


def rotated(x: torch.Tensor, weight, eps, rope_rows: torch.Tensor):
    """float64 [T, heads, D] normalised per head and rotated, and the sum |x1| + |x2| of each pair."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt(x.pow(2).mean(dim=-1, keepdim=True) + eps) * weight.double()
    D = x.shape[-1]
    cos, sin = rope_rows.double().unsqueeze(1).split(D // 2, dim=-1)
    a, b = x[..., :D // 2], x[..., D // 2:]
    both = a.abs() + b.abs()
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1), torch.cat([both, both], dim=-1)
