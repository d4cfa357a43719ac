"""Performance cases of what serving adds to the attention half of a decoder layer: caches that keep only the
tokens that attention weighs most, positions with several axes, and adapters of many requests.

A case is one pass of one kind (``op``) over one layer:

  weigh     causal attention of each sequence's last ``queries`` tokens over its part of the cache, and beside it
            the weights that each cached token got from the last ``last`` of them, summed over the rows and over the
            query heads that share a key / value head and added to what earlier calls gave it
  evict     of each sequence's cache, ``budget`` tokens kept per key / value head: the ``recent`` last ones and
            those of the others with the largest weights; kept tokens fill the places of evicted ones, and what the
            cache holds of the kept ones is read back
  write     queries and keys of ``seqs`` x ``queries`` new tokens normalised per head (``norm``) and rotated by
            positions on three axes (time, height, width), keys and values stored, and read back
  adapters  low-rank adapters added to a projection's output: each sequence's tokens take one of ``adapters`` of
            rank up to ``rank`` (odd ones half of it), every eighth sequence none

``heads`` / ``kv_heads`` / ``dim`` / ``hidden``: 32/4/128/2048 with head norms is Qwen3-30B-A3B, 32/8/128/4096
Mixtral-8x7B, 16/16/128/2048 Qwen1.5-MoE-A2.7B.  ``cache`` is its format, ``page`` the tokens of a page.
``context`` is the longest sequence, new tokens included; where ``ragged``, the others are shorter (down to a
quarter), and so are their new tokens.

The cache: keys [pages, kv_heads, page, dim], values [pages, kv_heads, page / U, dim, U] with U = 16 bytes'
worth of tokens (8 bf16, 16 int8), and for int8 one fp32 scale per token and head, [pages, kv_heads, page].
Slot s is token s % page of page s // page.  Weights: fp32 [seqs, kv_heads, at least context].
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

EPS = 1e-6
THETA = 1e6
MODELS = {  # heads, kv_heads, dim, head norms, hidden
    "qwen3": (32, 4, 128, True, 2048),
    "mixtral": (32, 8, 128, False, 4096),
    "qwen15": (16, 16, 128, False, 2048),
    "small": (14, 2, 64, True, 896),
}


def _case(name, op, model, *, seqs, queries, context=0, cache="bf16", page=64, ragged=False, **more):
    heads, kv_heads, dim, norm, hidden = MODELS[model]
    c = {"op": op, "heads": heads, "kv_heads": kv_heads, "dim": dim, "norm": norm, "hidden": hidden, "cache": cache,
         "page": page, "seqs": seqs, "queries": queries, "context": max(context, queries), "ragged": ragged}
    c.update(more)
    return dict({"name": name}, **c) if name else c


def listed():
    return [
        # one chat request, one token
        _case("weigh_one_qwen3_bf16", "weigh", "qwen3", seqs=1, queries=1, context=517, last=1),
        # a full serving batch at mixed lengths
        _case("weigh_batch_qwen3_int8", "weigh", "qwen3", seqs=64, queries=1, context=8192, cache="int8", page=128,
              ragged=True, last=1),
        # a prompt whose every token counts
        _case("weigh_prompt_qwen3_bf16", "weigh", "qwen3", seqs=1, queries=8192, context=8192, last=8192),
        # the last chunks of three prompts, whose last 64 tokens say what the rest is worth
        _case("weigh_chunk_mixtral_int8", "weigh", "mixtral", seqs=3, queries=1021, context=9000, cache="int8",
              ragged=True, last=64),
        # a request that has grown 64 tokens past its budget
        _case("evict_one_qwen3_bf16", "evict", "qwen3", seqs=1, queries=1, context=2112, budget=2048, recent=128),
        # one long prompt brought to its budget
        _case("evict_prompt_mixtral_bf16", "evict", "mixtral", seqs=1, queries=1, context=30011, budget=4096,
              recent=256, page=256),
        # a batch of prompts brought to theirs; the shorter ones are below it
        _case("evict_batch_qwen3_int8", "evict", "qwen3", seqs=64, queries=1, context=8190, cache="int8", page=128,
              ragged=True, budget=2500, recent=100),
        # a decode step of 16 requests stores one token each
        _case("write_decode_qwen3_int8", "write", "qwen3", seqs=16, queries=1, context=4096, cache="int8",
              interleaved=True),
        # prompts with images and a video
        _case("write_prompt_mixtral_bf16", "write", "mixtral", seqs=3, queries=5003, context=5003, ragged=True,
              interleaved=False),
        # one request with an adapter, one token, beside the queries', keys' and values' projection
        _case("adapters_one_qwen3", "adapters", "qwen3", seqs=1, queries=1, adapters=4, rank=16, part="qkv"),
        # a full serving batch beside the output projection
        _case("adapters_batch_mixtral", "adapters", "mixtral", seqs=64, queries=1, adapters=24, rank=32, part="o"),
        # prompts of eight requests
        _case("adapters_prompts_mixtral", "adapters", "mixtral", seqs=8, queries=1501, adapters=8, rank=64,
              part="qkv", ragged=True),
    ]


def draw(rng: random.Random):
    def size(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    op = rng.choice(["weigh", "weigh", "weigh", "evict", "evict", "write", "adapters", "adapters"])
    model, cache, page = rng.choice(list(MODELS)), rng.choice(["bf16", "int8"]), rng.choice([64, 128, 256])
    seqs, ragged = size(1, 64), rng.random() < 0.7
    more = {}
    if op == "weigh" and rng.random() < 0.5:
        queries, context = 1, min(size(1, 262144 // seqs), 32768)
        more = {"last": 1}
    elif op == "weigh":
        seqs = size(1, 8)
        queries = size(2, 4096 // seqs)
        context = queries + size(1, 8192 // seqs)
        more = {"last": rng.choice([queries, size(1, queries)])}
    elif op == "evict":
        queries, context = 1, min(size(2, 262144 // seqs), 32768)
        budget = size(1, context)
        more = {"budget": budget, "recent": min(budget, size(1, 512))}
    elif op == "write":
        queries = size(1, max(1, 8192 // seqs))
        context = queries + size(1, 4096)
        more = {"interleaved": rng.random() < 0.5}
    else:
        queries = size(1, max(1, 8192 // seqs)) if rng.random() < 0.5 else 1
        context = queries
        more = {"adapters": size(1, 32), "rank": size(1, 64), "part": rng.choice(["qkv", "o"])}
    return _case("", op, model, seqs=seqs, queries=queries, context=context, cache=cache, page=page, ragged=ragged,
                 **more)


# ------------------------------------------------------------------ sizes
def _lengths(case):
    """(new tokens, length) of each sequence: the first is the longest."""
    cuts = [1.0 - 0.75 * ((b * 37) % 64) / 64.0 if case["ragged"] else 1.0 for b in range(case["seqs"])]
    news = [max(1, int(case["queries"] * cut)) for cut in cuts]
    return [(n, max(n, int(case["context"] * cut))) for n, cut in zip(news, cuts)]


def _adapter_of(case):
    """The adapter of each sequence, -1: none."""
    return [-1 if b % 8 == 7 else (b * 5 + b // 8) % case["adapters"] for b in range(case["seqs"])]


def _rank_of(case, adapter):
    return max(1, case["rank"] // 2) if adapter % 2 else case["rank"]


def _parts(case):
    """Width of what the adapters read, and of the outputs that they share a reading for."""
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    return (case["hidden"], (hq * d, hk * d, hk * d)) if case["part"] == "qkv" else (hq * d, (case["hidden"],))


def _sections(case):
    """Frequencies of time, height and width."""
    half = case["dim"] // 2
    return (half - 2 * (3 * half // 8), 3 * half // 8, 3 * half // 8)


def _moved(case, length):
    """(kept, at most so many moved into evicted places, the recent ones)"""
    keep = min(case["budget"], length)
    window = min(case["recent"], keep)
    front = keep - window
    return keep, min(front, length - keep), window if length > keep else 0


def work(case):
    lengths = _lengths(case)
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    tokens, total = sum(n for n, _ in lengths), sum(length for _, length in lengths)
    row = 2 * hk * (d * 2 if case["cache"] == "bf16" else d + 4)   # one token of the cache
    out = 2 * hk * d * 2                                           # the same in the activations' type
    if case["op"] == "weigh":
        pairs = sum(n * (length - n) + n * (n + 1) // 2 for n, length in lengths)
        return {"bytes": total * (row + 8 * hk) + 2 * tokens * hq * d * 2, "flops": 4 * d * hq * pairs}
    if case["op"] == "evict":
        kept = sum(_moved(case, length)[0] for _, length in lengths)
        window = sum(_moved(case, length)[2] for _, length in lengths)
        # (how many kept tokens lie behind their budget depends on the weights: a share of them as if spread evenly)
        into = sum(m * min(1.0, k / length) for (k, m, _), (_, length) in
                   zip((_moved(case, length) for _, length in lengths), lengths))
        nbytes = 4 * hk * (total + kept) + 2 * row * (into + window) + kept * (row + out + 8)
        return {"bytes": int(nbytes), "flops": total * hk}
    if case["op"] == "write":
        nbytes = tokens * ((2 * hq + 2 * hk) * d * 2 + d * 4 + 32 + 2 * row + out)
        return {"bytes": nbytes, "flops": tokens * (hq + 2 * hk) * d * 8}
    width, outs = _parts(case)
    used = {a for a in _adapter_of(case) if a >= 0}
    weights = sum(_rank_of(case, a) * 2 * (len(outs) * width + sum(outs)) for a in used)
    adapted = [(n, _rank_of(case, a)) for (n, _), a in zip(lengths, _adapter_of(case)) if a >= 0]
    flops = sum(2 * n * r * (len(outs) * width + sum(outs)) for n, r in adapted)
    return {"bytes": tokens * (width * 2 + 2 * sum(outs) * 2 + 8) + weights, "flops": flops}


# ------------------------------------------------------------------ inputs
def _rope_table(positions, dim, dtype=torch.float32):
    inv = THETA ** (-torch.arange(0, dim, 2, device="cuda", dtype=torch.float64) / dim)
    angle = positions.double().unsqueeze(-1) * inv
    return torch.cat([angle.cos(), angle.sin()], dim=-1).to(dtype)


def _axes(case):
    """The axis of each frequency: in three runs, or dealt out in turn while an axis has any left."""
    left, out = list(_sections(case)), []
    if not case["interleaved"]:
        return [axis for axis, count in enumerate(left) for _ in range(count)]
    while any(left):
        for axis in range(3):
            if left[axis]:
                left[axis] -= 1
                out.append(axis)
    return out


def _media_positions(first, n):
    """Positions [3, n] of n tokens after ``first`` others: text, where one number serves all axes, and in turn
    images and videos of t x h x w patches, after which text goes on behind the largest number."""
    spans, at, i = [], first, 0
    shapes = [(1, 12, 16), (4, 8, 10), (1, 24, 20)]
    while sum(x.shape[1] for x in spans) < n:
        spans.append((at + torch.arange(37)).expand(3, -1))
        t, h, w = shapes[i % 3]
        grid = torch.stack(torch.meshgrid(torch.arange(t), torch.arange(h), torch.arange(w), indexing="ij"))
        spans.append(at + 37 + grid.reshape(3, -1))
        at, i = at + 37 + max(t, h, w), i + 1
    return torch.cat(spans, dim=1)[:, :n]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    hq, hk, d, page, op = case["heads"], case["kv_heads"], case["dim"], case["page"], case["op"]
    lengths = _lengths(case)
    seqs, tokens = case["seqs"], sum(n for n, _ in lengths)

    def randn(*shape):
        return torch.empty(*shape, dtype=torch.bfloat16, device="cuda").normal_(generator=g)

    s = {"case": case, "tokens": tokens}
    s["n"] = torch.tensor([n for n, _ in lengths], dtype=torch.int32, device="cuda")
    seq_of = torch.repeat_interleave(torch.arange(seqs, device="cuda"), s["n"].long())
    if op == "adapters":
        width, outs = _parts(case)
        n, r = case["adapters"], case["rank"]
        s["x"], s["base"] = randn(tokens, width), randn(tokens, sum(outs))
        s["index"] = torch.tensor(_adapter_of(case), device="cuda")[seq_of]
        ranks = torch.tensor([_rank_of(case, a) for a in range(n)], device="cuda")
        inside = (torch.arange(r, device="cuda") < ranks.unsqueeze(1)).to(torch.bfloat16)
        s["a"] = randn(n, len(outs), r, width).mul_(width ** -0.5).mul_(inside.view(n, 1, r, 1))
        s["b"] = randn(n, sum(outs), r).mul_(r ** -0.5).mul_(inside.view(n, 1, r))
        s["scales"] = torch.empty(n, len(outs), device="cuda").uniform_(0.25, 2.0, generator=g)
        if own:
            s["adapters"] = _adapters(case, s)
        return s

    width = (case["context"] + page - 1) // page
    pages = seqs * width + 3
    s["lens"] = torch.tensor([length for _, length in lengths], dtype=torch.int32, device="cuda")
    s["starts"] = torch.nn.functional.pad(s["n"].cumsum(0), (1, 0)).to(torch.int32)
    s["max_n"], s["max_len"] = max(n for n, _ in lengths), max(length for _, length in lengths)
    table = torch.randperm(pages, generator=g, device="cuda")[:seqs * width].view(seqs, width)
    s["table"] = table.to(torch.int32)
    # the cache as earlier calls left it
    unit = 8 if case["cache"] == "bf16" else 16
    shapes = (pages, hk, page, d), (pages, hk, page // unit, d, unit)
    if case["cache"] == "bf16":
        s["k"], s["v"] = randn(*shapes[0]), randn(*shapes[1])
        s["ks"] = s["vs"] = None
    else:
        s["k"], s["v"] = (torch.randint(-127, 128, shape, generator=g, dtype=torch.int8, device="cuda")
                          for shape in shapes)
        s["ks"], s["vs"] = (torch.empty(pages, hk, page, device="cuda").uniform_(0.008, 0.024, generator=g)
                            for _ in range(2))

    def slots_of(seq, position):
        return table[seq, position // page] * page + position % page

    if op in ("weigh", "evict"):
        # sums of earlier calls: most of it on few tokens, none on some
        w = torch.empty(seqs, hk, width * page, device="cuda").exponential_(generator=g).pow_(3)
        w.mul_(torch.rand(w.shape, generator=g, device="cuda") > 0.1)
        inside = torch.arange(width * page, device="cuda") < (s["lens"] - s["n"] * (op == "weigh")).view(seqs, 1, 1)
        s["weights"] = w.masked_fill_(~inside, 0.0)
    nth = torch.arange(tokens, device="cuda") - s["starts"].long()[seq_of]
    place = (s["lens"].long() - s["n"].long())[seq_of] + nth
    if op == "weigh":
        s["q"] = 2 * randn(tokens, hq, d)
    elif op == "evict":
        s["budgets"] = torch.full((seqs,), case["budget"], dtype=torch.int32, device="cuda")
        kept = torch.tensor([_moved(case, length)[0] for _, length in lengths], device="cuda")
        s["max_kept"] = int(kept.max())
        seq = torch.repeat_interleave(torch.arange(seqs, device="cuda"), kept)
        first = torch.nn.functional.pad(kept.cumsum(0), (1, 0))
        s["slots"] = slots_of(seq, torch.arange(seq.numel(), device="cuda") - first[seq])
    else:
        qkv = randn(tokens, (hq + 2 * hk) * d)  # one projection's output, its heads side by side
        s["q"], s["new_k"], s["new_v"] = (x.unflatten(1, (-1, d)) for x in
                                          qkv.split([hq * d, hk * d, hk * d], dim=1))
        s["axes"] = _axes(case)
        s["axis_of"] = torch.tensor(s["axes"], device="cuda")
        s["positions"] = torch.cat([_media_positions(length - n, n) for n, length in lengths], dim=1).cuda()
        s["slots"] = slots_of(seq_of, place)
        s["rope"] = _rope_table(torch.arange(case["context"] + 1, device="cuda"), d)
        s["q_norm"] = s["k_norm"] = None
        if case["norm"]:
            s["q_norm"], s["k_norm"] = 1 + 0.1 * randn(d), 1 + 0.1 * randn(d)
    if own:
        s["attention"] = _handle(case, s)
    return s


def _package():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nano-ktrans_amd")
    if path not in sys.path:
        sys.path.insert(1, path)
    import nano_ktrans_amd

    return nano_ktrans_amd


def _handle(case, s):
    """The layer's cache as a serving program holds it, with the same contents."""
    attention = _package().NativeAttention(
        num_heads=case["heads"], num_kv_heads=case["kv_heads"], head_dim=case["dim"], num_pages=s["k"].shape[0],
        page_size=case["page"], cache_format=case["cache"])
    attention.k_cache.copy_(s["k"])
    attention.v_cache.copy_(s["v"])
    if s["ks"] is not None:
        attention.k_scales.copy_(s["ks"])
        attention.v_scales.copy_(s["vs"])
    return attention


def _adapters(case, s):
    """The adapters as a serving program holds them."""
    width, outs = _parts(case)
    adapters = _package().NativeAdapters(num_adapters=case["adapters"], in_features=width, out_features=outs,
                                         max_rank=case["rank"])
    for i in range(case["adapters"]):
        r = _rank_of(case, i)
        for part, b in enumerate(s["b"][i].split(outs)):
            adapters.load(i, s["a"][i, part, :r], b[:, :r], scale=float(s["scales"][i, part]), part=part)
    return adapters


# ------------------------------------------------------------------ one pass
@torch.no_grad()
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    op = s["case"]["op"]
    if op == "adapters":
        return {"out": s["adapters"].forward(s["x"], s["base"], s["index"])}
    a = s["attention"]
    if op == "write":
        q = a.write(s["q"], s["new_k"], s["new_v"], s["positions"], s["slots"], s["rope"], q_norm=s["q_norm"],
                    k_norm=s["k_norm"], eps=EPS, axes=s["axes"])
        k, v = a.read(s["slots"])
        return {"q": q, "k": k, "v": v}
    if op == "evict":
        lens, weights = a.evict(s["table"], s["lens"], s["weights"], s["budgets"], s["case"]["recent"],
                                max_seq_len=s["max_len"])
        k, v = a.read(s["slots"])
        return {"lens": lens, "weights": weights, "k": k, "v": v}
    if s["max_n"] == 1:  # a decode step: one query per sequence
        out = a.forward_weights(s["q"], s["weights"], s["table"], s["lens"], max_seq_len=s["max_len"])
    else:
        out = a.forward_weights(s["q"], s["weights"], s["table"], s["lens"], s["starts"], max_queries=s["max_n"],
                                max_seq_len=s["max_len"], last=s["case"]["last"])
    return {"out": out, "weights": s["weights"]}


def _norm_rope(x, weight, cos, sin):
    """fp32 [T, heads, D], normalised per head where there is a weight, and rotated."""
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + EPS) * weight.float()
    a, b = x.chunk(2, dim=-1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)


def _place(s, slots):
    """Index of the slots' rows in the keys [pages, page] and the values [pages, units, in a unit]."""
    page, unit = s["case"]["page"], s["v"].shape[4]
    p, r = slots // page, slots % page
    return p, r, r // unit, r % unit


def _quantized(x):
    """int8 codes and scales of fp32 rows."""
    scale = x.abs().amax(dim=-1, keepdim=True) / 127
    scale = torch.where(scale > 0, scale, 1.0)
    return torch.round(x / scale).to(torch.int8), scale.squeeze(-1)


def _store(s, slots, k, v):
    """fp32 rows [T, kv_heads, D] into the cache."""
    p, r, u, i = _place(s, slots)
    if s["ks"] is not None:
        (k, s["ks"][p, :, r]), (v, s["vs"][p, :, r]) = _quantized(k), _quantized(v)
    s["k"][p, :, r] = k.to(s["k"].dtype)
    s["v"][p, :, u, :, i] = v.to(s["v"].dtype)


def _load(s, slots):
    """fp32 rows [T, kv_heads, D] of the cache."""
    p, r, u, i = _place(s, slots)
    k, v = s["k"][p, :, r].float(), s["v"][p, :, u, :, i].float()
    if s["ks"] is not None:
        k, v = k * s["ks"][p, :, r].unsqueeze(-1), v * s["vs"][p, :, r].unsqueeze(-1)
    return k, v


def _read_back(s):
    k, v = _load(s, s["slots"])
    return {"k": k.to(torch.bfloat16), "v": v.to(torch.bfloat16)}


def _run_plain(s):
    return {"adapters": _plain_adapters, "write": _plain_write, "evict": _plain_evict,
            "weigh": _plain_weigh}[s["case"]["op"]](s)


def _plain_adapters(s):
    """One product with all adapters' A, what is not the token's own adapter's set to zero, one with all B."""
    (n, parts, r, width), outs = s["a"].shape, _parts(s["case"])[1]
    low = torch.matmul(s["x"].float(), s["a"].float().view(n * parts * r, width).T).view(-1, n, parts, r)
    mine = s["index"].view(-1, 1) == torch.arange(n, device="cuda")
    low = torch.where(mine.view(-1, n, 1, 1), low * s["scales"].view(1, n, parts, 1), 0.0)
    up = s["b"].float().permute(0, 2, 1).reshape(n * r, -1).split(outs, dim=1)
    more = [torch.matmul(low[:, :, p].reshape(-1, n * r), b) for p, b in enumerate(up)]
    return {"out": (s["base"].float() + torch.cat(more, dim=1)).to(torch.bfloat16)}


def _plain_write(s):
    d = s["case"]["dim"]
    where = s["positions"][s["axis_of"]].T                     # [T, D / 2]: each frequency's position
    cos, sin = (s["rope"][:, half].gather(0, where).unsqueeze(1) for half in (slice(0, d // 2), slice(d // 2, d)))
    q = _norm_rope(s["q"], s["q_norm"], cos, sin)
    _store(s, s["slots"], _norm_rope(s["new_k"], s["k_norm"], cos, sin), s["new_v"].float())
    return dict(_read_back(s), q=q.to(torch.bfloat16))


def _plain_evict(s):
    case, w = s["case"], s["weights"]
    page, width, most = case["page"], w.shape[2], s["max_kept"]
    lens = s["lens"].long().view(-1, 1, 1)
    keep = torch.minimum(lens, s["budgets"].view(-1, 1, 1))
    window = keep.clamp(max=case["recent"])
    others, front = lens - window, keep - window
    place = torch.arange(width, device="cuda").expand_as(w)
    order = torch.where(place < others, w, -1.0).sort(dim=2, descending=True, stable=True).indices
    kept = torch.zeros_like(w, dtype=torch.bool).scatter_(2, order, place < front)
    # places of evicted tokens and kept tokens behind the front, the i-th of each at i
    hole, behind = ~kept & (place < front), kept & (place >= front)
    behind = behind.to(torch.uint8).sort(dim=2, descending=True, stable=True).indices
    nth = hole.long().cumsum(dim=2) - 1
    source = torch.where(hole, behind.gather(2, nth.clamp(min=0)), place)
    source = torch.where(place >= front, (others + place - front).clamp(max=width - 1), source)
    inside = place < keep
    weights = torch.where(inside, w.gather(2, source), 0.0)
    table = s["table"].long()
    seq, head = (torch.arange(x, device="cuda") for x in w.shape[:2])
    seq, head = seq.view(-1, 1, 1).expand(-1, w.shape[1], most), head.view(1, -1, 1).expand(w.shape[0], -1, most)
    inside = inside[:, :, :most]
    seq, head, to, at = (x[inside] for x in (seq, head, place[:, :, :most], source[:, :, :most]))
    (p, r, u, i), (tp, tr, tu, ti) = (_place(s, table[seq, x // page] * page + x % page) for x in (at, to))
    s["k"][tp, head, tr] = s["k"][p, head, r]
    s["v"][tp, head, tu, :, ti] = s["v"][p, head, u, :, i]
    if s["ks"] is not None:
        s["ks"][tp, head, tr] = s["ks"][p, head, r]
        s["vs"][tp, head, tr] = s["vs"][p, head, r]
    return dict(_read_back(s), lens=keep.view(-1).to(torch.int32), weights=weights)


def _plain_weigh(s):
    """Every sequence padded to the longest, scores in 32 bits."""
    case = s["case"]
    page, seqs, n, length = case["page"], case["seqs"], s["max_n"], s["max_len"]
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    group = hq // hk
    position = torch.arange(length, device="cuda")
    k, v = _load(s, (s["table"].long()[:, position // page] * page + position % page).view(-1))
    inside = position < s["lens"].unsqueeze(1)                                    # [seqs, length]
    k = k.view(seqs, length, hk, d).permute(0, 2, 3, 1)
    v = v.view(seqs, length, hk, d).permute(0, 2, 1, 3).masked_fill(~inside.view(seqs, 1, length, 1), 0.0)
    nth = torch.arange(n, device="cuda")
    row = (s["starts"][:-1].unsqueeze(1) + nth).clamp(max=s["tokens"] - 1).long()  # [seqs, n]
    real = nth < s["n"].unsqueeze(1)
    context = (s["lens"] - s["n"]).view(seqs, 1, 1)
    sees = (position <= context + nth.view(1, n, 1)) & inside.unsqueeze(1)
    q = s["q"][row].float().view(seqs, n, hk, group, d).permute(0, 2, 1, 3, 4).reshape(seqs, hk, n * group, d)
    score = torch.matmul(q, k).mul_(d ** -0.5).view(seqs, hk, n, group, length)
    score = score.masked_fill_(~sees.view(seqs, 1, n, 1, length), -math.inf)
    top = score.amax(dim=-1, keepdim=True)
    p = score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(dim=-1, keepdim=True)
    p = p.div_(torch.where(total > 0, total, 1.0)).view(seqs, hk, n * group, length)
    out = torch.matmul(p, v)
    out = out.view(seqs, hk, n, group, d).permute(0, 2, 1, 3, 4).reshape(seqs, n, hq, d)
    counts = real & (nth >= s["n"].unsqueeze(1) - case["last"])
    p = p.view(seqs, hk, n, group, length).masked_fill_(~counts.view(seqs, 1, n, 1, 1), 0.0)
    s["weights"][:, :, :length] += p.view(seqs, hk, n * group, length).sum(dim=2, dtype=torch.float64)
    return {"out": out[real].to(torch.bfloat16), "weights": s["weights"]}


# ------------------------------------------------------------------ the same in 64 bits
def _value(s, slot, which):
    """float64 rows of the cache at the slots, [T, kv_heads, D], from its layout."""
    if which == "k":
        flat = s["k"].transpose(1, 2).reshape(-1, s["k"].shape[1], s["k"].shape[3])
        scales = s["ks"]
    else:
        flat = s["v"].permute(0, 2, 4, 1, 3).reshape(-1, s["v"].shape[1], s["v"].shape[3])
        scales = s["vs"]
    x = flat[slot].double()
    if scales is not None:
        x = x * scales.double().transpose(1, 2).reshape(-1, scales.shape[1])[slot].unsqueeze(-1)
    return x


def _sequence_values(s, b, length):
    """float64 keys and values of sequence b, [length, kv_heads, D]."""
    page = s["case"]["page"]
    pages = s["table"][b].long()[:(length + page - 1) // page]
    part = {name: None if s[name] is None else s[name][pages] for name in ("k", "v", "ks", "vs")}
    every = torch.arange(length, device="cuda")
    return _value(part, every, "k"), _value(part, every, "v")


def _exact_rotated(x, weight, turn):
    x = x.double()
    if weight is not None:
        x = x / (x.pow(2).mean(dim=-1, keepdim=True) + EPS).sqrt() * weight.double()
    half = x.shape[-1] // 2
    z = torch.complex(x[..., :half], x[..., half:]) * turn.unsqueeze(1)
    return torch.cat([z.real, z.imag], dim=-1)


def _exact_stored(x, fmt):
    if fmt == "bf16":
        return x
    step = x.abs().amax(dim=-1, keepdim=True) / 127
    return torch.where(step > 0, torch.round(x / step) * step, 0.0)


def _exact_adapters(case, s):
    out = s["base"].double()
    outs = _parts(case)[1]
    for i in range(case["adapters"]):
        rows = (s["index"] == i).nonzero().squeeze(1)
        at = 0
        for part, columns in enumerate(outs):
            low = s["x"][rows].double() @ s["a"][i, part].double().T
            out[rows, at:at + columns] += float(s["scales"][i, part]) * (low @ s["b"][i, at:at + columns].double().T)
            at += columns
    return {"out": out}


def _exact_write(case, s):
    half = case["dim"] // 2
    angle = torch.stack([s["positions"][axis].double() * THETA ** (-i / half) for i, axis in enumerate(s["axes"])], 1)
    turn = torch.polar(torch.ones_like(angle), angle)
    return {"q": _exact_rotated(s["q"], s["q_norm"], turn),
            "k": _exact_stored(_exact_rotated(s["new_k"], s["k_norm"], turn), case["cache"]),
            "v": _exact_stored(s["new_v"].double(), case["cache"])}


def _exact_evict(case, s):
    keys, values = [], []
    weights = torch.zeros_like(s["weights"], dtype=torch.float64)
    for b, (_, length) in enumerate(_lengths(case)):
        keep = min(case["budget"], length)
        window = min(case["recent"], keep)
        front = keep - window
        k, v = _sequence_values(s, b, length)
        for h in range(case["kv_heads"]):
            w = s["weights"][b, h, :length].double()
            heavy = w[:length - window].cpu().numpy()
            best = sorted((-heavy).argsort(kind="stable")[:front].tolist())
            stays = set(x for x in best if x < front)
            coming = iter(x for x in best if x >= front)
            source = [i if i in stays else next(coming) for i in range(front)]
            source = torch.tensor(source + list(range(length - window, length)), device="cuda", dtype=torch.int64)
            weights[b, h, :keep] = w[source]
            k[:keep, h], v[:keep, h] = k[source, h], v[source, h]
        keys.append(k[:keep])
        values.append(v[:keep])
    return {"lens": None, "weights": weights, "k": torch.cat(keys), "v": torch.cat(values)}


def _exact_weigh(case, s):
    d, group = case["dim"], case["heads"] // case["kv_heads"]
    starts = s["starts"].tolist()
    out = torch.zeros(s["tokens"], case["heads"], d, dtype=torch.float64, device="cuda")
    weights = s["weights"].double()
    for b, (n, length) in enumerate(_lengths(case)):
        keys, values = _sequence_values(s, b, length)
        mine = torch.arange(n, device="cuda").unsqueeze(1)
        hidden = torch.arange(length, device="cuda").unsqueeze(0) > length - n + mine
        for h in range(case["heads"]):
            q = s["q"][starts[b]:starts[b + 1], h].double()
            p = (q @ keys[:, h // group].T / math.sqrt(d)).masked_fill(hidden, -math.inf).softmax(dim=-1)
            out[starts[b]:starts[b + 1], h] = p @ values[:, h // group]
            weights[b, h // group, :length] += p[max(0, n - case["last"]):].sum(dim=0)
    return {"out": out, "weights": weights}


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    return {"adapters": _exact_adapters, "write": _exact_write, "evict": _exact_evict,
            "weigh": _exact_weigh}[case["op"]](case, s)
