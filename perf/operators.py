"""Performance cases of the attention half of a decoder layer: the calls that a program serving a
mixture-of-experts model makes between two MoE layers, through ``NativeAttention``.

A case is one pass of one kind (``op``) over one layer's paged cache:

  write   queries and keys of ``seqs`` x ``queries`` new tokens normalised per head (``norm``) and rotated, keys
          and values stored in the cache, and what the cache holds of them read back
  read    the keys and values of whole sequences, in the activations' type
  attend  causal attention of each sequence's last ``queries`` tokens over its part of the cache
  tree    the same for drafted tokens that see the context and their own ancestors
  keep    the accepted nodes of a drafted tree moved to the end of the context, and the drafted part read back

``heads`` / ``kv_heads`` / ``dim``: 32/4/128 with head norms is Qwen3-30B-A3B, 32/8/128 Mixtral-8x7B, 16/16/128
Qwen1.5-MoE-A2.7B.  ``cache`` is its format, ``page`` the tokens of a page.  ``context`` is the longest
sequence, new tokens included; where ``ragged``, the others are shorter (down to a quarter), and so are
their new tokens.

The cache: keys [pages, kv_heads, page, dim], values [pages, kv_heads, page / U, dim, U] with U = 16 bytes'
worth of tokens (8 bf16, 16 int8), and for int8 one fp32 scale per token and head, [pages, kv_heads, page].
Slot s is token s % page of page s // page.
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
MODELS = {  # heads, kv_heads, dim, head norms
    "qwen3": (32, 4, 128, True),
    "mixtral": (32, 8, 128, False),
    "qwen15": (16, 16, 128, False),
    "small": (14, 2, 64, True),
}


def _case(name, op, model, cache, *, seqs, queries, context, page=64, ragged=False):
    heads, kv_heads, dim, norm = MODELS[model]
    c = {"op": op, "heads": heads, "kv_heads": kv_heads, "dim": dim, "norm": norm, "cache": cache, "page": page,
         "seqs": seqs, "queries": queries, "context": context, "ragged": ragged}
    return dict({"name": name}, **c) if name else c


def listed():
    return [
        # a decode step of 16 requests stores one token each
        _case("write_decode_qwen3_int8", "write", "qwen3", "int8", seqs=16, queries=1, context=4096),
        # a prompt of 16384 tokens, a head of keys for every head of queries
        _case("write_prompt_qwen15_bf16", "write", "qwen15", "bf16", seqs=1, queries=16384, context=16384, page=256),
        # one short request's cache handed on (to another process, to a prefix store)
        _case("read_one_qwen3_int8", "read", "qwen3", "int8", seqs=1, queries=1, context=777),
        # eight long requests' caches handed on
        _case("read_many_mixtral_bf16", "read", "mixtral", "bf16", seqs=8, queries=1, context=8100, ragged=True),
        # the smallest step: one chat request, one token
        _case("decode_one_qwen3_bf16", "attend", "qwen3", "bf16", seqs=1, queries=1, context=517),
        # a full serving batch at mixed lengths
        _case("decode_batch_qwen3_int8", "attend", "qwen3", "int8", seqs=64, queries=1, context=8192, page=128,
              ragged=True),
        # a long prompt at once
        _case("prompt_qwen3_bf16", "attend", "qwen3", "bf16", seqs=1, queries=8192, context=8192),
        # chunks of three prompts, the earlier chunks in the cache
        _case("chunk_mixtral_int8", "attend", "mixtral", "int8", seqs=3, queries=1021, context=9000, ragged=True),
        # one request verifies a draft of 12 tokens
        _case("tree_one_qwen3_bf16", "tree", "qwen3", "bf16", seqs=1, queries=12, context=2000),
        # a batch of requests verifies drafts of up to 48 tokens
        _case("tree_batch_mixtral_int8", "tree", "mixtral", "int8", seqs=16, queries=48, context=6000, ragged=True),
        # after which each keeps the accepted ones
        _case("keep_one_qwen3_bf16", "keep", "qwen3", "bf16", seqs=1, queries=12, context=2000),
        _case("keep_batch_mixtral_int8", "keep", "mixtral", "int8", seqs=64, queries=64, context=2500, ragged=True),
    ]


def draw(rng: random.Random):
    def size(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    op = rng.choice(["write", "read", "attend", "attend", "attend", "tree", "keep"])
    model, cache, page = rng.choice(list(MODELS)), rng.choice(["bf16", "int8"]), rng.choice([64, 128, 256])
    seqs, ragged = size(1, 64), rng.random() < 0.7
    if op == "write":
        queries = size(1, max(1, 8192 // seqs))
        context = queries + size(1, 4096)
    elif op == "read":
        queries, context = 1, size(2, 65536 // seqs)
    elif op == "attend" and rng.random() < 0.5:
        queries, context = 1, size(1, 262144 // seqs)
        context = min(context, 32768)
    elif op == "attend":
        seqs = size(1, 8)
        queries = size(2, 4096 // seqs)
        context = queries + size(1, 8192 // seqs)
    else:
        queries = size(2, 128)
        seqs = min(seqs, 1024 // queries)
        context = queries + size(1, 8192)
    return _case("", op, model, cache, seqs=max(1, seqs), queries=queries, context=context, page=page, ragged=ragged)


# ------------------------------------------------------------------ sizes
def _lengths(case):
    """(new tokens, length) of each sequence: the first is the longest."""
    out = []
    for b in range(case["seqs"]):
        cut = 1.0 - 0.75 * ((b * 37) % 64) / 64.0 if case["ragged"] else 1.0
        n = max(1, int(case["queries"] * cut))
        out.append((n, max(n, int(case["context"] * cut))))
    return out


def work(case):
    lengths = _lengths(case)
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    tokens, total = sum(n for n, _ in lengths), sum(length for _, length in lengths)
    row = 2 * hk * (d * 2 if case["cache"] == "bf16" else d + 4)   # one token of the cache
    out = 2 * hk * d * 2                                           # the same in the activations' type
    if case["op"] == "write":
        nbytes = tokens * ((2 * hq + 2 * hk) * d * 2 + d * 4 + 16 + 2 * row + out)
        return {"bytes": nbytes, "flops": tokens * (hq + 2 * hk) * d * 8}
    if case["op"] == "read":
        return {"bytes": total * (row + out + 8), "flops": total * 2 * hk * d}
    if case["op"] == "keep":
        moved = sum(_kept(n) for n, _ in lengths)
        return {"bytes": moved * 2 * row + tokens * (row + out + 8), "flops": tokens * 2 * hk * d}
    pairs = sum(n * (length - n) + n * (n + 1) // 2 for n, length in lengths)
    return {"bytes": total * row + 2 * tokens * hq * d * 2, "flops": 4 * d * hq * pairs}


def _kept(n):
    """Accepted nodes of a draft of n."""
    return max(1, min(n, 1 + n // 5))


# ------------------------------------------------------------------ inputs
def _rope_table(positions, dim, dtype=torch.float32):
    inv = THETA ** (-torch.arange(0, dim, 2, device="cuda", dtype=torch.float64) / dim)
    angle = positions.double().unsqueeze(-1) * inv
    return torch.cat([angle.cos(), angle.sin()], dim=-1).to(dtype)


def _trees(lengths, g):
    """Each drafted token's ancestors and itself as bits of int64 words, [tokens, words]."""
    most = max(n for n, _ in lengths)
    words = (most + 63) // 64
    seqs = len(lengths)
    reach = torch.randint(1, 9, (seqs, most), generator=g, device="cuda")
    sees = torch.zeros(seqs, most, words * 64, dtype=torch.bool, device="cuda")
    every = torch.arange(seqs, device="cuda")
    for i in range(most):
        parent = (i - reach[:, i]).clamp(min=0)
        if i:
            sees[:, i] = sees[every, parent]
        sees[:, i, i] = True
    weight = torch.ones(64, dtype=torch.int64, device="cuda") << torch.arange(64, device="cuda")
    bits = (sees.view(seqs, most, words, 64) * weight).sum(dim=-1)
    rows = torch.arange(most, device="cuda") < torch.tensor([n for n, _ in lengths], device="cuda").unsqueeze(1)
    return bits[rows].contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    hq, hk, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    lengths = _lengths(case)
    seqs, width = case["seqs"], (case["context"] + page - 1) // page
    tokens = sum(n for n, _ in lengths)
    pages = seqs * width + 3

    def randn(*shape):
        return torch.empty(*shape, dtype=torch.bfloat16, device="cuda").normal_(generator=g)

    s = {"case": case, "tokens": tokens}
    s["n"] = torch.tensor([n for n, _ in lengths], dtype=torch.int32, device="cuda")
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

    seq_of = torch.repeat_interleave(torch.arange(seqs, device="cuda"), s["n"].long())
    nth = torch.arange(tokens, device="cuda") - s["starts"].long()[seq_of]
    place = (s["lens"].long() - s["n"].long())[seq_of] + nth
    if case["op"] == "write":
        qkv = randn(tokens, (hq + 2 * hk) * d)  # one projection's output, its heads side by side
        s["q"], s["new_k"], s["new_v"] = (x.unflatten(1, (-1, d)) for x in
                                          qkv.split([hq * d, hk * d, hk * d], dim=1))
        s["positions"], s["slots"] = place, slots_of(seq_of, place)
        s["rope"] = _rope_table(torch.arange(case["context"], device="cuda"), d)
        s["q_norm"] = s["k_norm"] = None
        if case["norm"]:
            s["q_norm"], s["k_norm"] = 1 + 0.1 * randn(d), 1 + 0.1 * randn(d)
    elif case["op"] == "read":
        lens = s["lens"].long()
        seq = torch.repeat_interleave(torch.arange(seqs, device="cuda"), lens)
        first = torch.nn.functional.pad(lens.cumsum(0), (1, 0))
        s["slots"] = slots_of(seq, torch.arange(seq.numel(), device="cuda") - first[seq])
    elif case["op"] == "keep":
        s["context"] = s["lens"] - s["n"]
        s["counts"] = torch.tensor([_kept(n) for n, _ in lengths], dtype=torch.int32, device="cuda")
        most = int(max(_kept(n) for n, _ in lengths))
        mix = torch.rand(seqs, s["max_n"], generator=g, device="cuda")
        mix = mix.masked_fill(torch.arange(s["max_n"], device="cuda") >= s["n"].unsqueeze(1), 2.0)
        picked = mix.argsort(dim=1)[:, :most]
        picked = picked.masked_fill(torch.arange(most, device="cuda") >= s["counts"].unsqueeze(1), s["max_n"])
        s["kept"] = picked.sort(dim=1).values.to(torch.int32)  # ascending; behind the count: not read
        s["slots"] = slots_of(seq_of, place)
    else:
        s["q"] = 2 * randn(tokens, hq, d)
        if case["op"] == "tree":
            s["tree"] = _trees(lengths, g)
    if own:
        s["attention"] = _handle(case, s)
    return s


def _handle(case, s):
    """The layer's cache as a serving program holds it, with the same contents."""
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nano-ktrans_amd")
    if path not in sys.path:
        sys.path.insert(1, path)
    from nano_ktrans_amd import NativeAttention

    attention = NativeAttention(num_heads=case["heads"], num_kv_heads=case["kv_heads"], head_dim=case["dim"],
                                num_pages=s["k"].shape[0], page_size=case["page"], cache_format=case["cache"])
    attention.k_cache.copy_(s["k"])
    attention.v_cache.copy_(s["v"])
    if s["ks"] is not None:
        attention.k_scales.copy_(s["ks"])
        attention.v_scales.copy_(s["vs"])
    return attention


# ------------------------------------------------------------------ one pass
@torch.no_grad()
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    a, op = s["attention"], s["case"]["op"]
    if op == "write":
        q = a.write(s["q"], s["new_k"], s["new_v"], s["positions"], s["slots"], s["rope"], q_norm=s["q_norm"],
                    k_norm=s["k_norm"], eps=EPS)
        k, v = a.read(s["slots"])
        return {"q": q, "k": k, "v": v}
    if op == "read":
        k, v = a.read(s["slots"])
        return {"k": k, "v": v}
    if op == "keep":
        a.keep(s["table"], s["context"], s["kept"], s["counts"])
        k, v = a.read(s["slots"])
        return {"k": k, "v": v}
    if op == "tree":
        return {"out": a.forward_tree(s["q"], s["tree"], s["table"], s["lens"], s["starts"], max_queries=s["max_n"],
                                      max_seq_len=s["max_len"])}
    if s["max_n"] == 1:  # a decode step: one query per sequence
        return {"out": a.forward(s["q"], s["table"], s["lens"], max_seq_len=s["max_len"])}
    return {"out": a.forward(s["q"], s["table"], s["lens"], s["starts"], max_queries=s["max_n"],
                             max_seq_len=s["max_len"])}


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


def _store(s, slots, k, v):
    """fp32 rows [T, kv_heads, D] into the cache."""
    p, r, u, i = _place(s, slots)
    if s["ks"] is not None:
        for x, scales, name in ((k, s["ks"], "k"), (v, s["vs"], "v")):
            scale = x.abs().amax(dim=-1, keepdim=True) / 127
            scale = torch.where(scale > 0, scale, 1.0)
            scales[p, :, r] = scale.squeeze(-1)
            codes = torch.round(x / scale).to(torch.int8)
            k, v = (codes, v) if name == "k" else (k, codes)
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
    case, op = s["case"], s["case"]["op"]
    if op == "write":
        cos, sin = s["rope"][s["positions"]].unsqueeze(1).chunk(2, dim=-1)
        q = _norm_rope(s["q"], s["q_norm"], cos, sin)
        _store(s, s["slots"], _norm_rope(s["new_k"], s["k_norm"], cos, sin), s["new_v"].float())
        return dict(_read_back(s), q=q.to(torch.bfloat16))
    if op == "read":
        return _read_back(s)
    page = case["page"]
    if op == "keep":
        seqs, most = s["kept"].shape
        moved = torch.arange(most, device="cuda") < s["counts"].unsqueeze(1)
        seq = torch.arange(seqs, device="cuda").unsqueeze(1).expand(-1, most)[moved]
        to = (s["context"].unsqueeze(1) + torch.arange(most, device="cuda"))[moved].long()
        at = (s["context"].unsqueeze(1) + s["kept"])[moved].long()
        slots = [s["table"][seq, x // page].long() * page + x % page for x in (at, to)]
        (p, r, u, i), (tp, tr, tu, ti) = _place(s, slots[0]), _place(s, slots[1])
        s["k"][tp, :, tr] = s["k"][p, :, r]
        s["v"][tp, :, tu, :, ti] = s["v"][p, :, u, :, i]
        if s["ks"] is not None:
            s["ks"][tp, :, tr] = s["ks"][p, :, r]
            s["vs"][tp, :, tr] = s["vs"][p, :, r]
        return _read_back(s)

    # attention: every sequence padded to the longest, scores in 32 bits
    seqs, n, length = case["seqs"], s["max_n"], s["max_len"]
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
    if op == "tree":
        drafted = position - context                                              # [seqs, 1, length]
        words = s["tree"][row]                                                    # [seqs, n, words]
        at = drafted.clamp(0, words.shape[2] * 64 - 1).expand(-1, n, -1)
        bit = (words.gather(2, at // 64) >> (at % 64)) & 1
        sees = (drafted < 0) | (bit == 1)
    else:
        sees = position <= context + nth.view(1, n, 1)
    sees = sees & inside.unsqueeze(1)
    q = s["q"][row].float().view(seqs, n, hk, group, d).permute(0, 2, 1, 3, 4).reshape(seqs, hk, n * group, d)
    score = torch.matmul(q, k).mul_(d ** -0.5).view(seqs, hk, n, group, length)
    score = score.masked_fill_(~sees.view(seqs, 1, n, 1, length), -math.inf)
    top = score.amax(dim=-1, keepdim=True)
    p = score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(dim=-1, keepdim=True).view(seqs, hk, n * group, 1)
    out = torch.matmul(p.view(seqs, hk, n * group, length), v) / torch.where(total > 0, total, 1.0)
    out = out.view(seqs, hk, n, group, d).permute(0, 2, 1, 3, 4).reshape(seqs, n, hq, d)
    return {"out": out[real].to(torch.bfloat16)}


# ------------------------------------------------------------------ the same in 64 bits
def _value(s, slot, which):
    """float64 rows of the cache at the slots, [T, kv_heads, D], from its layout."""
    page = s["case"]["page"]
    if which == "k":
        flat = s["k"].transpose(1, 2).reshape(-1, s["k"].shape[1], s["k"].shape[3])
        scales = s["ks"]
    else:
        flat = s["v"].permute(0, 2, 4, 1, 3).reshape(-1, s["v"].shape[1], s["v"].shape[3])
        scales = s["vs"]
    x = flat[slot].double()
    if scales is not None:
        x = x * scales.double().transpose(1, 2).reshape(-1, scales.shape[1])[slot].unsqueeze(-1)
    assert flat.shape[0] % page == 0
    return x


def _exact_rotated(x, weight, positions):
    x = x.double()
    if weight is not None:
        x = x / (x.pow(2).mean(dim=-1, keepdim=True) + EPS).sqrt() * weight.double()
    d = x.shape[-1]
    turn = _rope_table(positions, d, torch.float64)
    z = torch.complex(x[..., :d // 2], x[..., d // 2:]) * torch.complex(turn[:, :d // 2], turn[:, d // 2:]).unsqueeze(1)
    return torch.cat([z.real, z.imag], dim=-1)


def _exact_stored(x, fmt):
    if fmt == "bf16":
        return x
    step = x.abs().amax(dim=-1, keepdim=True) / 127
    return torch.where(step > 0, torch.round(x / step) * step, 0.0)


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    op, page = case["op"], case["page"]
    if op == "write":
        return {"q": _exact_rotated(s["q"], s["q_norm"], s["positions"]),
                "k": _exact_stored(_exact_rotated(s["new_k"], s["k_norm"], s["positions"]), case["cache"]),
                "v": _exact_stored(s["new_v"].double(), case["cache"])}
    if op == "read":
        return {"k": _value(s, s["slots"], "k"), "v": _value(s, s["slots"], "v")}
    starts = s["starts"].tolist()
    if op == "keep":
        out = {"k": _value(s, s["slots"], "k"), "v": _value(s, s["slots"], "v")}
        for x in out.values():
            old = x.clone()
            for b, count in enumerate(s["counts"].tolist()):
                x[starts[b]:starts[b] + count] = old[starts[b] + s["kept"][b, :count].long()]
        return out
    hk, d = case["kv_heads"], case["dim"]
    group = case["heads"] // hk
    out = torch.zeros(s["tokens"], case["heads"], d, dtype=torch.float64, device="cuda")
    for b, (n, length) in enumerate(_lengths(case)):
        where = torch.arange(length, device="cuda")
        slots = s["table"][b].long()[where // page] * page + where % page
        p_slots, inverse = torch.unique(slots // page, return_inverse=True)
        part = dict(s, k=s["k"][p_slots], v=s["v"][p_slots],
                    ks=None if s["ks"] is None else s["ks"][p_slots], vs=None if s["vs"] is None else s["vs"][p_slots])
        keys, values = (_value(part, inverse * page + slots % page, which) for which in ("k", "v"))
        mine = torch.arange(n, device="cuda").unsqueeze(1)
        hidden = where.unsqueeze(0) > length - n + mine
        if op == "tree":
            words = s["tree"][starts[b]:starts[b + 1]]
            node = (where - (length - n)).clamp(min=0)
            on = torch.stack([(words[:, j // 64] >> (j % 64)) & 1 for j in range(n)], dim=1).bool()
            hidden = (where >= length - n).unsqueeze(0) & ~on[:, node]
        for h in range(case["heads"]):
            q = s["q"][starts[b]:starts[b + 1], h].double()
            weight = (q @ keys[:, h // group].T / math.sqrt(d)).masked_fill(hidden, -math.inf).softmax(dim=-1)
            out[starts[b]:starts[b + 1], h] = weight @ values[:, h // group]
    return {"out": out}
