"""The attention half and the whole decoder layer as they are used: prompts, chunks, decode steps, drafted
trees and what is kept of them, over one cache per layer.

``FusedAttentionBlock`` is compared with a plain 64-bit attention between the same library projections.
Whole layers are compared with each other: the same tokens reach the same hidden states whichever calls
they come in (all at once, in chunks, one by one, as a draft).  Two such runs round the same values to bf16
in different places: at most about 12 roundings per layer and run (rotated rows, weights, attention,
projection, two residual sums, norms, the experts' activations and outputs), each with a relative rms of
2^-8 / sqrt(3), so 2 layers and 2 runs give at most sqrt(2 * 2 * 12) * 2^-8 / sqrt(3) = 1.6e-2 of the
vectors' rms; two int8 roundings per layer and run (steps of max|row| / 127, about 2.9 rms / 127, off by
a step / sqrt(12), 6.6e-3 of the rms) make it 2.4e-2: the bound is 2.5e-2.  Every expert is chosen, so
that no rounding decides a routing."""
import sys

import pytest
import torch
from torch import nn

from attn_cases import DEV, U, causal, dense, generator, make_attention, randn, reference, rotated
from nano_ktrans_amd import (AttentionBatch, FusedAttentionBlock, FusedDecoderLayer, HybridMoE, PackedSparseExpertMLP,
                             rope_table, tree_mask_from_parents)
from nano_ktrans_amd.layers.moe_block import FusedMoEBlock

pytestmark = pytest.mark.gpu

H, HQ, HK, D, PAGE = 256, 8, 2, 64, 64
EPS = 1e-6


def announce(msg):
    sys.__stderr__.write(f"[gpu-case] {msg}\n")
    sys.__stderr__.flush()


class RMSNorm(nn.Module):
    def __init__(self, weight):
        super().__init__()
        self.weight = nn.Parameter(weight, requires_grad=False)
        self.eps = EPS

    def forward(self, x):
        f = x.float()
        return (f * torch.rsqrt(f.pow(2).mean(-1, keepdim=True) + EPS)).to(x.dtype) * self.weight


def linear(g, n, k, bias=False):
    lin = nn.Linear(k, n, bias=bias).to(DEV, torch.bfloat16)
    with torch.no_grad():
        lin.weight.copy_(randn(g, n, k).float() * k ** -0.5)
        if bias:
            lin.bias.copy_(randn(g, n) * 0.1)
    return lin


def attention_block(g, fmt, qk_norm, num_pages, bias=False):
    attn = make_attention(HQ, HK, D, fmt, PAGE, num_pages)
    norms = (RMSNorm(1 + 0.1 * randn(g, D)), RMSNorm(1 + 0.1 * randn(g, D))) if qk_norm else (None, None)
    return FusedAttentionBlock(RMSNorm(1 + 0.1 * randn(g, H)), linear(g, (HQ + 2 * HK) * D, H, bias),
                               linear(g, H, HQ * D), attn, rope_table(4096, D, 1e4, DEV), *norms)


def decoder(seed, fmt, num_pages, layers=2):
    g = generator(seed)
    out = []
    for _ in range(layers):
        experts = {}
        for e in range(4):
            mlp = PackedSparseExpertMLP(H, 256).to(DEV, torch.bfloat16)
            with torch.no_grad():
                for p in mlp.parameters():
                    p.copy_(randn(g, *p.shape).float() * p.shape[1] ** -0.5)
            experts[str(e)] = mlp
        moe = HybridMoE(4, 4, H, 256, nn.ModuleDict(experts), torch.ones(4, dtype=torch.bool), 0, "",
                        router_use_softmax=True, experts_are_packed=True, gate=linear(g, 4, H), max_tokens=4096)
        out.append(FusedDecoderLayer(attention_block(g, fmt, True, num_pages),
                                     FusedMoEBlock(RMSNorm(1 + 0.1 * randn(g, H)), moe)))
    return out


def batch_of(layers, table, firsts, counts, mask=None, depths=None, decode=False):
    """The batch of counts[b] new tokens behind firsts[b] earlier ones; depths: positions of drafted tokens."""
    attn = layers[0].attention_block.attention
    seqs = torch.repeat_interleave(torch.arange(len(counts), device=DEV), torch.tensor(counts, device=DEV))
    places = torch.cat([torch.arange(f, f + n, device=DEV) for f, n in zip(firsts, counts)])
    positions = places
    if depths is not None:
        positions = torch.cat([f + torch.tensor(d, device=DEV) for f, d in zip(firsts, depths)])
    lens = torch.tensor([f + n for f, n in zip(firsts, counts)], dtype=torch.int32, device=DEV)
    starts = torch.cat([torch.zeros(1, dtype=torch.int64), torch.tensor(counts).cumsum(0)]).to(DEV, torch.int32)
    return AttentionBatch(positions, attn.slots(table, seqs, places), table, lens, None if decode else starts,
                          None if decode else max(counts), int(max(f + n for f, n in zip(firsts, counts))), mask)


@torch.no_grad()
def run(layers, x, batch):
    for layer in layers:
        x = layer(x, batch)
    return x


def near(a, b):
    a, b = a.double(), b.double()
    rel = float((a - b).norm() / b.norm())
    assert rel <= 2.5e-2, f"hidden states differ by {rel:.3e}"


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
@pytest.mark.parametrize("qk_norm,bias", [(True, False), (False, True)])
@pytest.mark.parametrize("counts,firsts", [([70, 9], [0, 0]), ([1, 1], [40, 127]), ([5, 30], [100, 64])])
def test_attention_block(gpu_device, fmt, qk_norm, bias, counts, firsts):
    announce(f"attention block {fmt} norm={qk_norm} bias={bias} rows {counts} after {firsts}")
    g = generator(sum(counts))
    block = attention_block(g, fmt, qk_norm, 12, bias)
    a = block.attention
    table = torch.randperm(12, generator=g, device=DEV)[:8].view(2, 4).to(torch.int32)
    layer = [FusedDecoderLayer(block, nn.Identity())]
    if max(firsts):
        run(layer, randn(g, sum(firsts), H), batch_of(layer, table, [0, 0], firsts))
    x = randn(g, sum(counts), H)
    batch = batch_of(layer, table, firsts, counts, decode=counts == [1, 1])
    got = run(layer, x, batch).double()
    with torch.no_grad():
        q, k, _ = block.qkv_proj(block.norm(x)).split([HQ * D, HK * D, HK * D], dim=1)
    rows = block.rope[batch.positions]
    q64, spread = rotated(q.unflatten(1, (HQ, D)), block.q_norm.weight if qk_norm else None, EPS, rows)
    # a rotated query is one bf16 rounding off this (and fp32 noise): where that is the other neighbour,
    # scores move by u |q_d k_d|; count the whole row's, u sum |q_d k_d| <= u |q| |k|
    q_bf = q64.to(torch.bfloat16).double()
    at = 0
    for b, (n, first) in enumerate(zip(counts, firsts)):
        where = torch.arange(first + n, device=DEV)
        keys, values = dense(a, a.slots(table, torch.full_like(where, b), where))
        want, A = reference(q_bf[at:at + n], keys, values, causal(n, first + n), a.scale)
        slack = 2 * U * a.scale * q_bf[at:at + n].norm(dim=-1).amax() * keys.norm(dim=-1).amax()
        off = (U * want.abs() + (U + U * U + 2.0 ** -9.9 + slack) * A).flatten(1)   # of the attention's rows
        w = block.o_proj.weight.double()
        out = want.flatten(1) @ w.T
        bound = off @ w.abs().T + 2.0 ** -24 * HQ * D * (want.flatten(1).abs() @ w.abs().T)
        bound = bound + U * (out.abs() + bound)                       # the projection's rounding
        sum_ = x[at:at + n].double() + out
        bound = bound + U * (sum_.abs() + bound)                      # the residual sum's
        assert bool(((got[at:at + n] - sum_).abs() <= bound).all()), f"sequence {b}"
        at += n
    assert not any(a.status().values())


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
def test_prompt_in_chunks_and_single_tokens(gpu_device, fmt):
    """The last tokens of two prompts: in one call, in uneven chunks, and then one by one."""
    announce(f"decoder: chunks and decode steps {fmt}")
    counts = [150, 97]
    table = torch.arange(8, dtype=torch.int32, device=DEV).view(2, 4).flip(0).contiguous()
    x = randn(generator(31), sum(counts), H)
    whole = decoder(30, fmt, 8)
    want = run(whole, x, batch_of(whole, table, [0, 0], counts))
    rows = [want[:150], want[150:]]
    tokens = [x[:150], x[150:]]
    parts = decoder(30, fmt, 8)
    at = [0, 0]
    for step in ([100, 3], [20, 64], [17, 17]):
        got = run(parts, torch.cat([t[f:f + n] for t, f, n in zip(tokens, at, step)]), batch_of(parts, table, at, step))
        near(got, torch.cat([r[f:f + n] for r, f, n in zip(rows, at, step)]))
        at = [f + n for f, n in zip(at, step)]
    for _ in range(13):
        got = run(parts, torch.cat([t[f:f + 1] for t, f in zip(tokens, at)]), batch_of(parts, table, at, [1, 1], decode=True))
        near(got, torch.cat([r[f:f + 1] for r, f in zip(rows, at)]))
        at = [f + 1 for f in at]
    for a, b in zip(whole, parts):
        a, b = a.attention_block.attention, b.attention_block.attention
        slots = a.slots(table, torch.zeros(150, dtype=torch.int64, device=DEV), torch.arange(150, device=DEV))
        for u, v in zip(a.read(slots), b.read(slots)):
            near(u, v)


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
def test_draft_verify_keep_and_go_on(gpu_device, fmt):
    """Two requests: a prompt, a drafted tree verified in one call, the accepted path kept, one more token.
    The same tokens without the draft, one by one, reach the same hidden states."""
    announce(f"decoder: draft, keep, decode {fmt}")
    counts = [60, 131]
    table = torch.randperm(9, generator=generator(40), device=DEV)[:8].view(2, 4).to(torch.int32)
    g = generator(41)
    prompt = randn(g, sum(counts), H)
    drafted = decoder(42, fmt, 9)
    plain = decoder(42, fmt, 9)
    near(run(drafted, prompt, batch_of(drafted, table, [0, 0], counts)),
         run(plain, prompt, batch_of(plain, table, [0, 0], counts)))
    parents = [[-1, 0, 0, 1, 2, 2, 5, 4], [-1, -1, 1, 2, 0]]
    paths = [[0, 2, 5, 6], [1, 2, 3]]                     # the accepted nodes
    depth = []
    for p in parents:
        d = []
        for q in p:
            d.append(d[q] + 1 if q >= 0 else 0)
        depth.append(d)
    nodes = [len(p) for p in parents]
    x = randn(g, sum(nodes), H)
    mask = tree_mask_from_parents(parents, DEV)
    tree = run(drafted, x, batch_of(drafted, table, counts, nodes, mask, depth))
    kept = torch.full((2, 4), 99, dtype=torch.int32)
    for b, path in enumerate(paths):
        kept[b, :len(path)] = torch.tensor(path, dtype=torch.int32)
    for layer in drafted:
        layer.attention_block.attention.keep(table, torch.tensor(counts, dtype=torch.int32, device=DEV), kept.to(DEV),
                                             torch.tensor([len(p) for p in paths], dtype=torch.int32, device=DEV))
    # the same path, token by token (the shorter one ends with a padding row of its own)
    start = [0, nodes[0]]
    at = list(counts)
    for i in range(4):
        live = [b for b in range(2) if i < len(paths[b])]
        rows = torch.cat([x[start[b] + paths[b][i]].unsqueeze(0) for b in live])
        batch = batch_of(plain, table[live], [at[b] for b in live], [1] * len(live), decode=True)
        got = run(plain, rows, batch)
        near(got, torch.cat([tree[start[b] + paths[b][i]].unsqueeze(0) for b in live]))
        for b in live:
            at[b] += 1
    assert at == [64, 134]
    for a, b in zip(drafted, plain):
        a, b = a.attention_block.attention, b.attention_block.attention
        for seq, length in enumerate(at):
            where = torch.arange(length, device=DEV)
            slots = a.slots(table, torch.full_like(where, seq), where)
            for u, v in zip(a.read(slots), b.read(slots)):
                near(u, v)
        a.check_status()
    last = randn(g, 2, H)
    near(run(drafted, last, batch_of(drafted, table, at, [1, 1], decode=True)),
         run(plain, last, batch_of(plain, table, at, [1, 1], decode=True)))


def test_padded_batch(gpu_device):
    """Padding tokens behind the last sequence: the others' rows are the same, theirs are numbers, and the cache
    holds the same.  The output carries no gradient."""
    announce("attention block: padded batch")
    g = generator(60)
    block = attention_block(g, "bf16", True, 4)
    a = block.attention
    layer = [FusedDecoderLayer(block, nn.Identity())]
    table = torch.arange(4, dtype=torch.int32, device=DEV).view(2, 2)
    x = randn(g, 40, H)
    batch = batch_of(layer, table, [0, 0], [30, 5])
    slots = a.slots(table, torch.zeros(30, dtype=torch.int64, device=DEV), torch.arange(30, device=DEV))
    want, cached = run(layer, x[:35], batch), a.read(slots)
    batch.positions = torch.nn.functional.pad(batch.positions, (0, 5))
    batch.slots = torch.nn.functional.pad(batch.slots, (0, 5), value=-1)
    torch.empty(40, HQ, D, dtype=torch.bfloat16, device=DEV).fill_(float("nan"))  # (memory that comes next)
    got = block(x.requires_grad_(), batch)
    assert not got.requires_grad and bool(torch.isfinite(got).all())
    # (the library projections may sum in another order at another batch size)
    near(got[:35], want)
    for u, v in zip(a.read(slots), cached):
        near(u, v)


def test_decode_loop_in_a_graph(gpu_device):
    """Two layers' decode step captured once; lengths, slots and positions move on the device between replays,
    beside eager work of another batch on the same layers."""
    announce("decoder: decode steps in a graph")
    layers = decoder(50, "int8", 16)
    eager = decoder(50, "int8", 16)
    table = torch.arange(8, dtype=torch.int32, device=DEV).view(2, 4)
    g = generator(51)
    prompt = randn(g, 100, H)
    for ls in (layers, eager):
        run(ls, prompt, batch_of(ls, table, [0, 0], [30, 70]))
    attn = layers[0].attention_block.attention
    x = randn(g, 2, H)
    lens = torch.tensor([31, 71], dtype=torch.int32, device=DEV)
    positions = torch.tensor([30, 70], device=DEV)
    slots = attn.slots(table, torch.arange(2, device=DEV), positions)
    batch = AttentionBatch(positions, slots, table, lens)
    run(layers, x, batch)  # warm-up: the same tokens are written again by the first replay
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(layers, x, batch)
    other = torch.arange(8, 16, dtype=torch.int32, device=DEV).view(2, 4)
    for step in range(40):  # the first sequence passes a page's end
        x.copy_(randn(g, 2, H))
        if step:
            lens += 1
            positions += 1
            slots.copy_(attn.slots(table, torch.arange(2, device=DEV), positions))
        graph.replay()
        want = run(eager, x, AttentionBatch(positions.clone(), slots.clone(), table, lens.clone()))
        run(layers, prompt, batch_of(layers, other, [0, 0], [30, 70]))
        torch.cuda.synchronize()
        assert torch.equal(out, want), step


def test_refusals(gpu_device):
    g = generator(1)
    block = attention_block(g, "bf16", True, 2)
    parts = (block.norm, block.qkv_proj, block.o_proj, block.attention, block.rope)
    with pytest.raises(ValueError, match="go together"):
        FusedAttentionBlock(*parts, q_norm=block.q_norm)
    other = RMSNorm(block.k_norm.weight)
    other.eps = 1e-5
    with pytest.raises(ValueError, match="eps"):
        FusedAttentionBlock(*parts, q_norm=block.q_norm, k_norm=other)
    with pytest.raises(ValueError, match="columns"):
        FusedAttentionBlock(block.norm, linear(g, 64, H), *parts[2:])
    with pytest.raises(ValueError, match="bf16"):
        block(torch.zeros(1, H, device=DEV), None)
