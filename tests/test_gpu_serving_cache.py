"""Whole decoder layers with adapters of their requests, positions on several axes, and caches that keep only the
tokens that attention weighs most: as a serving program uses them together."""
import sys

import pytest
import torch
from torch import nn

from attn_cases import DEV, dense, generator, randn
from nano_ktrans_amd import AttentionBatch, FusedAttentionBlock, NativeAdapters, media_positions, rope_axes
from nano_ktrans_amd import _native as N
from test_gpu_decoder_layer import D, H, HK, HQ, PAGE, attention_block, decoder, linear, near

pytestmark = pytest.mark.gpu

OUTS = (HQ * D, HK * D, HK * D)
AXES = rope_axes([12, 10, 10], interleaved=True)
WIDTH = 6 * PAGE


def announce(msg):
    sys.__stderr__.write(f"[gpu-case] {msg}\n")
    sys.__stderr__.flush()


def adapted(g, block):
    """The block with three adapters beside each projection, and its frequencies dealt out to three axes."""
    qkv = NativeAdapters(num_adapters=3, in_features=H, out_features=OUTS, max_rank=8)
    o = NativeAdapters(num_adapters=3, in_features=HQ * D, out_features=H, max_rank=24)
    for i in range(3):
        for p, out in enumerate(OUTS):
            qkv.load(i, randn(g, 8 - i, H) * H ** -0.5, randn(g, out, 8 - i) * 0.3, scale=0.5 + i, part=p)
        o.load(i, randn(g, 24, HQ * D) * (HQ * D) ** -0.5, randn(g, H, 24) * 0.2)
    block.qkv_adapters, block.o_adapters, block.rope_axes = qkv, o, tuple(AXES)
    return block


def layers_of(seed, fmt):
    g = generator(seed + 1)
    out = decoder(seed, fmt, 20)
    for layer in out:
        adapted(g, layer.attention_block)
    return out


def batch_of(layers, table, firsts, positions, adapters, last=None):
    """New tokens behind firsts[b] cached ones, at positions[b] [3, n]."""
    attn = layers[0].attention_block.attention
    counts = [p.shape[1] for p in positions]
    n = torch.tensor(counts, device=DEV)
    seqs = torch.repeat_interleave(torch.arange(len(counts), device=DEV), n)
    places = torch.cat([torch.arange(f, f + c, device=DEV) for f, c in zip(firsts, counts)])
    lens = torch.tensor(firsts, device=DEV, dtype=torch.int32) + n.to(torch.int32)
    starts = torch.nn.functional.pad(n.cumsum(0), (1, 0)).to(torch.int32)
    return AttentionBatch(torch.cat(positions, dim=1).to(DEV), attn.slots(table, seqs, places), table, lens, starts,
                          max(counts), None, adapters=torch.tensor(adapters, device=DEV)[seqs], last=last)


def prompts():
    """A prompt with an image and a video, a short text, one with an image: positions and the next ones."""
    made = [media_positions([20, (1, 8, 10), 30, (4, 4, 5), 11]), media_positions([37]),
            media_positions([3, (1, 12, 12), 40])]
    return [p for p, _ in made], [n for _, n in made]


@torch.no_grad()
def run(layers, x, batch, weights):
    for layer, w in zip(layers, weights):
        x = layer(x, batch, w)
    return x


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
def test_block_is_its_operators(gpu_device, fmt):
    """The block's result is that of the public calls one after the other, bit for bit."""
    announce(f"block of operators {fmt}")
    g = generator(3)
    block = adapted(g, attention_block(g, fmt, True, 20))
    a = block.attention
    table = torch.randperm(20, generator=g, device=DEV)[:18].view(3, 6).to(torch.int32)
    positions, _ = prompts()
    holder = [type("Layer", (), {"attention_block": block})]
    batch = batch_of(holder, table, [0, 0, 0], positions, [1, -1, 2], last=16)
    x = randn(g, batch.positions.shape[1], H)
    w, w2 = torch.zeros(3, HK, WIDTH, device=DEV), torch.zeros(3, HK, WIDTH, device=DEV)
    got = block(x, batch, w)
    held = [t.clone() for t in (a.k_cache, a.v_cache)]
    with torch.no_grad():
        normed = block.norm(x)
        qkv = block.qkv_adapters.forward(normed, block.qkv_proj(normed), batch.adapters)
        q = a.write(*qkv.split(OUTS, dim=1), batch.positions, batch.slots, block.rope, block.q_norm.weight,
                    block.k_norm.weight, block.q_norm.eps, axes=AXES)
        out = a.forward_weights(q, w2, table, batch.seq_lens, batch.query_starts, max_queries=batch.max_queries,
                                last=16).flatten(1)
        want = x + block.o_adapters.forward(out, block.o_proj(out), batch.adapters)
    assert torch.equal(got, want) and torch.equal(w, w2) and bool(w.any())
    assert all(torch.equal(s, t) for s, t in zip(held, (a.k_cache, a.v_cache)))
    # the options do what they say: without any one of them the result is another
    for change in ({"adapters": None}, {"adapters": batch.adapters.roll(1)},
                   {"positions": batch.positions.roll(1, dims=0)}):
        other = block(x, AttentionBatch(**dict(vars(batch), **change)))
        assert not torch.equal(other, got)
    none = AttentionBatch(**dict(vars(batch), adapters=torch.full_like(batch.adapters, -1)))
    assert torch.equal(block(x, none), block(x, AttentionBatch(**dict(vars(batch), adapters=None))))
    a.check_status()


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
def test_prompts_eviction_and_decode(gpu_device, fmt):
    """Prompts, eviction to 96 tokens, decode steps past it, eviction again: each sequence alone gives what the
    batch gives, in eager calls and in a replayed graph of a whole step."""
    announce(f"serving with eviction {fmt}")
    budget, recent = 96, 16
    positions, nexts = prompts()
    adapters = [1, -1, 2]
    g = generator(5)
    x = [randn(g, p.shape[1], H) for p in positions]
    steps = [randn(g, 3, H) for _ in range(5)]

    def serve(rows, graph):
        layers = layers_of(7, fmt)
        B = len(rows)
        table = torch.arange(18, device=DEV, dtype=torch.int32).view(3, 6)[rows]
        weights = [torch.zeros(B, HK, WIDTH, device=DEV) for _ in layers]
        batch = batch_of(layers, table, [0] * B, [positions[b] for b in rows], [adapters[b] for b in rows], last=32)
        outs = [run(layers, torch.cat([x[b] for b in rows]), batch, weights)]
        lens = batch.seq_lens
        at = torch.tensor([nexts[b] for b in rows], device=DEV)
        index = torch.tensor([adapters[b] for b in rows], device=DEV)
        state = {"x": torch.zeros(B, H, dtype=torch.bfloat16, device=DEV), "lens": lens.clone(), "at": at}

        def evict():
            for layer, w in zip(layers, weights):
                new, _ = layer.attention_block.attention.evict(table, state["lens"], w, budget, recent, out=w)
            state["lens"].copy_(new)

        def step():
            attn = layers[0].attention_block.attention
            slots = attn.slots(table, torch.arange(B, device=DEV), state["lens"].long())
            state["lens"] += 1
            b = AttentionBatch(state["at"].expand(3, -1), slots, table, state["lens"], max_seq_len=WIDTH,
                               adapters=index)
            state["out"] = run(layers, state["x"], b, weights)
            state["at"] += 1
            evict()

        evict()
        lengths = state["lens"].tolist()
        if graph:
            kept = {name: t.clone() for name, t in state.items()}
            caches = [t for layer in layers for t in (layer.attention_block.attention.k_cache,
                                                      layer.attention_block.attention.v_cache,
                                                      layer.attention_block.attention.k_scales,
                                                      layer.attention_block.attention.v_scales) if t is not None]
            held = [t.clone() for t in caches + weights]
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                step()
                captured = torch.cuda.CUDAGraph()
                with torch.cuda.graph(captured, stream=side):
                    step()
            torch.cuda.current_stream().wait_stream(side)
            for t, old in zip(caches + weights, held):
                t.copy_(old)
            for name, old in kept.items():
                state[name].copy_(old)
        for s in steps:
            state["x"].copy_(s[rows])
            captured.replay() if graph else step()
            outs.append(state["out"].clone())
        torch.cuda.synchronize()
        for layer in layers:
            layer.attention_block.attention.check_status()
            layer.attention_block.qkv_adapters.check_status()
        keys = [dense(layer.attention_block.attention, layer.attention_block.attention.slots(
            table, torch.zeros(96, dtype=torch.int64, device=DEV), torch.arange(96, device=DEV)))[0] for layer in layers]
        return outs, lengths, state["lens"].tolist(), weights, keys

    outs, lengths, after, weights, keys = serve([0, 1, 2], graph=False)
    assert lengths == [96, 37, 96] and after == [96, 42, 96]
    for w in weights:  # zeros behind what is kept, none where a token is
        assert not bool(w[0, :, 96:].any()) and not bool(w[1, :, 42:].any()) and bool((w[:, :, :37] > 0).any())
    again = serve([0, 1, 2], graph=True)
    assert all(torch.equal(s, t) for s, t in zip(outs, again[0]))
    assert all(torch.equal(s, t) for s, t in zip(weights, again[3])) and after == again[2]
    assert all(torch.equal(s, t) for s, t in zip(keys, again[4]))
    at = 0
    for b in range(3):
        alone = serve([b], graph=False)
        n = positions[b].shape[1]
        near(outs[0][at:at + n], alone[0][0])
        at += n
        if b == 1:  # (nothing is evicted: the same tokens, other sums)
            for s, t in zip(outs[1:], alone[0][1:]):
                near(s[b:b + 1], t)


def test_block_refuses(gpu_device):
    g = generator(9)
    block = attention_block(g, "bf16", False, 4)
    args = (block.norm, block.qkv_proj, block.o_proj, block.attention, block.rope)
    small = NativeAdapters(num_adapters=1, in_features=H, out_features=OUTS[:2], max_rank=4)
    for kw in ({"qkv_adapters": small}, {"o_adapters": small}):
        with pytest.raises(ValueError):
            FusedAttentionBlock(*args, **kw)
    table = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    at = torch.zeros(1, dtype=torch.int64, device=DEV)
    batch = AttentionBatch(at, at, table, torch.ones(1, dtype=torch.int32, device=DEV),
                           tree_mask=torch.ones(1, 1, dtype=torch.int64, device=DEV))
    with pytest.raises(ValueError, match="drafted"):
        block(randn(g, 1, H), batch, torch.zeros(1, HK, PAGE, device=DEV))
    block.rope_axes = tuple(AXES)
    with pytest.raises(ValueError, match="positions"):
        block(randn(g, 1, H), AttentionBatch(at, at, table, batch.seq_lens))
