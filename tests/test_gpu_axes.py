"""Positions with several axes on the GPU: head norms, rotation and the cache write, against the plain 64-bit
implementation in attn_cases.py (which has the tolerances)."""
import sys

import pytest
import torch

from attn_cases import DEV, U, dense, generator, make_attention, poison, randn, rotated
from nano_ktrans_amd import _native as N
from nano_ktrans_amd import media_positions, rope_axes, rope_table

pytestmark = pytest.mark.gpu


def announce(msg):
    sys.__stderr__.write(f"[gpu-case] {msg}\n")
    sys.__stderr__.flush()


def rope_rows(rope, positions, axes):
    """[T, D]: each frequency's cosine and sine from its own axis's row."""
    at = positions[torch.tensor(axes, device=positions.device)].T
    half = rope.shape[1] // 2
    return torch.cat([rope[:, :half].gather(0, at), rope[:, half:].gather(0, at)], dim=1)


def sections_of(dim, kind):
    half = dim // 2
    return {"one": [half], "three": [half - 2 * (3 * half // 8), 3 * half // 8, 3 * half // 8], "odd": [5, half - 8, 3],
            "four": [half - 21, 7, 7, 7], "empty": [0, half - 1, 1]}[kind]


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(32, 4, 128, 64), (14, 2, 64, 128), (3, 1, 128, 256)])
@pytest.mark.parametrize("tokens,kind,interleaved,norm", [(1, "three", False, True), (7, "odd", True, False),
                                                          (64, "four", False, False), (333, "three", True, True),
                                                          (1500, "empty", False, True), (1100, "one", False, False)])
def test_write_axes(gpu_device, heads, kv_heads, dim, page, fmt, tokens, kind, interleaved, norm):
    announce(f"write axes {heads}/{kv_heads}/{dim} {fmt} T={tokens} {kind} {interleaved}")
    g = generator(tokens + heads)
    attn = make_attention(heads, kv_heads, dim, fmt, page, 1600 // page + 2)
    poison(attn)
    axes = rope_axes(sections_of(dim, kind), interleaved)
    num_axes = len(sections_of(dim, kind))
    qkv = randn(g, tokens, (heads + 2 * kv_heads) * dim)
    q, k, v = (x.unflatten(1, (-1, dim)) for x in qkv.split([heads * dim, kv_heads * dim, kv_heads * dim], dim=1))
    slots = 3 + torch.arange(tokens, device=DEV)
    rope = rope_table(9000, dim, 1e6, DEV)
    positions = torch.randint(0, 9000, (num_axes, tokens), generator=g, device=DEV)
    positions[:, 0] = 8999
    if tokens > 6:  # padding, on any axis anywhere
        slots[3] = -1
        positions[num_axes - 1, 3] = -40
    weights = {"q_norm": 1 + 0.1 * randn(g, dim), "k_norm": 1 + 0.1 * randn(g, dim)} if norm else {}
    out = attn.write(q, k, v, positions, slots, rope, axes=axes, **weights)
    stored = slots >= 0
    table = rope_rows(rope, positions.clamp(0, 8999), axes)
    want, spread = rotated(q, weights.get("q_norm"), 1e-6, table)
    bound = U * want.abs() + 2.0 ** -20 * spread * (1 + U) + 2.0 ** -130
    assert bool(((out.double() - want).abs() <= bound)[stored].all())
    if tokens > 6:
        assert not bool(out[3].any())
    want, spread = rotated(k, weights.get("k_norm"), 1e-6, table)
    got_k, got_v = dense(attn, slots[stored])
    for got, want, err in ((got_k, want[stored], 2.0 ** -20 * spread[stored]), (got_v, v[stored].double(), 0.0)):
        if fmt == "bf16":
            bound = U * want.abs() + err * (1 + U)
        else:
            bound = want.abs().amax(dim=-1, keepdim=True) / 127 * (0.5 + 2.0 ** -15) + err
        assert bool(((got - want).abs() <= bound + 2.0 ** -130).all())
    attn.check_status()


def test_equal_axes_are_one_axis(gpu_device):
    """Text: the same position on all axes gives write's own bits, in both caches."""
    announce("write axes as one")
    g = generator(5)
    for fmt in ("bf16", "int8"):
        a, b = (make_attention(8, 2, 128, fmt, 64, 40) for _ in range(2))
        q, k, v = randn(g, 1500, 8, 128), randn(g, 1500, 2, 128), randn(g, 1500, 2, 128)
        rope = rope_table(3000, 128, 1e6, DEV)
        at = torch.randint(0, 3000, (1500,), generator=g, device=DEV)
        slots = torch.randperm(2000, generator=g, device=DEV)[:1500]
        w = {"q_norm": 1 + 0.1 * randn(g, 128), "k_norm": 1 + 0.1 * randn(g, 128)}
        x = a.write(q, k, v, at, slots, rope, **w)
        y = b.write(q, k, v, at.expand(3, -1), slots, rope, axes=rope_axes([16, 24, 24]), **w)
        assert torch.equal(x, y) and torch.equal(a.k_cache, b.k_cache) and torch.equal(a.v_cache, b.v_cache)
        if fmt == "int8":
            assert torch.equal(a.k_scales, b.k_scales) and torch.equal(a.v_scales, b.v_scales)


@pytest.mark.parametrize("axis", [0, 1, 2])
@pytest.mark.parametrize("bad", [-1, 50, 2 ** 40])
def test_position_out_of_range(gpu_device, axis, bad):
    """On one axis only: reported, its queries zero, nothing of it stored."""
    g = generator(6)
    attn = make_attention(8, 2, 64, "bf16", 64, 2)
    positions = torch.randint(0, 50, (3, 9), generator=g, device=DEV)
    positions[axis, 4] = bad
    out = attn.write(randn(g, 9, 8, 64), randn(g, 9, 2, 64), randn(g, 9, 2, 64), positions,
                     torch.arange(9, device=DEV), rope_table(50, 64, device=DEV), axes=rope_axes([8, 12, 12]))
    assert not bool(out[4].any()) and bool(out[3].any() and out[5].any())
    k, v = dense(attn, torch.arange(9, device=DEV))
    assert not bool(k[4].any() or v[4].any()) and bool(k[5].any())
    with pytest.raises(N.NativeError, match="bad_position"):
        attn.check_status()


def test_graph(gpu_device):
    """Replays follow the positions in the captured tensor."""
    g = generator(7)
    attn, twin = (make_attention(8, 2, 128, "int8", 64, 4) for _ in range(2))
    axes, rope = rope_axes([24, 20, 20], interleaved=True), rope_table(500, 128, device=DEV)
    q, k, v = randn(g, 5, 8, 128), randn(g, 5, 2, 128), randn(g, 5, 2, 128)
    positions, slots = torch.zeros(3, 5, dtype=torch.int64, device=DEV), torch.arange(5, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = attn.write(q, k, v, positions, slots, rope, axes=axes)
    torch.cuda.current_stream().wait_stream(side)
    for step in range(3):
        positions.copy_(torch.randint(0, 500, (3, 5), generator=g, device=DEV))
        graph.replay()
        want = twin.write(q, k, v, positions, slots, rope, axes=axes)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(attn.k_cache, twin.k_cache)


def test_refused(gpu_device):
    attn = make_attention(8, 2, 64, "bf16", 64, 2)
    g = generator(8)
    q, k, v = randn(g, 3, 8, 64), randn(g, 3, 2, 64), randn(g, 3, 2, 64)
    rope, slots = rope_table(50, 64, device=DEV), torch.arange(3, device=DEV)
    positions, _ = media_positions([3], device=DEV)
    axes = rope_axes([8, 12, 12])
    for at, ax in ((positions, axes[:-1]), (positions, axes[:-1] + [3]), (positions, axes[:-1] + [-1]),
                   (positions[:2], axes), (positions[:, :2], axes), (positions[0], axes),
                   (positions[0].expand(5, -1), axes), (positions.float(), axes), (positions, axes[:-1] + [200])):
        with pytest.raises((ValueError, N.NativeError)):
            attn.write(q, k, v, at, slots, rope, axes=ax)
    with pytest.raises(ValueError):
        attn.write(q, k, v, positions, slots, rope)
