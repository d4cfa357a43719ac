"""Eviction: long recent windows, and calls beside each other.  Compared for equality, as in test_gpu_evict.py."""
import pytest
import torch

from attn_cases import DEV
from test_gpu_evict import announce, check, fill, make, state

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt,dim,page", [("bf16", 128, 64), ("int8", 128, 256), ("bf16", 64, 128), ("int8", 64, 64)])
@pytest.mark.parametrize("lengths,budget,recent", [
    ([3000, 2900], 2899, 1025), ([4096, 4000], 3990, 3000), ([4096], 2500, 2500), ([4000], 3999, 3999),
    ([4100, 9000], 4090, 3000), ([9000, 8100], 8000, 5000), ([9000], 4000, 2500), ([40000, 36000], 35990, 20000),
    ([4097], 4096, 1024)])
@pytest.mark.parametrize("in_place", [False, True])
def test_long_windows(gpu_device, lengths, budget, recent, fmt, dim, page, in_place):
    """Recent windows over what one turn of a workgroup takes, moved by less than their length: weights and cache are
    read and written over each other."""
    announce(f"evict {lengths} to {budget} recent {recent} {fmt} {dim} page {page} {in_place}")
    attn, table, weights, _ = make(lengths, 2, dim, fmt, page, seed=budget)
    check(attn, table, lengths, weights, budget, recent, **({"out": weights} if in_place else {}))


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
@pytest.mark.parametrize("length,budget,recent", [(3000, 1500, 200), (9000, 5000, 1500), (34000, 20000, 300)])
def test_two_streams_at_once(gpu_device, fmt, length, budget, recent):
    """Two sequences of one cache by a captured call, two others by an eager one on another stream, with nothing
    between them: the cache and the weights are those of the calls one after the other."""
    announce(f"evict on two streams {length} {fmt}")
    lengths = [length, length - 100, length // 2, length]
    attn, table, weights, g = make(lengths, 2, 128, fmt, 64, seed=41)
    twin = make(lengths, 2, 128, fmt, 64, seed=41)[0]
    lens = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[0]):
        first = attn.evict(table[:2], lens[:2], weights[:2], budget, recent)
    for _ in range(3):
        fill(attn, g)
        for x, y in zip(state(attn), (t for t in (twin.k_cache, twin.v_cache, twin.k_scales, twin.v_scales) if t is not None)):
            y.copy_(x)
        weights.copy_(torch.rand(weights.shape, generator=g, device=DEV))
        torch.cuda.synchronize()
        with torch.cuda.stream(streams[0]):
            graph.replay()
        with torch.cuda.stream(streams[1]):
            second = attn.evict(table[2:], lens[2:], weights[2:], budget, recent)
        torch.cuda.synchronize()
        for b, got in ((slice(0, 2), first), (slice(2, 4), second)):
            want = twin.evict(table[b], lens[b], weights[b], budget, recent)
            assert all(torch.equal(x, y) for x, y in zip(got, want))
        assert all(torch.equal(x, y) for x, y in zip(state(attn), state(twin)))
    attn.check_status()
