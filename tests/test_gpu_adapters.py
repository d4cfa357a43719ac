"""Low-rank adapters beside a projection on the GPU, against a plain 64-bit implementation.

Tolerance, with S[t, c] = |scale| sum_r (sum_i |x_i a_ri|) |b_cr|: the first product's fp32 sums are off by
(in + 8) 2^-24 of their terms' sizes, low enters the second product to 2^-16 of itself, that one's sums are off by
(2 rank + 8) 2^-24; all of these under (2^-15 + (in + 2 rank + 64) 2^-24) S.  The sum with base is rounded to fp32,
2^-24 |want|, and then once to bf16, U |want| and U of the error before it."""
import sys

import pytest
import torch

from attn_cases import DEV, U, generator, randn
from nano_ktrans_amd import NativeAdapters
from nano_ktrans_amd import _native as N

pytestmark = pytest.mark.gpu


def announce(msg):
    sys.__stderr__.write(f"[gpu-case] {msg}\n")
    sys.__stderr__.flush()


class Problem:
    """Adapters of mixed ranks; some parts and some adapters without any."""

    def __init__(self, n, width, outs, max_rank, seed, ranks=None):
        self.g = g = generator(seed)
        self.n, self.width, self.outs, self.max_rank = n, width, outs, max_rank
        self.adapters = NativeAdapters(num_adapters=n, in_features=width, out_features=outs, max_rank=max_rank)
        self.parts = {}
        for i in range(n):
            for p, out in enumerate(outs):
                if n > 2 and (i + p) % 5 == 4:
                    continue
                rank = ranks[i] if ranks else max(1, max_rank - (3 * i + p) % max_rank)
                a, b = randn(g, rank, width) * width ** -0.5, randn(g, out, rank) * 0.5
                scale = 0.25 + (i % 7) / 3.0
                self.adapters.load(i, a, b, scale, part=p)
                self.parts[i, p] = (a, b, torch.tensor(scale, dtype=torch.float32).item())

    def inputs(self, tokens):
        return randn(self.g, tokens, self.width), randn(self.g, tokens, sum(self.outs))

    def check(self, x, base, index, got):
        want, S = base.double(), torch.zeros(base.shape, dtype=torch.float64, device=DEV)
        for (i, p), (a, b, scale) in self.parts.items():
            rows = (index == i).nonzero().squeeze(1)
            at = sum(self.outs[:p])
            columns = slice(at, at + self.outs[p])
            want[rows, columns] += scale * (x[rows].double() @ a.double().T) @ b.double().T
            S[rows, columns] = abs(scale) * (x[rows].double().abs() @ a.double().abs().T) @ b.double().abs().T
        err = (2.0 ** -15 + (self.width + 2 * self.max_rank + 64) * 2.0 ** -24) * S + 2.0 ** -24 * want.abs()
        off = (got.double() - want).abs() - (U * want.abs() + (1 + U) * err)
        assert bool((off <= 0).all()), f"worst {float(off.max())} over its bound"
        none = (index < 0) | (index >= self.n)
        assert torch.equal(got[none], base[none])


SHAPES = [(4, 2048, (4096, 512, 512), 16), (24, 4096, (4096,), 32), (6, 896, (896, 128, 128), 64), (3, 64, (64,), 128),
          (40, 128, (128, 64, 192, 64), 5), (1, 192, (256,), 1), (5, 320, (64, 64), 100), (4, 640, (192, 64, 64, 64), 128)]


@pytest.mark.parametrize("n,width,outs,max_rank", SHAPES)
@pytest.mark.parametrize("tokens", [1, 2, 31, 33, 64, 200, 700, 1111])
def test_forward(gpu_device, n, width, outs, max_rank, tokens):
    """Tokens in any order of adapters; runs of one adapter; in place."""
    announce(f"adapters {n} of {max_rank}, {width} -> {outs}, T={tokens}")
    p = Problem(n, width, outs, max_rank, seed=tokens)
    x, base = p.inputs(tokens)
    mixed = torch.randint(-1, n, (tokens,), generator=p.g, device=DEV)
    if tokens == 1:
        mixed[0] = n - 1
    runs = (torch.arange(tokens, device=DEV) // 45) % (n + 1) - int(tokens > 45)
    for index in (mixed, runs):
        before = base.clone()
        got = p.adapters.forward(x, base, index)
        assert torch.equal(base, before)
        p.check(x, base, index, got)
        assert torch.equal(got, p.adapters.forward(x, base, index))
        place = base.clone()
        assert p.adapters.forward(x, place, index.to(torch.int32), out=place) is place
        assert torch.equal(place, got)
    p.adapters.check_status()


@pytest.mark.parametrize("n,width,outs,max_rank,tokens", [
    (4096, 64, (64,), 4, 5000), (3, 256, (128, 64, 64), 64, 9001), (2, 128, (64,), 64, 6000), (3, 192, (64,), 16, 20000),
    (2, 128, (64, 64, 64, 128), 128, 4500)])
def test_many_tokens(gpu_device, n, width, outs, max_rank, tokens):
    """More tokens than are grouped at once, more adapters than tiles, every number of blocks of A."""
    announce(f"adapters {n} of {max_rank}, {width} -> {outs}, T={tokens}")
    p = Problem(n, width, outs, max_rank, seed=tokens)
    x, base = p.inputs(tokens)
    index = torch.randint(-1, n + 1, (tokens,), generator=p.g, device=DEV)
    got = p.adapters.forward(x, base, index)
    p.check(x, base, index, got)
    with pytest.raises(N.NativeError):
        p.adapters.check_status()
    place = base.clone()
    p.adapters.forward(x, place, index, out=place)
    assert torch.equal(place, got)


@pytest.mark.parametrize("tokens", [1, 40, 600])
def test_strides_and_offsets(gpu_device, tokens):
    """Parts of wider arrays, with aligned rows (as they are) and others (copied)."""
    announce(f"adapters strided T={tokens}")
    p = Problem(5, 256, (128, 64), 16, seed=3)
    g = p.g
    index = torch.randint(-1, 5, (tokens,), generator=g, device=DEV)
    wide_x, wide_b = randn(g, tokens, 800), randn(g, tokens, 640)
    for at in (0, 16, 5):
        x, base = wide_x[:, at:at + 256], wide_b[:, at:at + 192]
        p.check(x, base, index, p.adapters.forward(x, base, index))
        p.check(x, base, index, p.adapters.forward(x, base.T.contiguous().T, index))
    first = wide_b.clone()
    view = wide_b[:, 64:256]
    got = p.adapters.forward(wide_x[:, :256], view, index, out=view)
    p.check(wide_x[:, :256], first[:, 64:256], index, got)
    wide_b[:, 64:256] = first[:, 64:256]
    assert torch.equal(wide_b, first)
    base = wide_b[:1, :192].expand(tokens, -1)  # one row for all tokens
    x = wide_x[:1, :256].expand(tokens, -1)
    p.check(x, base, index, p.adapters.forward(x, base, index))


@pytest.mark.parametrize("tokens", [3, 70, 600])
def test_other_requests_stay_out_of_it(gpu_device, tokens):
    """NaN and infinity in one request's tokens or adapter reach nothing of the others."""
    announce(f"adapters NaN T={tokens}")
    p = Problem(4, 128, (64,), 8, seed=4, ranks=[8, 3, 8, 8])
    x, base = p.inputs(tokens)
    index = torch.arange(tokens, device=DEV) % 4 - 1
    want = p.adapters.forward(x, base, index)
    sick = x.clone()
    sick[1, 3], sick[2, 5] = float("nan"), float("inf")
    p.adapters.load(2, torch.full((8, 128), float("nan"), device=DEV), torch.full((64, 8), float("inf"), device=DEV))
    got = p.adapters.forward(sick, base, index)
    well = index != 2
    well[1:3] = False
    assert torch.equal(got[well], want[well]) and int(well.sum()) > 0
    assert bool(torch.isnan(got[1]).all())
    p.adapters.clear(2)
    got = p.adapters.forward(x, base, index)
    assert torch.equal(got[index == 2], base[index == 2]) and torch.equal(got[index != 2], want[index != 2])


def test_infinities_keep_their_sign(gpu_device):
    """One rank, one infinite feature: the sum is an infinity of the product's sign, not NaN (the ranks that the
    adapter does not have take no part)."""
    adapters = NativeAdapters(num_adapters=1, in_features=64, out_features=64, max_rank=32)
    a, b = torch.ones(1, 64, device=DEV), torch.ones(64, 1, device=DEV)
    b[32:] = -1
    adapters.load(0, a, b)
    x = torch.zeros(2, 64, dtype=torch.bfloat16, device=DEV)
    x[0, 9] = float("inf")
    x[1, 9] = 3.0e38
    out = adapters.forward(x, torch.zeros(2, 64, dtype=torch.bfloat16, device=DEV), torch.zeros(2, dtype=torch.int64, device=DEV))
    assert bool((out[0, :32] == float("inf")).all() and (out[0, 32:] == float("-inf")).all())
    assert torch.equal(out[1, :32], x[1, 9].expand(32)) and torch.equal(out[1, 32:], -x[1, 9].expand(32))


def test_reload_and_other_types(gpu_device):
    """A smaller rank replaces a larger one whole; other types are rounded to bf16."""
    p = Problem(2, 128, (64, 128), 16, seed=6, ranks=[16, 16])
    x, base = p.inputs(50)
    index = torch.arange(50, device=DEV) % 2
    a, b = torch.randn(2, 128, generator=p.g, device=DEV), torch.randn(128, 2, generator=p.g, device=DEV)
    p.adapters.load(1, a.double().cpu(), b.half(), 0.5, part=1)
    p.parts[1, 1] = (a.to(torch.bfloat16), b.half().to(torch.bfloat16), 0.5)
    p.check(x, base, index, p.adapters.forward(x, base, index))


def test_bad_indexes(gpu_device):
    p = Problem(3, 64, (64,), 4, seed=7)
    x, base = p.inputs(40)
    index = torch.arange(40, device=DEV) % 3
    index[5], index[39] = 3, 2 ** 40
    index[6], index[7] = -1, -2 ** 40
    got = p.adapters.forward(x, base, index)
    p.check(x, base, index, got)
    with pytest.raises(N.NativeError, match="bad_adapter"):
        p.adapters.check_status()
    p.adapters.check_status()


def test_graph_and_streams(gpu_device):
    """Replays follow the captured tensors and what is loaded; two graphs and an eager call beside them."""
    p = Problem(4, 256, (128, 64), 16, seed=8)
    x, base = p.inputs(20)
    index = torch.arange(20, device=DEV) % 5 - 1
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                graphs.append((graph, p.adapters.forward(x, base, index)))
            graphs[-1] = (graph, graphs[-1][1])
    torch.cuda.current_stream().wait_stream(side)
    for step in range(3):
        x.copy_(randn(p.g, 20, 256))
        index.copy_(torch.randint(-1, 4, (20,), generator=p.g, device=DEV))
        a, b = randn(p.g, 16, 256), randn(p.g, 128, 16)
        p.adapters.load(1, a, b, 2.0)
        p.parts[1, 0] = (a, b, 2.0)
        for graph, _ in graphs:
            graph.replay()
        eager = p.adapters.forward(x, base, index)
        torch.cuda.synchronize()
        assert all(torch.equal(out, eager) for _, out in graphs)
        p.check(x, base, index, eager)


def test_empty_and_refused(gpu_device):
    p = Problem(2, 64, (64, 64), 4, seed=9)
    x, base = p.inputs(6)
    index = torch.zeros(6, dtype=torch.int64, device=DEV)
    assert p.adapters.forward(x[:0], base[:0], index[:0]).shape == (0, 128)
    wide = randn(p.g, 6, 320)
    for args, kw in (((x[:5], base, index), {}), ((x, base[:, :32], index), {}), ((x, base, index[:4]), {}),
                     ((x.float(), base, index), {}), ((x, base.float(), index), {}), ((x, base, index.float()), {}),
                     ((x.cpu(), base, index), {}), ((x, base, index.cpu()), {}), ((x[0], base, index), {}),
                     ((x, base, index), {"out": wide[:, 1:129]}), ((x, base, index), {"out": base.T.contiguous().T}),
                     ((x, wide[:, :128], index), {"out": wide[:, 8:136]}), ((wide[:, 128:192], base, index), {"out": wide[:, 128:256]}),
                     ((x, base, index), {"out": base[:1].expand(6, -1)})):
        with pytest.raises((ValueError, N.NativeError)):
            p.adapters.forward(*args, **kw)
    a, b = torch.zeros(4, 64, device=DEV), torch.zeros(64, 4, device=DEV)
    for args, kw in (((2, a, b), {}), ((-1, a, b), {}), ((0, a, b), {"part": 2}), ((0, a[:, :63], b), {}),
                     ((0, a, b[:63]), {}), ((0, a[:3], b), {}), ((0, torch.zeros(5, 64), torch.zeros(64, 5)), {}),
                     ((0, a[:0], b[:, :0]), {}), ((0, a.int(), b), {})):
        with pytest.raises(ValueError):
            p.adapters.load(*args, **kw)
    for kw in (dict(in_features=65), dict(out_features=96), dict(max_rank=129), dict(num_adapters=0)):
        with pytest.raises(N.NativeError):
            NativeAdapters(**dict(dict(num_adapters=2, in_features=64, out_features=64, max_rank=4), **kw))
