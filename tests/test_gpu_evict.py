"""Eviction from the paged cache, against a plain implementation: every value moves unchanged, so all is compared
for equality."""
import sys

import pytest
import torch

from attn_cases import DEV, dense, generator, make_attention
from nano_ktrans_amd import _native as N

pytestmark = pytest.mark.gpu


def announce(msg):
    sys.__stderr__.write(f"[gpu-case] {msg}\n")
    sys.__stderr__.flush()


def sources(weights, budget, recent):
    """Where each place of one sequence's one head gets its token from: plain lists."""
    n = len(weights)
    keep = min(budget, n)
    if keep == n:
        return list(range(n))
    window = min(recent, keep)
    front, rest = keep - window, n - window
    heavy = sorted(range(rest), key=lambda i: (weights[i] != weights[i], -weights[i] if weights[i] == weights[i] else 0, i))
    stays = set(heavy[:front])
    coming = [i for i in sorted(stays) if i >= front]
    out = []
    for i in range(front):
        out.append(i if i in stays else coming.pop(0))
    return out + list(range(rest, n))


def fill(attn, g):
    """Every value of the cache different as far as its type allows."""
    if attn.cache_format == "bf16":
        for x in (attn.k_cache, attn.v_cache):
            x.copy_(torch.randn(x.shape, generator=g, device=DEV))
    else:
        for x in (attn.k_cache, attn.v_cache):
            x.copy_(torch.randint(-127, 128, x.shape, generator=g, device=DEV))
        for x in (attn.k_scales, attn.v_scales):
            x.copy_(torch.rand(x.shape, generator=g, device=DEV) + 0.5)


def rows(attn, table, b, length):
    at = torch.arange(length, device=DEV)
    return dense(attn, attn.slots(table, torch.full_like(at, b), at))


def state(attn):
    return [x.clone() for x in (attn.k_cache, attn.v_cache, attn.k_scales, attn.v_scales) if x is not None]


def check(attn, table, lengths, weights, budgets, recent, **kw):
    B, W = table.shape
    old = [rows(attn, table, b, n) for b, n in enumerate(lengths)]
    before = state(attn)
    w0 = weights.clone()
    lens = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    new_lens, out = attn.evict(table, lens, weights, budgets, recent, **kw)
    per = budgets.tolist() if isinstance(budgets, torch.Tensor) else [budgets] * B
    assert new_lens.tolist() == [min(x, n) for x, n in zip(per, lengths)]
    if out.data_ptr() != weights.data_ptr():
        assert torch.equal(weights.nan_to_num(nan=-7.0), w0.nan_to_num(nan=-7.0))
    for b, n in enumerate(lengths):
        keep = min(per[b], n)
        for h in range(attn.num_kv_heads):
            src = torch.tensor(sources(w0[b, h, :n].tolist(), per[b], recent), dtype=torch.int64, device=DEV)
            assert len(src) == keep
            k, v = rows(attn, table, b, keep)
            assert torch.equal(k[:, h], old[b][0][src, h]), f"keys of sequence {b} head {h}"
            assert torch.equal(v[:, h], old[b][1][src, h]), f"values of sequence {b} head {h}"
            assert torch.equal(out[b, h, :keep].nan_to_num(nan=-7.0), w0[b, h, src].nan_to_num(nan=-7.0))
        assert not bool(out[b, :, keep:].any())
    # nothing but the kept tokens' places has changed
    now = state(attn)
    unit = attn.v_cache.shape[4]
    for b, n in enumerate(lengths):
        at = torch.arange(min(per[b], n), device=DEV)
        slots = attn.slots(table, torch.full_like(at, b), at)
        page, r = slots // attn.page_size, slots % attn.page_size
        now[0][page, :, r] = before[0][page, :, r]
        now[1][page, :, r // unit, :, r % unit] = before[1][page, :, r // unit, :, r % unit]
        for i in range(2, len(now)):
            now[i][page, :, r] = before[i][page, :, r]
    assert all(torch.equal(a, b) for a, b in zip(now, before))
    attn.check_status()
    return new_lens, out


def make(lengths, kv_heads, dim, fmt, page, seed=0):
    g = generator(seed)
    W = max(1, max((n + page - 1) // page for n in lengths))
    pages = len(lengths) * W + 2
    attn = make_attention(2 * kv_heads, kv_heads, dim, fmt, page, pages)
    fill(attn, g)
    table = torch.randperm(pages, generator=g, device=DEV)[:len(lengths) * W].view(-1, W).to(torch.int32)
    weights = torch.rand(len(lengths), kv_heads, W * page, generator=g, device=DEV) ** 6
    weights *= torch.rand(weights.shape, generator=g, device=DEV) > 0.2  # (many zeros: ties)
    return attn, table, weights, g


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
@pytest.mark.parametrize("kv_heads,dim,page", [(4, 128, 64), (8, 128, 256), (2, 64, 128), (1, 64, 64)])
@pytest.mark.parametrize("lengths,budget,recent", [
    ([1], 1, 1), ([1], 0, 0), ([2], 1, 0), ([2], 1, 1), ([65], 64, 16), ([300, 1, 0, 64], 64, 0), ([700, 130], 128, 128),
    ([700, 130], 100, 400), ([1000], 900, 30), ([1000, 999], 333, 1), ([2100], 17, 4), ([1500], 1400, 300),
])
def test_evict(gpu_device, kv_heads, dim, page, fmt, lengths, budget, recent):
    announce(f"evict {kv_heads}x{dim} page {page} {fmt} {lengths} to {budget} recent {recent}")
    attn, table, weights, _ = make(lengths, kv_heads, dim, fmt, page, seed=len(lengths) + budget)
    check(attn, table, lengths, weights, budget, recent)


@pytest.mark.parametrize("fmt,dim,page", [("bf16", 128, 64), ("int8", 128, 256), ("bf16", 64, 128), ("int8", 64, 64)])
@pytest.mark.parametrize("length", [4100, 16500, 40000])
@pytest.mark.parametrize("share,recent", [(0.2, 200), (0.95, 64), (0.004, 3)])
def test_long_sequences(gpu_device, length, share, recent, fmt, dim, page):
    """Each of the selection's ways of holding its keys, many moves and few."""
    announce(f"evict {length} to {share} {fmt} {dim} page {page}")
    attn, table, weights, _ = make([length, length // 3], 2, dim, fmt, page, seed=length)
    check(attn, table, [length, length // 3], weights, int(length * share), recent)


@pytest.mark.parametrize("kind", ["equal", "zeros", "negative", "nan", "infinite", "tiny", "close", "ascending", "descending"])
def test_selection(gpu_device, kind):
    """Ties go to the earlier position; NaN below all; signs, infinities and the smallest differences count."""
    announce(f"evict selection {kind}")
    n = 1234
    attn, table, weights, g = make([n, n], 2, 64, "bf16", 64, seed=3)
    r = torch.rand(weights.shape, generator=g, device=DEV)
    weights = {
        "equal": torch.full_like(weights, 0.375),
        "zeros": torch.where(r < 0.5, 0.0, -0.0),
        "negative": r - 0.5,
        "nan": torch.where(r < 0.3, float("nan"), torch.where(r < 0.4, float("-inf"), r)),
        "infinite": torch.where(r < 0.3, float("inf"), torch.where(r < 0.4, float("-inf"), r)),
        "tiny": (r * 40).floor() * 2.0 ** -149,
        "close": (0x3f800000 + (r * 700).to(torch.int32)).view(torch.float32),
        "ascending": torch.arange(weights.shape[2], device=DEV).float().expand_as(weights).clone(),
        "descending": -torch.arange(weights.shape[2], device=DEV).float().expand_as(weights).clone(),
    }[kind]
    weights[:, :, n:] = 0
    for budget, recent in ((1000, 10), (500, 0), (200, 150), (3, 1)):
        check(attn, table, [n, n], weights, budget, recent)


def test_budgets_per_sequence_in_place_strided_and_int64(gpu_device):
    announce("evict budgets")
    lengths = [500, 100, 0, 777, 300]
    attn, table, weights, g = make(lengths, 4, 128, "bf16", 64, seed=8)
    budgets = torch.tensor([100, 200, 5, 0, 299], device=DEV)
    check(attn, table, lengths, weights, budgets, 32, out=weights)
    attn, table, weights, g = make(lengths, 4, 128, "int8", 64, seed=9)
    whole = torch.rand(4, 7, 1000, generator=g, device=DEV)
    view = whole[:, 1:6, 3:900].transpose(0, 1)
    new = torch.empty(5, 4, 2000, device=DEV)[:, :, 9:906]
    check(attn, table.long(), lengths, view, budgets, 7, max_seq_len=777, out=new)
    check(attn, table, lengths, view, budgets, 7, out=view)


def test_twice_and_then_attention(gpu_device):
    """Attention over what is left equals attention over those tokens alone, wherever they lie."""
    from attn_cases import check_rows, reference

    announce("evict twice")
    attn, table, weights, g = make([400], 2, 64, "bf16", 64, seed=12)
    lens, w = check(attn, table, [400], weights, 300, 20)
    lens, w = check(attn, table, [300], w, 150, 20, out=w)
    k, v = rows(attn, table, 0, 150)
    q = torch.randn(1, 4, 64, generator=g, device=DEV).to(torch.bfloat16)
    got = attn.forward(q, table, lens)
    want, A = reference(q, k, v, torch.ones(1, 150, dtype=torch.bool, device=DEV), attn.scale)
    check_rows(got, want, A)


def test_out_of_range(gpu_device):
    """Reported, and left as it was."""
    announce("evict out of range")
    lengths = [300, 300, 300, 200]
    attn, table, weights, g = make(lengths, 2, 64, "bf16", 64, seed=13)
    before = state(attn)
    budgets = torch.tensor([-1, 100, 100, 100], device=DEV)
    lens = torch.tensor([300, -5, 400, 2 ** 20], device=DEV)
    new, out = attn.evict(table, lens, weights, budgets, 10)
    assert new.tolist() == [300, -5, 400, 2 ** 20]
    assert torch.equal(out, weights)
    assert all(torch.equal(a, b) for a, b in zip(state(attn), before))
    seen = attn.status()
    assert seen["bad_kept"] and seen["bad_length"] and not seen["bad_page"]
    with pytest.raises(N.NativeError, match="bad_kept"):
        attn.check_status()
    # a page that is none: its tokens stay, the rest moves
    table[0, 4] = -1
    w = torch.zeros_like(weights)
    w[0, :, 250], w[0, :, 270] = 1, 2  # (page 4 holds tokens 256 .. 319)
    k, v = rows(attn, table[:, :4], 0, 256)
    new, out = attn.evict(table[:1], torch.tensor([290], device=DEV), w[:1], 2, 0)
    assert new.tolist() == [2] and out[0, :, :2].tolist() == [[1.0, 2.0]] * 2
    got_k, got_v = rows(attn, table[:, :4], 0, 2)
    assert torch.equal(got_k, k[[250, 1]]) and torch.equal(got_v, v[[250, 1]])
    with pytest.raises(N.NativeError, match="bad_page"):
        attn.check_status()


def test_graph(gpu_device):
    """Captured with the attention that fills the weights: replays follow lengths and weights."""
    announce("evict in a graph")
    attn, table, weights, g = make([500, 320], 2, 64, "int8", 64, seed=14)
    twin, _, _, _ = make([500, 320], 2, 64, "int8", 64, seed=14)
    lens = torch.tensor([500, 320], dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            new, out = attn.evict(table, lens, weights, 128, 32)
    torch.cuda.current_stream().wait_stream(side)
    for step in range(3):
        lens.copy_(torch.tensor([500 - 100 * step, 320 - step], device=DEV))
        weights.copy_(torch.rand(weights.shape, generator=g, device=DEV))
        graph.replay()
        want_lens, want = twin.evict(table, lens, weights, 128, 32)
        torch.cuda.synchronize()
        assert torch.equal(new, want_lens) and torch.equal(out, want)
        assert all(torch.equal(a, b) for a, b in zip(state(attn), state(twin)))


def test_refused(gpu_device):
    attn, table, weights, _ = make([200, 100], 2, 64, "bf16", 64, seed=15)
    lens = torch.tensor([200, 100], dtype=torch.int32, device=DEV)
    for args, kw in (((table, lens, weights.half(), 10, 2), {}), ((table, lens, weights[:1], 10, 2), {}),
                     ((table, lens[:1], weights, 10, 2), {}), ((table, lens, weights, 10, -1), {}),
                     ((table, lens, weights, torch.tensor([1.0, 2.0], device=DEV), 2), {}),
                     ((table, lens, weights, 10, 2), {"out": weights[:, :, :64]}),
                     ((table, lens, weights[:, :1].expand(-1, 2, -1), 10, 2), {}),
                     ((table, lens, weights[:, :, :200], 10, 2), {"out": weights[:, :, 8:208]})):
        with pytest.raises((ValueError, N.NativeError)):
            attn.evict(*args, **kw)
    assert attn.evict(table[:0], lens[:0], weights[:0], 10, 2)[0].shape == (0,)
