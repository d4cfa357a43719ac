"""Adapters: calls that a serving program makes beside others, and inputs at the edge of what is allowed.  Tolerances
as in test_gpu_adapters.py."""
import pytest
import torch

from attn_cases import DEV, randn
from nano_ktrans_amd import NativeAdapters
from test_gpu_adapters import Problem, announce

pytestmark = pytest.mark.gpu


def test_index_that_changes_during_calls(gpu_device):
    """Another stream writes one of two index arrays while calls run: each token gets the adapter of one of the
    two, whole and bit for bit, and nothing outside of the output is written."""
    announce("adapters, index changes")
    tokens, columns = 5000, 192
    p = Problem(6, 256, (128, 64), 16, seed=21)
    x, base = p.inputs(tokens)
    choices = [torch.randint(-1, 6, (tokens,), generator=p.g, device=DEV) for _ in range(2)]
    wants = [p.adapters.forward(x, base, index) for index in choices]
    for index, want in zip(choices, wants):
        p.check(x, base, index, want)
    index = choices[0].clone()
    outs = [torch.full((tokens + 200, columns), 7.0, dtype=torch.bfloat16, device=DEV) for _ in range(40)]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        with torch.cuda.stream(side):
            for j in range(4):
                index.copy_(choices[j % 2])
        p.adapters.forward(x, base, index, out=out[100:-100])
    torch.cuda.synchronize()
    for out in outs:
        got = out[100:-100]
        of = [(got == want).all(dim=1) for want in wants]
        assert bool((of[0] | of[1]).all())
        assert bool((out[:100] == 7.0).all() and (out[-100:] == 7.0).all())
    p.adapters.check_status()
    got = p.adapters.forward(x, base, index)
    assert torch.equal(got, wants[1])


@pytest.mark.parametrize("tokens", [5, 64, 200])
@pytest.mark.parametrize("max_rank", [8, 32, 64, 100])
def test_ranks_past_the_largest(gpu_device, tokens, max_rank):
    """The ranks' buffer is an ordinary tensor: numbers that no adapter can have are those that it can."""
    announce(f"adapters with ranks past {max_rank}, T={tokens}")
    p = Problem(3, 128, (64, 128), max_rank, seed=22, ranks=[max_rank] * 3)
    x, base = p.inputs(tokens)
    index = torch.arange(tokens, device=DEV) % 4 - 1
    largest = next(r for r in (16, 32, 64, 128) if max_rank <= r)  # (what was not loaded is zero)
    p.adapters.ranks.copy_(torch.tensor([[largest, 1], [largest, largest], [0, largest]]))
    want = p.adapters.forward(x, base, index)
    p.adapters.ranks.copy_(torch.tensor([[129, 1], [2 ** 31 - 1, 5000], [-(2 ** 31), 1 << 20]]))
    assert torch.equal(p.adapters.forward(x, base, index), want)


@pytest.mark.parametrize("tokens", [3, 64, 90])
def test_infinite_adapters(gpu_device, tokens):
    """An infinity in B times what is exactly a bf16 number (or itself an infinity) is an infinity of the product's
    sign; times zero it is NaN, as in the formula."""
    announce(f"adapters with infinities T={tokens}")
    adapters = NativeAdapters(num_adapters=1, in_features=64, out_features=64, max_rank=16)
    a, b = torch.ones(1, 64, device=DEV), torch.full((64, 1), float("inf"), device=DEV)
    b[32:] = float("-inf")
    adapters.load(0, a, b)
    x = torch.zeros(tokens, 64, dtype=torch.bfloat16, device=DEV)
    x[0, 9], x[1, 9] = 3.0, float("-inf")
    base = torch.zeros(tokens, 64, dtype=torch.bfloat16, device=DEV)
    out = adapters.forward(x, base, torch.zeros(tokens, dtype=torch.int64, device=DEV))
    want = torch.full((64,), float("inf"), dtype=torch.bfloat16, device=DEV)
    want[32:] = float("-inf")
    assert torch.equal(out[0], want) and torch.equal(out[1], -want)
    assert bool(torch.isnan(out[2:]).all())


@pytest.mark.parametrize("tokens", [60, 300, 3000])
def test_two_streams_at_once(gpu_device, tokens):
    """A captured call replayed on one stream beside eager calls on two others, with nothing between them."""
    announce(f"adapters on three streams T={tokens}")
    p = Problem(5, 512, (256, 128), 32, seed=23)
    inputs = [p.inputs(tokens) + (torch.randint(-1, 5, (tokens,), generator=p.g, device=DEV),) for _ in range(3)]
    alone = [p.adapters.forward(*x) for x in inputs]
    for (x, base, index), want in zip(inputs, alone):
        p.check(x, base, index, want)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[0]):
        captured = p.adapters.forward(*inputs[0])
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(8):
        with torch.cuda.stream(streams[0]):
            graph.replay()
        for i in (1, 2):
            with torch.cuda.stream(streams[i]):
                outs[i - 1].append(p.adapters.forward(*inputs[i]))
    torch.cuda.synchronize()
    assert torch.equal(captured, alone[0])
    for i in (1, 2):
        assert all(torch.equal(out, alone[i]) for out in outs[i - 1])
    p.adapters.check_status()
