"""``FusedAttentionBlock`` against a plain 64-bit attention between the same library projections, on the queries
that the block itself used, so that what is left is the attention's own error (attn_cases.py has its bound `off`
per value).  Through the output projection W that error is held by its norm over a row's hidden values:

    |got - (x + W want)| <= |off| s(W) + 2^-24 K |W| (|want| + off)       the projection's fp32 sums
                            + u (|W want| + the above) + u (|x + W want| + the above)   two roundings to bf16

s(W) the largest singular value.  A bound that a wrong attention passes as well would show nothing: each case also
checks that it tells apart an attention of zeros, of uniform weights, of another head's queries, of another mask
and of another sequence."""
import sys

import pytest
import torch
from torch import nn

from attn_cases import DEV, U, causal, dense, generator, randn, reference, tree_sees
from nano_ktrans_amd import FusedDecoderLayer, tree_mask_from_parents
from test_gpu_decoder_layer import D, H, HK, HQ, attention_block, batch_of, run

pytestmark = pytest.mark.gpu


def announce(msg):
    sys.__stderr__.write(f"[gpu-case] {msg}\n")
    sys.__stderr__.flush()


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
@pytest.mark.parametrize("qk_norm,bias", [(True, False), (False, True)])
@pytest.mark.parametrize("counts,firsts,drafted", [
    ([70, 9], [0, 0], False), ([1, 1], [3, 12], False), ([5, 30], [20, 64], False), ([7, 20], [11, 30], True)])
def test_attention_block_on_its_own_queries(gpu_device, fmt, qk_norm, bias, counts, firsts, drafted):
    announce(f"attention block {fmt} norm={qk_norm} bias={bias} rows {counts} after {firsts} drafted={drafted}")
    g = generator(sum(counts) + 100)
    block = attention_block(g, fmt, qk_norm, 12, bias)
    a = block.attention
    table = torch.randperm(12, generator=g, device=DEV)[:8].view(2, 4).to(torch.int32)
    layer = [FusedDecoderLayer(block, nn.Identity())]
    if max(firsts):
        run(layer, randn(g, sum(firsts), H), batch_of(layer, table, [0, 0], firsts))
    x = randn(g, sum(counts), H)
    mask = tree_mask_from_parents([[(j - 1) // 2 for j in range(n)] for n in counts], DEV) if drafted else None
    batch = batch_of(layer, table, firsts, counts, mask, decode=counts == [1, 1])
    got = run(layer, x, batch).double()
    held = a.k_cache.clone()
    with torch.no_grad():
        q, k, v = block.qkv_proj(block.norm(x)).split([HQ * D, HK * D, HK * D], dim=1)
    norms = {"q_norm": block.q_norm.weight, "k_norm": block.k_norm.weight, "eps": block.q_norm.eps} if qk_norm else {}
    q = a.write(q, k, v, batch.positions, batch.slots, block.rope, **norms)
    assert torch.equal(held, a.k_cache)  # (the projection repeats its bits: so do the queries)
    assert not any(a.status().values())

    w = block.o_proj.weight.detach().double()
    largest = float(torch.linalg.matrix_norm(w.cpu(), 2))
    rows = [torch.arange(f + n, device=DEV) for f, n in zip(firsts, counts)]
    cached = [dense(a, a.slots(table, torch.full_like(r, b), r)) for b, r in enumerate(rows)]
    at = [0, counts[0], sum(counts)]

    def expected(b, queries, sees, scale, keys_of=None):
        keys, values = cached[b if keys_of is None else keys_of]
        n = sees.shape[1]
        want, A = reference(queries[at[b]:at[b + 1]], keys[:n], values[:n], sees[:, :keys.shape[0]], scale)
        return want.flatten(1), A.flatten(1)

    for b, (n, first) in enumerate(zip(counts, firsts)):
        mine = slice(at[b], at[b + 1])
        sees = causal(n, first + n) if mask is None else tree_sees(mask[mine], n, first + n)
        want, A = expected(b, q, sees, a.scale)
        off = U * want.abs() + (U + U * U + 2.0 ** -9.9) * A
        out = want @ w.T
        total = x[mine].double() + out
        bound = off.norm(dim=1) * largest + 2.0 ** -24 * HQ * D * ((want.abs() + off) @ w.abs().T).norm(dim=1)
        bound = bound + U * (out.norm(dim=1) + bound)
        bound = bound + U * (total.norm(dim=1) + bound)
        assert bool(((got[mine] - total).norm(dim=1) <= bound).all()), f"sequence {b}"

        other = sees.clone()
        if mask is None and n > 1:
            other[:] = True                        # no causal mask
        elif mask is None:
            other[:, -1] = False                   # its own token unseen
        else:
            other = causal(n, first + n)           # a draft taken for a chunk
        wrong = {"zeros": torch.zeros_like(want), "uniform weights": expected(b, q, sees, 0.0)[0],
                 "another head's queries": expected(b, q.roll(1, dims=1), sees, a.scale)[0],
                 "another mask": expected(b, q, other, a.scale)[0]}
        if len(cached[1 - b][0]) >= first + n:
            wrong["another sequence"] = expected(b, q, sees, a.scale, keys_of=1 - b)[0]
        for what, value in wrong.items():
            missed = (got[mine] - (x[mine].double() + value @ w.T)).norm(dim=1) <= bound
            assert not bool(missed.all()), f"sequence {b}: {what} would pass"
