"""Attention in the launches of large and uneven batches, against the plain 64-bit implementation in attn_cases.py:
many sequences, chunks that a rule forces, long parts, and joins of many workgroups.  Page tables name only the pages
that a sequence needs."""
import sys

import pytest
import torch

from attn_cases import DEV, Problem, causal, check_rows, dense, generator, make_attention, poison, put, randn, reference, \
    split_rows, tree_sees
from nano_ktrans_amd import tree_mask_from_parents

pytestmark = pytest.mark.gpu


def announce(msg):
    sys.__stderr__.write(f"[gpu-case] {msg}\n")
    sys.__stderr__.flush()


def starts_of(counts):
    return torch.tensor(split_rows(counts), dtype=torch.int32, device=DEV)


def make_uneven(lengths, *, heads, kv_heads, dim, fmt, page, seed):
    """As make_problem, with as many pages as the sequences' tokens need: the table's other entries are -1."""
    g = generator(seed)
    need = [(n + page - 1) // page for n in lengths]
    attn = make_attention(heads, kv_heads, dim, fmt, page, sum(need) + 3)
    poison(attn)
    pages = torch.randperm(attn.num_pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(lengths), max(1, max(need))), -1, dtype=torch.int32, device=DEV)
    at = split_rows(need)
    for b, n in enumerate(need):
        table[b, :n] = pages[at[b]:at[b] + n]
    seqs = torch.repeat_interleave(torch.arange(len(lengths), device=DEV), torch.tensor(lengths, device=DEV))
    places = torch.cat([torch.arange(n, device=DEV) for n in lengths])
    slots = attn.slots(table, seqs, places)
    for part in slots.split(1 << 15):
        put(attn, part, randn(g, part.numel(), kv_heads, dim).float(), randn(g, part.numel(), kv_heads, dim).float())
    attn.check_status()
    ks, vs = [], []
    for part in slots.split(lengths):
        k, v = dense(attn, part)
        ks.append(k)
        vs.append(v)
    return Problem(attn, table, torch.tensor(lengths, dtype=torch.int32, device=DEV), list(lengths), ks, vs)


def check(p, counts, q, got, mask=None, every=1):
    """Every `every`-th row of each sequence, its first and its last."""
    at = split_rows(counts)
    for b, (n, length) in enumerate(zip(counts, p.lengths)):
        if n == 0:
            continue
        rows = sorted({*range(0, n, every), n - 1})
        sees = causal(n, length) if mask is None else tree_sees(mask[at[b]:at[b + 1]], n, length)
        pick = torch.tensor(rows, device=DEV)
        want, A = reference(q[at[b] + pick], p.k[b], p.v[b], sees[pick], p.attn.scale)
        check_rows(got[at[b] + pick], want, A, f"sequence {b} ({n} rows, {length} tokens)")
    assert not any(p.attn.status().values())


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
@pytest.mark.parametrize("seqs", [65, 130, 300])
def test_many_sequences_of_mixed_rows(gpu_device, fmt, seqs):
    """More sequences than one round of the search by 64 lanes holds, some without rows, in the launch that finds
    a tile's sequence; causal and drafted."""
    announce(f"{seqs} sequences of mixed rows {fmt}")
    g = generator(seqs)
    counts = torch.randint(0, 8, (seqs,), generator=g, device=DEV).tolist()
    for b in range(0, seqs, 9):
        counts[b] = 0
    counts[1], counts[seqs // 2], counts[seqs - 1] = 70, 33, 150
    context = torch.randint(0, 200, (seqs,), generator=g, device=DEV).tolist()
    lengths = [n + c for n, c in zip(counts, context)]
    p = make_uneven(lengths, heads=8, kv_heads=2, dim=64, fmt=fmt, page=64, seed=seqs)
    q = randn(g, sum(counts), 8, 64)
    check(p, counts, q, p.attn.forward(q, p.table, p.lens, starts_of(counts)), every=5)
    mask = tree_mask_from_parents([[(j - 1) // 2 for j in range(n)] for n in counts], DEV)
    check(p, counts, q, p.attn.forward_tree(q, mask, p.table, p.lens, starts_of(counts)), mask, every=5)


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
@pytest.mark.parametrize("seqs,longest", [(32, [5000, 4097, 2049]), (270, [9000, 4096, 4100])])
def test_single_tokens_in_forced_chunks(gpu_device, fmt, seqs, longest):
    """Batches that fill the card, in chunks of 2048 tokens (of 4096 where workgroups are many): a few long
    sequences in parts beside short ones in one."""
    announce(f"{seqs} single tokens, longest {longest} {fmt}")
    g = generator(seqs)
    lengths = torch.randint(1, 60, (seqs,), generator=g, device=DEV).tolist()
    for b, n in zip((0, seqs // 2, seqs - 1), longest):
        lengths[b] = n
    lengths[5] = 2048
    p = make_uneven(lengths, heads=32, kv_heads=4, dim=128, fmt=fmt, page=64, seed=seqs)
    q = randn(g, seqs, 32, 128)
    got = p.attn.forward(q, p.table, p.lens, max_seq_len=max(lengths))
    check(p, [1] * seqs, q, got)
    assert torch.equal(got, p.attn.forward(q, p.table, p.lens, max_seq_len=max(lengths)))


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
def test_drafts_of_few_rows_in_parts(gpu_device, fmt):
    """40 drafts of up to 64 rows, one on a long context: more items than the join's groups per row are for."""
    announce(f"40 drafts, one of a long context {fmt}")
    g = generator(40)
    counts = torch.randint(1, 17, (40,), generator=g, device=DEV).tolist()
    counts[7], counts[20] = 16, 0
    context = torch.randint(0, 300, (40,), generator=g, device=DEV).tolist()
    context[7], context[8] = 6000, 1500
    lengths = [n + c for n, c in zip(counts, context)]
    p = make_uneven(lengths, heads=8, kv_heads=2, dim=128, fmt=fmt, page=64, seed=41)
    q = randn(g, sum(counts), 8, 128)
    mask = tree_mask_from_parents([[(j - 1) // 3 for j in range(n)] for n in counts], DEV)
    bounds = {"max_queries": 16, "max_seq_len": max(lengths)}
    check(p, counts, q, p.attn.forward_tree(q, mask, p.table, p.lens, starts_of(counts), **bounds), mask)
    check(p, counts, q, p.attn.forward(q, p.table, p.lens, starts_of(counts), **bounds))


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
@pytest.mark.parametrize("counts,contexts", [([2100, 40], [0, 100]), ([2100, 40], [900, 5000]), ([1300, 700], [2000, 13000])])
def test_prompts_of_many_workgroups(gpu_device, fmt, counts, contexts):
    """512 to 1535 tile workgroups: not split while they are short, in three parts of long contexts, the last of
    which hold more pages than a wave keeps at a time (64)."""
    announce(f"many tile workgroups {fmt} rows {counts} contexts {contexts}")
    lengths = [n + c for n, c in zip(counts, contexts)]
    p = make_uneven(lengths, heads=32, kv_heads=32, dim=64, fmt=fmt, page=64, seed=sum(contexts))
    q = randn(generator(9), sum(counts), 32, 64)
    got = p.attn.forward(q, p.table, p.lens, starts_of(counts), max_queries=max(counts), max_seq_len=max(lengths))
    check(p, counts, q, got, every=61)
    mask = torch.full((sum(counts), (max(counts) + 63) // 64), -1, dtype=torch.int64, device=DEV)  # all of the draft
    got = p.attn.forward_tree(q, mask, p.table, p.lens, starts_of(counts), max_queries=max(counts),
                              max_seq_len=max(lengths))
    check(p, counts, q, got, mask, every=61)
