"""The attention half of a decoder layer, and the whole layer.

nano_ktrans/models/mixtral.py:191-205 runs, before the MoE half:

    residual = hidden_states
    hidden_states = self.input_layernorm(hidden_states)
    hidden_states = self.self_attn(hidden_states, positions)    # projections, rotation, cache, attention
    hidden_states = residual + hidden_states

``FusedAttentionBlock`` computes the same over the paged cache of a
``NativeAttention``: the projections are the caller's nn.Linear modules; head
norms (architectures with ``use_qk_norm``), rotation and the cache write are
one launch on the projection's output, attention one or two.
``FusedDecoderLayer`` follows it with the MoE half (``FusedMoEBlock``).  Both are
for inference: their outputs carry no gradient.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch
from torch import nn

from ..native_attention import NativeAttention


@dataclass
class AttentionBatch:
    """Where a batch's tokens are: the same for every layer of a model (``NativeAttention.forward``)."""

    positions: torch.Tensor                       # [T] of the rotation
    slots: torch.Tensor                           # [T] in the cache; negative: padding
    page_table: torch.Tensor                      # [sequences, pages]
    seq_lens: torch.Tensor                        # [sequences], these tokens included
    query_starts: Optional[torch.Tensor] = None   # [sequences + 1]; None: one token per sequence
    max_queries: Optional[int] = None
    max_seq_len: Optional[int] = None
    tree_mask: Optional[torch.Tensor] = None      # [T, words]: drafted tokens


class FusedAttentionBlock(nn.Module):
    """hidden + o_proj(attention(norm(hidden))).

    qkv_proj: nn.Linear(H, (num_heads + 2 num_kv_heads) * head_dim), queries, keys and values in this order;
    o_proj: nn.Linear(num_heads * head_dim, H); q_norm / k_norm: modules with ``weight`` [head_dim] and
    ``eps`` (both or neither); rope: ``rope_table``."""

    def __init__(self, input_layernorm: nn.Module, qkv_proj: nn.Module, o_proj: nn.Module, attention: NativeAttention,
                 rope: torch.Tensor, q_norm: Optional[nn.Module] = None, k_norm: Optional[nn.Module] = None):
        super().__init__()
        if (q_norm is None) != (k_norm is None):
            raise ValueError("q_norm and k_norm go together")
        if q_norm is not None and q_norm.eps != k_norm.eps:
            raise ValueError(f"q_norm.eps={q_norm.eps} and k_norm.eps={k_norm.eps} differ")
        a = attention
        width = (a.num_heads + 2 * a.num_kv_heads) * a.head_dim
        if qkv_proj.out_features != width or o_proj.in_features != a.num_heads * a.head_dim:
            raise ValueError(f"qkv_proj gives {qkv_proj.out_features} columns, expected {width}; o_proj takes "
                             f"{o_proj.in_features}, expected {a.num_heads * a.head_dim}")
        self.norm = input_layernorm
        self.qkv_proj = qkv_proj
        self.o_proj = o_proj
        self.attention = attention
        self.rope = rope
        self.q_norm = q_norm
        self.k_norm = k_norm

    @torch.no_grad()
    def forward(self, hidden_states: torch.Tensor, batch: AttentionBatch) -> torch.Tensor:
        if hidden_states.dtype != torch.bfloat16:
            raise ValueError("FusedAttentionBlock needs bf16 hidden states")
        a = self.attention
        x = hidden_states.reshape(-1, hidden_states.shape[-1])
        qkv = self.qkv_proj(self.norm(x))
        q, k, v = qkv.split([a.num_heads * a.head_dim, a.num_kv_heads * a.head_dim, a.num_kv_heads * a.head_dim], dim=1)
        norms = {}
        if self.q_norm is not None:
            norms = {"q_norm": self.q_norm.weight, "k_norm": self.k_norm.weight, "eps": float(self.q_norm.eps)}
        q = a.write(q, k, v, batch.positions, batch.slots, self.rope, **norms)
        where = (batch.page_table, batch.seq_lens, batch.query_starts)
        bounds = {"max_queries": batch.max_queries, "max_seq_len": batch.max_seq_len}
        # in place of the queries: rows behind the last sequence (padding) stay numbers
        if batch.tree_mask is None:
            out = a.forward(q, *where, **bounds, out=q)
        else:
            out = a.forward_tree(q, batch.tree_mask, *where, **bounds, out=q)
        return hidden_states + self.o_proj(out.flatten(1)).view(hidden_states.shape)


class FusedDecoderLayer(nn.Module):
    """Attention half, then MoE half: ``moe_block(attention_block(hidden, batch))``."""

    def __init__(self, attention_block: FusedAttentionBlock, moe_block: nn.Module):
        super().__init__()
        self.attention_block = attention_block
        self.moe_block = moe_block

    def forward(self, hidden_states: torch.Tensor, batch: AttentionBatch) -> torch.Tensor:
        return self.moe_block(self.attention_block(hidden_states, batch))
