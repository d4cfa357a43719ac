"""The attention half of a decoder layer, and the whole layer.

nano_ktrans/models/mixtral.py:191-205 runs, before the MoE half:

    residual = hidden_states
    hidden_states = self.input_layernorm(hidden_states)
    hidden_states = self.self_attn(hidden_states, positions)    # projections, rotation, cache, attention
    hidden_states = residual + hidden_states

``FusedAttentionBlock`` computes the same over the paged cache of a
``NativeAttention``: the projections are the caller's nn.Linear modules; head
norms (architectures with ``use_qk_norm``), rotation and the cache write are
one launch on the projection's output, attention one or two.  Beside that it takes
low-rank adapters of the batch's requests on either projection (``NativeAdapters``),
positions on several axes, and a tensor that sums what each cached token got of the
attention, for ``NativeAttention.evict``.
``FusedDecoderLayer`` follows it with the MoE half (``FusedMoEBlock``).  Both are
for inference: their outputs carry no gradient.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Sequence

import torch
from torch import nn

from ..native_adapters import NativeAdapters
from ..native_attention import NativeAttention


@dataclass
class AttentionBatch:
    """Where a batch's tokens are: the same for every layer of a model (``NativeAttention.forward``)."""

    positions: torch.Tensor                       # [T] of the rotation, or [axes, T]
    slots: torch.Tensor                           # [T] in the cache; negative: padding
    page_table: torch.Tensor                      # [sequences, pages]
    seq_lens: torch.Tensor                        # [sequences], these tokens included
    query_starts: Optional[torch.Tensor] = None   # [sequences + 1]; None: one token per sequence
    max_queries: Optional[int] = None
    max_seq_len: Optional[int] = None
    tree_mask: Optional[torch.Tensor] = None      # [T, words]: drafted tokens
    adapters: Optional[torch.Tensor] = None       # [T] each token's adapter, negative: none; None: no token has one
    last: Optional[int] = None                    # whose rows count for the weights of cached tokens; None: all


class FusedAttentionBlock(nn.Module):
    """hidden + o_proj(attention(norm(hidden))).

    qkv_proj: nn.Linear(H, (num_heads + 2 num_kv_heads) * head_dim), queries, keys and values in this order;
    o_proj: nn.Linear(num_heads * head_dim, H); q_norm / k_norm: modules with ``weight`` [head_dim] and
    ``eps`` (both or neither); rope: ``rope_table``; rope_axes: the axis of each frequency (``rope_axes``), for
    positions on several axes; qkv_adapters / o_adapters: ``NativeAdapters`` beside the projections."""

    def __init__(self, input_layernorm: nn.Module, qkv_proj: nn.Module, o_proj: nn.Module, attention: NativeAttention,
                 rope: torch.Tensor, q_norm: Optional[nn.Module] = None, k_norm: Optional[nn.Module] = None,
                 rope_axes: Optional[Sequence[int]] = None, qkv_adapters: Optional[NativeAdapters] = None,
                 o_adapters: Optional[NativeAdapters] = None):
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
        for name, adapters, linear in (("qkv", qkv_adapters, qkv_proj), ("o", o_adapters, o_proj)):
            if adapters is not None and (adapters.in_features, adapters.columns) != (linear.in_features,
                                                                                     linear.out_features):
                raise ValueError(f"{name}_adapters take {adapters.in_features} features to {adapters.columns} columns, "
                                 f"{name}_proj {linear.in_features} to {linear.out_features}")
        self.norm = input_layernorm
        self.qkv_proj = qkv_proj
        self.o_proj = o_proj
        self.attention = attention
        self.rope = rope
        self.q_norm = q_norm
        self.k_norm = k_norm
        self.rope_axes = None if rope_axes is None else tuple(rope_axes)
        self.qkv_adapters = qkv_adapters
        self.o_adapters = o_adapters

    @torch.no_grad()
    def forward(self, hidden_states: torch.Tensor, batch: AttentionBatch,
                weights: Optional[torch.Tensor] = None) -> torch.Tensor:
        """weights: this layer's fp32 [sequences, kv_heads, positions], to which the attention's weights are added
        (``NativeAttention.forward_weights``, of the rows that ``batch.last`` names)."""
        if hidden_states.dtype != torch.bfloat16:
            raise ValueError("FusedAttentionBlock needs bf16 hidden states")
        if weights is not None and batch.tree_mask is not None:
            raise ValueError("the weights of drafted tokens are not summed: some of them will not be kept")
        a = self.attention
        x = hidden_states.reshape(-1, hidden_states.shape[-1])
        normed = self.norm(x)
        qkv = self.qkv_proj(normed)
        if self.qkv_adapters is not None and batch.adapters is not None:
            qkv = self.qkv_adapters.forward(normed, qkv, batch.adapters, out=qkv)
        q, k, v = qkv.split([a.num_heads * a.head_dim, a.num_kv_heads * a.head_dim, a.num_kv_heads * a.head_dim], dim=1)
        norms = {}
        if self.q_norm is not None:
            norms = {"q_norm": self.q_norm.weight, "k_norm": self.k_norm.weight, "eps": float(self.q_norm.eps)}
        q = a.write(q, k, v, batch.positions, batch.slots, self.rope, axes=self.rope_axes, **norms)
        where = (batch.page_table, batch.seq_lens, batch.query_starts)
        bounds = {"max_queries": batch.max_queries, "max_seq_len": batch.max_seq_len}
        # in place of the queries: rows behind the last sequence (padding) stay numbers
        if weights is not None:  # (which are told from the queries once more, after the output)
            out = a.forward_weights(q, weights, *where, **bounds, last=batch.last, out=torch.zeros_like(q))
        elif batch.tree_mask is None:
            out = a.forward(q, *where, **bounds, out=q)
        else:
            out = a.forward_tree(q, batch.tree_mask, *where, **bounds, out=q)
        out = out.flatten(1)
        projected = self.o_proj(out)
        if self.o_adapters is not None and batch.adapters is not None:
            projected = self.o_adapters.forward(out, projected, batch.adapters, out=projected)
        return hidden_states + projected.view(hidden_states.shape)


class FusedDecoderLayer(nn.Module):
    """Attention half, then MoE half: ``moe_block(attention_block(hidden, batch, weights))``."""

    def __init__(self, attention_block: FusedAttentionBlock, moe_block: nn.Module):
        super().__init__()
        self.attention_block = attention_block
        self.moe_block = moe_block

    def forward(self, hidden_states: torch.Tensor, batch: AttentionBatch,
                weights: Optional[torch.Tensor] = None) -> torch.Tensor:
        # (an attention half that knows of no weights is called without them)
        args = () if weights is None else (weights,)
        return self.moe_block(self.attention_block(hidden_states, batch, *args))
