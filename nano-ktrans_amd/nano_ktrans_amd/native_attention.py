"""One layer's paged key / value cache and the attention over it, driven through
the C ABI (include/nkt_attn.h).

``NativeAttention`` owns the cache (torch tensors in HBM) and enqueues on
torch's current HIP stream.  No call synchronises the host (``status`` and
``check_status`` do).  Activations are bf16; the cache holds bf16 or int8 with one
fp32 scale per token and head.  For inference: no call gives gradients.

A serving program keeps, per batch, a page table [sequences, pages], the
sequences' lengths, and where its new tokens go:

    q = attn.write(q, k, v, positions, attn.slots(page_table, seq_of_token, positions), rope,
                   q_norm=..., k_norm=...)
    out = attn.forward(q, page_table, seq_lens)                                   # one token per sequence
    out = attn.forward(q, page_table, seq_lens, query_starts, max_queries=...)    # prompts, chunks
    out = attn.forward_tree(q, tree_mask, page_table, seq_lens, query_starts)     # drafted tokens
    attn.keep(page_table, context_lens, kept, counts)                             # the accepted ones
"""
from __future__ import annotations

import ctypes
from typing import Dict, Optional, Sequence, Tuple

import torch

from . import _native as N

_FORMATS = {"bf16": N.CACHE_BF16, "int8": N.CACHE_INT8}

# words of the status tensor: the kernels' (bits added atomically), and two that ``slots`` writes: the first says
# nothing, the second that a token's page was bad
_STATUS_KERNELS, _STATUS_SLOTS = 0, 2

# the current stream's handle without building a Stream object (2 us of a 12 us call)
_current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)


def rope_table(max_position: int, head_dim: int, theta: float = 1e6, device=None) -> torch.Tensor:
    """fp32 [max_position, head_dim]: the cosines, then the sines, of position * theta^(-2 i / head_dim),
    i < head_dim / 2.  The angles are taken in 64 bits: a far position times an fp32 frequency would be off
    by a good part of a turn."""
    inv = theta ** (-torch.arange(0, head_dim, 2, dtype=torch.float64) / head_dim)
    angle = torch.arange(max_position, dtype=torch.float64).unsqueeze(1) * inv
    return torch.cat([angle.cos(), angle.sin()], dim=1).to(torch.float32).to(device if device is not None else "cpu")


def tree_mask_from_parents(parents: Sequence[Sequence[int]], device=None) -> torch.Tensor:
    """The tree mask of a batch of drafts: parents[b][j] is the draft-local index of token j's parent in
    sequence b (below j), or -1 for a token that follows the context.  Returns int64 [tokens, words]: each
    token sees its ancestors and itself."""
    words = max([1] + [(len(p) + 63) // 64 for p in parents])
    rows = []
    for b, tree in enumerate(parents):
        sees = []
        for j, parent in enumerate(tree):
            if not -1 <= parent < j:
                raise ValueError(f"draft {b}: token {j} has parent {parent}, expected -1 .. {j - 1}")
            sees.append((sees[parent] if parent >= 0 else 0) | 1 << j)
        rows += [[(bits >> (64 * w) & (1 << 64) - 1) for w in range(words)] for bits in sees]
    signed = [[w - (1 << 64) if w >> 63 else w for w in row] for row in rows]
    return torch.tensor(signed, dtype=torch.int64).reshape(-1, words).to(device if device is not None else "cpu")


class NativeAttention:
    """One layer's cache: shapes, pages and the calls on them.

    ``k_cache`` [num_pages, num_kv_heads, page_size, head_dim], ``v_cache`` [num_pages, num_kv_heads,
    page_size / U, head_dim, U] (U = 8 bf16 or 16 int8 tokens: 16 bytes) and, for "int8", ``k_scales`` and
    ``v_scales`` [num_pages, num_kv_heads, page_size] are ordinary tensors; ``read`` gives rows of them in
    their natural order.  A call takes its temporary memory from torch's allocator, so calls on different
    streams and captured graphs do not share any.  What is written on one stream and read on another needs
    the caller's event between the two, as with any tensor."""

    def __init__(
        self,
        *,
        num_heads: int,
        num_kv_heads: int,
        head_dim: int,
        num_pages: int,
        page_size: int = 64,
        cache_format: str = "bf16",
        scale: Optional[float] = None,
        device: Optional[torch.device] = None,
    ):
        self.device = torch.device(device if device is not None else "cuda")
        if self.device.type != "cuda" or not torch.cuda.is_available():
            raise N.NativeError(
                "attention runs only on a ROCm GPU (gfx950); got device "
                f"{self.device} with torch.cuda.is_available()={torch.cuda.is_available()}")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        if cache_format not in _FORMATS:
            raise ValueError(f"cache_format must be one of {sorted(_FORMATS)}, got {cache_format!r}")
        self.lib = N.lib()
        self.err = N.ErrBuf()
        self.num_heads = num_heads
        self.num_kv_heads = num_kv_heads
        self.head_dim = head_dim
        self.num_pages = num_pages
        self.page_size = page_size
        self.cache_format = cache_format
        self.scale = float(scale) if scale is not None else max(head_dim, 1) ** -0.5
        if not 0.0 < self.scale < 1e30:
            raise ValueError(f"scale must be a positive number, got {scale}")
        h = self.lib.nkt_attn_create(num_heads, num_kv_heads, head_dim, _FORMATS[cache_format], page_size, num_pages,
                                     self.err.buf, self.err.size)
        if not h:
            raise N.NativeError(f"nkt_attn_create failed: {self.err.buf.value.decode()}")
        self.handle = ctypes.c_void_p(h)
        self._entry = {name: getattr(self.lib, name) for name in N.ATTN_SYMBOLS}
        self._ws_bytes: Dict[Tuple[int, int, int, int], int] = {}
        int8 = cache_format == "int8"
        unit = 16 if int8 else 8
        dtype = torch.int8 if int8 else torch.bfloat16
        # zeroed: a page handed to a sequence before it is written holds numbers
        self.k_cache = torch.zeros(num_pages, num_kv_heads, page_size, head_dim, dtype=dtype, device=self.device)
        self.v_cache = torch.zeros(num_pages, num_kv_heads, page_size // unit, head_dim, unit, dtype=dtype,
                                   device=self.device)
        self.k_scales = self.v_scales = None
        if int8:
            self.k_scales = torch.zeros(num_pages, num_kv_heads, page_size, device=self.device)
            self.v_scales = torch.zeros_like(self.k_scales)
        self._status = torch.zeros(4, dtype=torch.int32, device=self.device)
        self._slots_status = self._status[_STATUS_SLOTS - 1:_STATUS_SLOTS + 1]
        ptrs = (ctypes.c_void_p * N.ATTN_NUM_BUFS)()
        for i, t in enumerate((self.k_cache, self.v_cache, self.k_scales, self.v_scales, self._status)):
            ptrs[i] = t.data_ptr() if t is not None else None
        self.err.check(self.lib.nkt_attn_bind_cache(self.handle, ptrs, self.err.buf, self.err.size),
                       "nkt_attn_bind_cache")

    def __del__(self):
        h = getattr(self, "handle", None)
        if h is not None and h.value:
            try:
                self.lib.nkt_attn_destroy(h)
            except Exception:
                pass

    # ------------------------------------------------------------------ arguments
    def _call(self, name: str, *args) -> None:
        """An entry point on this layer's device and torch's current stream there."""
        fn, index, err = self._entry[name], self.device.index, self.err
        if torch.cuda.current_device() == index:
            rc = fn(self.handle, *args, _current_stream(index), err.buf, err.size)
        else:
            with torch.cuda.device(self.device):
                rc = fn(self.handle, *args, _current_stream(index), err.buf, err.size)
        if rc != N.NKT_OK:
            err.check(rc, name)

    def _on_device(self, t: torch.Tensor, name: str) -> None:
        if t.device != self.device:
            raise ValueError(f"{name} on {t.device}, layer on {self.device}")

    def _ints(self, t: torch.Tensor, dtype: torch.dtype, shape: Tuple[int, ...], name: str) -> torch.Tensor:
        self._on_device(t, name)
        if t.dtype != dtype:
            if t.dtype not in (torch.int32, torch.int64):
                raise ValueError(f"{name} must be an integer tensor, got {t.dtype}")
            # (what 32 bits do not hold stays out of range, rather than what its lower half says)
            t = t.to(dtype) if dtype == torch.int64 else t.clamp(-2 ** 31, 2 ** 31 - 1).to(dtype)
        if t.shape != shape:
            raise ValueError(f"{name} is {tuple(t.shape)}, expected {shape}")
        return t if t.is_contiguous() else t.contiguous()

    def _rows(self, t: torch.Tensor, heads: int, name: str) -> torch.Tensor:
        """[T, heads, head_dim] bf16 (or [T, heads * head_dim])."""
        self._on_device(t, name)
        if t.dtype != torch.bfloat16:
            raise ValueError(f"{name} dtype {t.dtype}, attention expects {torch.bfloat16}")
        shape = t.shape
        if len(shape) == 2 and shape[1] == heads * self.head_dim:
            return t.unflatten(1, (heads, self.head_dim))
        if len(shape) != 3 or shape[1] != heads or shape[2] != self.head_dim:
            raise ValueError(f"{name} is {tuple(shape)}, expected [tokens, {heads}, {self.head_dim}]")
        return t

    def _strided(self, t: torch.Tensor, heads: int, name: str) -> torch.Tensor:
        """Rows whose heads are contiguous and whose tokens are 8-byte aligned: as they are, else a copy."""
        t = self._rows(t, heads, name)
        s = t.stride()
        fits = s[2] == 1 and (s[1] == self.head_dim or heads == 1) and s[0] % 4 == 0 and t.data_ptr() % 8 == 0
        return t if fits else t.clone(memory_format=torch.contiguous_format)

    def _dense(self, t: torch.Tensor, heads: int, name: str) -> torch.Tensor:
        t = self._rows(t, heads, name)
        fits = t.is_contiguous() and t.data_ptr() % 16 == 0
        return t if fits else t.clone(memory_format=torch.contiguous_format)

    def _out(self, out: Optional[torch.Tensor], tokens: int, heads: int, name: str = "out") -> torch.Tensor:
        if out is None:
            return torch.empty(tokens, heads, self.head_dim, dtype=torch.bfloat16, device=self.device)
        if out.dtype != torch.bfloat16 or tuple(out.shape) != (tokens, heads, self.head_dim) \
                or not out.is_contiguous() or out.device != self.device or out.data_ptr() % 16:
            raise ValueError(f"{name} must be a contiguous, 16-byte aligned [{tokens}, {heads}, {self.head_dim}] "
                             f"{torch.bfloat16} tensor on {self.device}")
        return out

    def _norm_weight(self, w: Optional[torch.Tensor], name: str) -> Optional[torch.Tensor]:
        if w is None:
            return None
        self._on_device(w, name)
        if w.numel() != self.head_dim:
            raise ValueError(f"{name} must have {self.head_dim} entries, got {w.numel()}")
        if w.dtype != torch.bfloat16 or w.dim() != 1 or not w.is_contiguous() or w.data_ptr() % 8:
            w = w.detach().to(torch.bfloat16).reshape(-1).clone(memory_format=torch.contiguous_format)
        return w

    # ------------------------------------------------------------------ cache
    def slots(self, page_table: torch.Tensor, seqs: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
        """int64 slots of the tokens at ``positions`` of the sequences ``seqs`` (rows of the page table): -1 for
        a negative position (padding), a slot past the cache, which ``write`` reports, for one past the table.
        A token whose entry of the table is no page of the cache (an unallocated one) gets a slot that nothing
        is stored at and is reported here, as ``bad_page``: ``write`` could not tell a negative one from padding."""
        B, W = page_table.shape
        seqs, positions = seqs.long(), positions.long()
        past = self.num_pages * self.page_size
        if B == 0 or W == 0:
            return torch.where(positions < 0, -1, past)
        # (each of these is a launch: ranges are told by what a clamp changes)
        at = torch.div(positions, self.page_size, rounding_mode="floor")
        seq, entry = seqs.clamp(0, B - 1), at.clamp(0, W - 1)
        inside = (seq == seqs) & (entry == at)
        pages = page_table[seq, entry]
        if pages.dtype == torch.int64:
            pages = pages.clamp(-1, self.num_pages)
        slots = torch.add(positions % self.page_size, pages, alpha=self.page_size)
        bad = inside & (slots != slots.clamp(0, past - 1))
        # (a word that only this call writes, and never reads: kernels on other streams add their bits to theirs)
        self._slots_status.index_fill_(0, bad.view(-1).long(), N.ATTN_STATUS["bad_page"])
        return torch.where(inside, slots, past).masked_fill(positions < 0, -1)

    def write(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor,
              rope: torch.Tensor, q_norm: Optional[torch.Tensor] = None, k_norm: Optional[torch.Tensor] = None,
              eps: float = 1e-6, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Queries and keys normalised per head (by ``q_norm`` / ``k_norm`` [head_dim], where given) and rotated
        by their positions' rows of ``rope`` (``rope_table``); keys and values stored at ``slots`` (negative:
        not stored, padding, at any position), the queries returned [T, num_heads, head_dim].  q, k and v may be
        parts of one projection's output.  Norm weights of another type are rounded to bf16, the activations'.
        The slots of one call have to be distinct."""
        q = self._strided(q, self.num_heads, "q")
        T = q.shape[0]
        k, v = self._strided(k, self.num_kv_heads, "k"), self._strided(v, self.num_kv_heads, "v")
        if k.shape[0] != T or v.shape[0] != T:
            raise ValueError(f"q has {T} tokens, k {k.shape[0]}, v {v.shape[0]}")
        positions = self._ints(positions, torch.int64, (T,), "positions")
        slots = self._ints(slots, torch.int64, (T,), "slots")
        self._on_device(rope, "rope")
        if rope.dtype != torch.float32 or rope.dim() != 2 or rope.shape[1] != self.head_dim \
                or not rope.is_contiguous() or rope.data_ptr() % 16:
            raise ValueError(f"rope must be a contiguous, 16-byte aligned fp32 [positions, {self.head_dim}] table")
        q_norm, k_norm = self._norm_weight(q_norm, "q_norm"), self._norm_weight(k_norm, "k_norm")
        out = self._out(out, T, self.num_heads)
        if T:
            self._call("nkt_attn_write", q.data_ptr(), q.stride(0), k.data_ptr(), k.stride(0), v.data_ptr(),
                       v.stride(0), positions.data_ptr(), slots.data_ptr(), rope.data_ptr(), rope.shape[0],
                       q_norm.data_ptr() if q_norm is not None else None,
                       k_norm.data_ptr() if k_norm is not None else None, eps, T, out.data_ptr())
        return out

    def read(self, slots: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        """The keys and values that the cache holds at ``slots`` [n], bf16 [n, num_kv_heads, head_dim] each;
        zeros for a negative slot."""
        slots = self._ints(slots, torch.int64, (slots.numel(),), "slots")
        n = slots.numel()
        k = torch.empty(n, self.num_kv_heads, self.head_dim, dtype=torch.bfloat16, device=self.device)
        v = torch.empty_like(k)
        if n:
            self._call("nkt_attn_read", slots.data_ptr(), n, k.data_ptr(), v.data_ptr())
        return k, v

    def _table(self, page_table: torch.Tensor) -> torch.Tensor:
        if page_table.dim() != 2:
            raise ValueError(f"page_table is {tuple(page_table.shape)}, expected [sequences, pages]")
        return self._ints(page_table, torch.int32, page_table.shape, "page_table")

    def keep(self, page_table: torch.Tensor, context_lens: torch.Tensor, kept: torch.Tensor,
             counts: torch.Tensor) -> None:
        """Moves the accepted tokens of each sequence's draft behind its context: the key and value at position
        context_lens[b] + kept[b, i] to context_lens[b] + i, i < counts[b].  kept [sequences, width] ascends in
        each row up to its count."""
        page_table = self._table(page_table)
        B, W = page_table.shape
        context_lens = self._ints(context_lens, torch.int32, (B,), "context_lens")
        if kept.dim() != 2:
            raise ValueError(f"kept is {tuple(kept.shape)}, expected [sequences, width]")
        kept = self._ints(kept, torch.int32, (B, kept.shape[1]), "kept")
        counts = self._ints(counts, torch.int32, (B,), "counts")
        self._call("nkt_attn_keep", page_table.data_ptr(), W, context_lens.data_ptr(), kept.data_ptr(),
                   kept.shape[1], counts.data_ptr(), B)

    # ------------------------------------------------------------------ attention
    def _workspace_bytes(self, *sizes: int) -> int:
        """nkt_attn_workspace_bytes of a forward call's sizes (a serving loop has few of them)."""
        need = self._ws_bytes.get(sizes)
        if need is None:
            nbytes = ctypes.c_size_t(0)
            self.err.check(self.lib.nkt_attn_workspace_bytes(self.handle, *sizes, ctypes.byref(nbytes), self.err.buf,
                                                             self.err.size), "nkt_attn_workspace_bytes")
            if len(self._ws_bytes) >= 4096:
                self._ws_bytes.clear()
            need = self._ws_bytes[sizes] = nbytes.value
        return need

    def _attend(self, name: str, q, head_args, page_table, seq_lens, query_starts, max_queries, max_seq_len, out):
        q = self._dense(q, self.num_heads, "q")
        T = q.shape[0]
        page_table = self._table(page_table)
        B, W = page_table.shape
        seq_lens = self._ints(seq_lens, torch.int32, (B,), "seq_lens")
        if query_starts is not None:
            query_starts = self._ints(query_starts, torch.int32, (B + 1,), "query_starts")
            max_queries = T if max_queries is None else min(int(max_queries), T)
        else:
            if T != B:
                raise ValueError(f"q has {T} rows for {B} sequences: pass query_starts")
            max_queries = 1
        most = W * self.page_size
        max_seq_len = most if max_seq_len is None else min(int(max_seq_len), most)
        out = self._out(out, T, self.num_heads)
        if T == 0 or B == 0:
            return out
        need = self._workspace_bytes(T, B, max_queries, max_seq_len)
        ws = torch.empty(need, dtype=torch.uint8, device=self.device) if need else None
        self._call(name, q.data_ptr(), *head_args, page_table.data_ptr(), W, seq_lens.data_ptr(),
                   query_starts.data_ptr() if query_starts is not None else None, T, B, max_queries, max_seq_len,
                   self.scale, out.data_ptr(), ws.data_ptr() if ws is not None else None, need)
        return out

    def forward(self, q: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor,
                query_starts: Optional[torch.Tensor] = None, *, max_queries: Optional[int] = None,
                max_seq_len: Optional[int] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Causal attention of each sequence's last rows over its part of the cache, [T, num_heads, head_dim].

        page_table [sequences, pages] and seq_lens [sequences] (this call's tokens included) describe the
        sequences; query_starts [sequences + 1] their rows of q (None: one row each, a decode step).
        max_queries and max_seq_len bound the rows of one sequence and the lengths: known to the caller
        without asking the device, they choose the launch (default: all of q, the whole page table).  A
        row that sees nothing is zero; rows behind the last sequence are left as ``out`` (which may be q
        itself) had them."""
        return self._attend("nkt_attn_forward", q, (), page_table, seq_lens, query_starts, max_queries, max_seq_len,
                            out)

    def forward_tree(self, q: torch.Tensor, tree_mask: torch.Tensor, page_table: torch.Tensor,
                     seq_lens: torch.Tensor, query_starts: Optional[torch.Tensor] = None, *,
                     max_queries: Optional[int] = None, max_seq_len: Optional[int] = None,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """``forward`` for drafted tokens: a row sees the tokens before the draft and, of the draft, the tokens j
        whose bit j % 64 of tree_mask[row, j // 64] (int64, ``tree_mask_from_parents``) is set."""
        if tree_mask.dim() != 2 or tree_mask.dtype != torch.int64:
            raise ValueError(f"tree_mask must be int64 [tokens, words], got {tree_mask.dtype} {tuple(tree_mask.shape)}")
        tree_mask = self._ints(tree_mask, torch.int64, (q.shape[0], tree_mask.shape[1]), "tree_mask")
        return self._attend("nkt_attn_forward_tree", q, (tree_mask.data_ptr(), tree_mask.shape[1]), page_table,
                            seq_lens, query_starts, max_queries, max_seq_len, out)

    # ------------------------------------------------------------------ status
    def status(self) -> Dict[str, bool]:
        """What calls found out of range on the device since the status was last cleared (synchronises)."""
        torch.cuda.synchronize(self.device)
        words = self._status.tolist()
        word = words[_STATUS_KERNELS] | words[_STATUS_SLOTS]
        return {name: bool(word & bit) for name, bit in N.ATTN_STATUS.items()}

    def check_status(self, clear: bool = True) -> None:
        """Raise ``NativeError`` if a call found something out of range (after clearing it when ``clear``)."""
        bad = [name for name, seen in self.status().items() if seen]
        if bad and clear:
            self._status.zero_()
            torch.cuda.synchronize(self.device)
        if bad:
            raise N.NativeError(f"attention status: {bad}")
