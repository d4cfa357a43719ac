"""Low-rank adapters of many requests beside a shared projection, driven through the C ABI (include/nkt_lora.h).

``NativeAdapters`` owns the adapters of one projection (torch tensors in HBM) and enqueues on torch's current HIP
stream.  No call synchronises the host (``status`` and ``check_status`` do).  Activations and adapters are bf16.  For
inference: no call gives gradients.

    adapters = NativeAdapters(num_adapters=16, in_features=2048, out_features=(4096, 512, 512), max_rank=32)
    adapters.load(3, a_q, b_q, scale=alpha / rank, part=0)      # a [rank, in], b [out, rank]
    qkv = qkv_proj(hidden)
    qkv = adapters.forward(hidden, qkv, index, out=qkv)         # index [T]: each token's adapter, -1: none
"""
from __future__ import annotations

import ctypes
from typing import Dict, Optional, Sequence, Union

import torch

from . import _native as N
from .native_attention import _current_stream


class NativeAdapters:
    """The adapters of one projection, or of several that share their input (``out_features`` a sequence: parts,
    side by side in the output, each with its own matrices).

    out[t, part] = base[t, part] + scale * (x[t] a^T) b^T with the a, b and scale of the token's adapter.  An adapter
    or part that nothing was loaded into adds nothing.  Adapters may be loaded and cleared between calls; what is
    loaded on one stream and used on another needs the caller's event between the two."""

    def __init__(self, *, num_adapters: int, in_features: int, out_features: Union[int, Sequence[int]], max_rank: int,
                 device: Optional[torch.device] = None):
        self.device = torch.device(device if device is not None else "cuda")
        if self.device.type != "cuda" or not torch.cuda.is_available():
            raise N.NativeError(
                "adapters run only on a ROCm GPU (gfx950); got device "
                f"{self.device} with torch.cuda.is_available()={torch.cuda.is_available()}")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.lib = N.lib()
        self.err = N.ErrBuf()
        self.num_adapters = num_adapters
        self.in_features = in_features
        self.out_features = (out_features,) if isinstance(out_features, int) else tuple(out_features)
        self.max_rank = max_rank
        parts = len(self.out_features)
        h = self.lib.nkt_lora_create(num_adapters, in_features, (ctypes.c_int * parts)(*self.out_features), parts,
                                     max_rank, self.err.buf, self.err.size)
        if not h:
            raise N.NativeError(f"nkt_lora_create failed: {self.err.buf.value.decode()}")
        self.handle = ctypes.c_void_p(h)
        self.columns = sum(self.out_features)
        self._rank = next(r for r in (16, 32, 64, 128) if max_rank <= r)
        self._blocks = (parts * self._rank + 31) // 32
        # the layouts of include/nkt_lora.h
        self.a = torch.zeros(num_adapters, self._blocks, in_features // 64, 4, 2, 32, 8, dtype=torch.bfloat16,
                             device=self.device)
        self.b = torch.zeros(num_adapters, self.columns // 64, self._rank // 16, 2, 2, 32, 8, dtype=torch.bfloat16,
                             device=self.device)
        self.scales = torch.zeros(num_adapters, parts, device=self.device)
        self.ranks = torch.zeros(num_adapters, parts, dtype=torch.int32, device=self.device)
        self._status = torch.zeros(4, dtype=torch.int32, device=self.device)
        ptrs = (ctypes.c_void_p * N.LORA_NUM_BUFS)()
        for i, t in enumerate((self.a, self.b, self.scales, self.ranks, self._status)):
            ptrs[i] = t.data_ptr()
        self.err.check(self.lib.nkt_lora_bind(self.handle, ptrs, self.err.buf, self.err.size), "nkt_lora_bind")
        self._ws_bytes: Dict[int, int] = {}

    def __del__(self):
        h = getattr(self, "handle", None)
        if h is not None and h.value:
            try:
                self.lib.nkt_lora_destroy(h)
            except Exception:
                pass

    # ------------------------------------------------------------------ adapters
    def _slot(self, adapter: int, part: int) -> None:
        if not 0 <= adapter < self.num_adapters:
            raise ValueError(f"adapter {adapter} outside [0, {self.num_adapters})")
        if not 0 <= part < len(self.out_features):
            raise ValueError(f"part {part} outside [0, {len(self.out_features)})")

    @torch.no_grad()
    def load(self, adapter: int, a: torch.Tensor, b: torch.Tensor, scale: float = 1.0, part: int = 0) -> None:
        """a [rank, in_features] and b [out_features[part], rank] of an adapter's part, of any rank up to max_rank;
        other types than bf16 are rounded to it.  Replaces what was there."""
        self._slot(adapter, part)
        rank, out = a.shape[0] if a.dim() else 0, self.out_features[part]
        if a.dim() != 2 or a.shape[1] != self.in_features or not 1 <= rank <= self.max_rank:
            raise ValueError(f"a is {tuple(a.shape)}, expected [1 .. {self.max_rank}, {self.in_features}]")
        if tuple(b.shape) != (out, rank):
            raise ValueError(f"b is {tuple(b.shape)}, expected {(out, rank)}")
        if not a.is_floating_point() or not b.is_floating_point():
            raise ValueError(f"a and b must be floating point, got {a.dtype} and {b.dtype}")
        R = self._rank
        rows = torch.zeros(R, self.in_features, dtype=torch.bfloat16, device=self.device)
        rows[:rank] = a.to(device=self.device, dtype=torch.bfloat16)
        at = part * R + torch.arange(R, device=self.device)
        self.a[adapter, at // 32, :, :, :, at % 32] = \
            rows.view(R, -1, 2, 4, 8).transpose(2, 3)
        columns = torch.zeros(out, R, dtype=torch.bfloat16, device=self.device)
        columns[:, :rank] = b.to(device=self.device, dtype=torch.bfloat16)
        first = sum(self.out_features[:part]) // 64
        self.b[adapter, first:first + out // 64] = \
            columns.view(out // 64, 32, 2, R // 16, 2, 8).permute(0, 3, 2, 4, 1, 5)
        self.scales[adapter, part] = float(scale)
        self.ranks[adapter, part] = rank

    @torch.no_grad()
    def clear(self, adapter: int) -> None:
        """The adapter adds nothing from here on."""
        self._slot(adapter, 0)
        for t in (self.a, self.b, self.scales, self.ranks):
            t[adapter].zero_()

    # ------------------------------------------------------------------ forward
    def _rows(self, t: torch.Tensor, tokens: Optional[int], width: int, name: str) -> torch.Tensor:
        if t.device != self.device:
            raise ValueError(f"{name} on {t.device}, adapters on {self.device}")
        if t.dtype != torch.bfloat16:
            raise ValueError(f"{name} dtype {t.dtype}, adapters expect {torch.bfloat16}")
        if t.dim() != 2 or t.shape[1] != width or (tokens is not None and t.shape[0] != tokens):
            raise ValueError(f"{name} is {tuple(t.shape)}, expected [{'tokens' if tokens is None else tokens}, {width}]")
        return t

    @staticmethod
    def _fits(t: torch.Tensor) -> bool:
        """Rows of 16-byte pieces."""
        return t.stride(1) == 1 and t.stride(0) % 8 == 0 and t.stride(0) >= 0 and t.data_ptr() % 16 == 0

    @torch.no_grad()
    def forward(self, x: torch.Tensor, base: torch.Tensor, index: torch.Tensor,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """base [T, columns] plus what each token's adapter makes of x [T, in_features], one rounding to bf16; index
        [T]: adapters, in any order, negative for none (the output is then base's).  ``out`` may be base.  An index
        past the adapters counts as none and is reported."""
        x = self._rows(x, None, self.in_features, "x")
        T = x.shape[0]
        base = self._rows(base, T, self.columns, "base")
        if index.device != self.device:
            raise ValueError(f"index on {index.device}, adapters on {self.device}")
        if index.dtype not in (torch.int32, torch.int64) or tuple(index.shape) != (T,):
            raise ValueError(f"index must be {T} integers, got {index.dtype} {tuple(index.shape)}")
        index = index.to(torch.int64).contiguous()
        if out is None:
            out = torch.empty(T, self.columns, dtype=torch.bfloat16, device=self.device)
        elif not self._fits(self._rows(out, T, self.columns, "out")):
            raise ValueError(f"out must have contiguous, 16-byte aligned rows, got strides {out.stride()}")
        if T == 0:
            return out
        if not self._fits(x):
            x = x.clone(memory_format=torch.contiguous_format)
        if not self._fits(base):
            base = base.clone(memory_format=torch.contiguous_format)
        need = self._ws_bytes.get(T)
        if need is None:
            nbytes = ctypes.c_size_t(0)
            self.err.check(self.lib.nkt_lora_workspace_bytes(self.handle, T, ctypes.byref(nbytes), self.err.buf,
                                                             self.err.size), "nkt_lora_workspace_bytes")
            if len(self._ws_bytes) >= 4096:
                self._ws_bytes.clear()
            need = self._ws_bytes[T] = nbytes.value
        ws = torch.empty(need, dtype=torch.uint8, device=self.device) if need else None
        args = (self.handle, x.data_ptr(), x.stride(0), base.data_ptr(), base.stride(0), index.data_ptr(), T,
                out.data_ptr(), out.stride(0), ws.data_ptr() if ws is not None else None, need)
        err, i = self.err, self.device.index
        if torch.cuda.current_device() == i:
            rc = self.lib.nkt_lora_forward(*args, _current_stream(i), err.buf, err.size)
        else:
            with torch.cuda.device(self.device):
                rc = self.lib.nkt_lora_forward(*args, _current_stream(i), err.buf, err.size)
        if rc != N.NKT_OK:
            err.check(rc, "nkt_lora_forward")
        return out

    # ------------------------------------------------------------------ status
    def status(self) -> Dict[str, bool]:
        """What calls found out of range on the device since the status was last cleared (synchronises)."""
        torch.cuda.synchronize(self.device)
        word = int(self._status[0])
        return {name: bool(word & bit) for name, bit in N.LORA_STATUS.items()}

    def check_status(self, clear: bool = True) -> None:
        """Raise ``NativeError`` if a call found something out of range (after clearing it when ``clear``)."""
        bad = [name for name, seen in self.status().items() if seen]
        if bad and clear:
            self._status.zero_()
            torch.cuda.synchronize(self.device)
        if bad:
            raise N.NativeError(f"adapters status: {bad}")
