"""C ABI of the adapters, checked without a GPU: declarations, sizes, and what is refused before a launch."""
import ctypes
import os
import re

import pytest

from nano_ktrans_amd import NativeAdapters
from nano_ktrans_amd import _native as N

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "nkt_lora.h")


def test_header_declarations_match_binding_and_library():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    declared = sorted(set(re.findall(r"\b(nkt_lora_\w+)\s*\(", text)))
    assert declared == sorted(N.LORA_SYMBOLS)
    for name in declared:
        assert hasattr(N.lib(), name), name


def _create(n=4, width=128, outs=(64, 128), rank=24):
    err = ctypes.create_string_buffer(256)
    array = (ctypes.c_int * max(1, len(outs)))(*outs) if outs is not None else None
    return N.lib().nkt_lora_create(n, width, array, 0 if outs is None else len(outs), rank, err, 256), err.value.decode()


@pytest.mark.parametrize("kw,msg", [
    (dict(n=0), "num_adapters"), (dict(n=4097), "num_adapters"), (dict(width=0), "in_features"),
    (dict(width=96), "in_features"), (dict(outs=None), "num_parts"), (dict(outs=()), "num_parts"),
    (dict(outs=(64,) * 5), "num_parts"), (dict(outs=(64, 96)), "out_features[1]"), (dict(outs=(0,)), "out_features[0]"),
    (dict(rank=0), "max_rank"), (dict(rank=129), "max_rank"), (dict(outs=(1 << 20, 64)), "2^20"),
    (dict(width=1 << 27), "2^31"),
])
def test_create_rejects(kw, msg):
    h, err = _create(**kw)
    assert not h
    assert msg in err


@pytest.mark.parametrize("rank,padded", [(1, 16), (16, 16), (17, 32), (64, 64), (65, 128)])
def test_sizes(rank, padded):
    h, err = _create(rank=rank)
    assert h, err
    L, eb, sz = N.lib(), ctypes.create_string_buffer(256), ctypes.c_size_t()
    rows = (2 * padded + 31) // 32 * 32
    for buf, want in enumerate((4 * rows * 128 * 2, 4 * 192 * padded * 2, 4 * 2 * 4, 4 * 2 * 4, 4)):
        assert L.nkt_lora_buffer_bytes(h, buf, ctypes.byref(sz), eb, 256) == 0 and sz.value == want
    assert L.nkt_lora_buffer_bytes(h, 5, ctypes.byref(sz), eb, 256) == -1
    assert L.nkt_lora_workspace_bytes(h, 64, ctypes.byref(sz), eb, 256) == 0 and sz.value == 0
    # grouped: 3 tiles of 32, and one more for each adapter and for those without
    assert L.nkt_lora_workspace_bytes(h, 70, ctypes.byref(sz), eb, 256) == 0
    assert sz.value == 8 * (2 * padded * 32 * 4 + 33 * 4)
    assert L.nkt_lora_workspace_bytes(h, -1, ctypes.byref(sz), eb, 256) == -1
    assert L.nkt_lora_forward(h, None, 0, None, 0, None, 0, None, 0, None, 0, None, eb, 256) == -1
    assert b"no buffers bound" in eb.value
    for bad in ((None, 0x10, 0x10, 0x10, 0x10), (0x10, 0x18, 0x10, 0x10, 0x10), (0x10, 0x10, 0x10, 0x10, None)):
        assert L.nkt_lora_bind(h, (ctypes.c_void_p * 5)(*bad), eb, 256) == -1 and b"buffer" in eb.value
    L.nkt_lora_destroy(h)
    assert L.nkt_lora_forward(None, None, 0, None, 0, None, 0, None, 0, None, 0, None, eb, 256) == -1


#          x         sx   base      sb   index   T  out       so   ws      bytes
FORWARD = [0x100000, 128, 0x200000, 192, 0x1000, 70, 0x300000, 192, 0x2000, 1 << 20]


@pytest.mark.parametrize("at,value,msg", [
    (0, None, b"null"), (2, None, b"null"), (4, None, b"null"), (6, None, b"null"), (0, 0x100008, b"aligned"),
    (1, 100, b"aligned"), (2, 0x200002, b"aligned"), (3, 100, b"aligned"), (6, 0x300004, b"aligned"), (7, 193, b"aligned"),
    (5, -1, b"num_tokens"), (5, 1 << 25, b"num_tokens"), (1, -128, b"strides"), (3, -192, b"strides"), (7, 128, b"strides"), (1, 1 << 28, b"strides"),
    (7, 0, b"strides"), (6, 0x200010, b"overlaps"), (6, 0x100010, b"overlaps"), (2, 0x300000 + 2 * 70 * 192 - 16, b"overlaps"),
    (8, None, b"workspace"), (9, 7 * 2 * 32 * 32 * 4 - 1, b"workspace"), (8, 0x2008, b"workspace"),
])
def test_forward_rejects(at, value, msg):
    h, err = _create()
    assert h, err
    L, eb = N.lib(), ctypes.create_string_buffer(256)
    assert L.nkt_lora_bind(h, (ctypes.c_void_p * 5)(*[0x10] * 5), eb, 256) == 0
    args = list(FORWARD)
    args[at] = value
    assert L.nkt_lora_forward(h, *args, None, eb, 256) == -1
    assert msg in eb.value
    args = list(FORWARD)
    args[5] = 0
    assert L.nkt_lora_forward(h, *args, None, eb, 256) == 0
    L.nkt_lora_destroy(h)


def test_no_cpu_fallback():
    with pytest.raises(N.NativeError):
        NativeAdapters(num_adapters=1, in_features=64, out_features=32, max_rank=4, device="cpu")
