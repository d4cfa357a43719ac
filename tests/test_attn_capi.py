"""C ABI of the attention half, checked without a GPU: declarations, sizes, and what is refused before a launch."""
import ctypes
import os
import re

import pytest
import torch

from nano_ktrans_amd import _native as N
from nano_ktrans_amd import rope_table, tree_mask_from_parents

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "nkt_attn.h")


def _declared():
    return sorted(set(re.findall(r"\b(nkt_attn_\w+)\s*\(", re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S))))


def test_header_declarations_match_binding_and_library():
    assert _declared() == sorted(N.ATTN_SYMBOLS)
    for name in _declared():
        assert hasattr(N.lib(), name), name


def _create(heads=8, kv=2, dim=128, fmt=N.CACHE_BF16, page=64, pages=10):
    err = ctypes.create_string_buffer(256)
    return N.lib().nkt_attn_create(heads, kv, dim, fmt, page, pages, err, 256), err.value.decode()


@pytest.mark.parametrize("kw,msg", [
    (dict(heads=0), "num_heads"), (dict(kv=0), "num_heads"), (dict(heads=7), "num_heads"),
    (dict(heads=2, kv=4), "num_heads"), (dict(heads=2048, kv=1), "num_heads"), (dict(dim=96), "head_dim"),
    (dict(dim=0), "head_dim"), (dict(fmt=2), "cache_format"), (dict(page=16), "page_size"), (dict(page=0), "page_size"),
    (dict(page=512), "page_size"), (dict(pages=0), "num_pages"), (dict(pages=1 << 31), "num_pages"),
])
def test_create_rejects(kw, msg):
    h, err = _create(**kw)
    assert not h
    assert msg in err


@pytest.mark.parametrize("fmt,es", [(N.CACHE_BF16, 2), (N.CACHE_INT8, 1)])
def test_cache_sizes(fmt, es):
    h, err = _create(fmt=fmt, pages=1 << 20, page=256)
    assert h, err
    eb, sz = ctypes.create_string_buffer(256), ctypes.c_size_t()
    rows = (1 << 20) * 2 * 256
    want = [rows * 128 * es, rows * 128 * es, rows * 4 if es == 1 else 0, rows * 4 if es == 1 else 0, 4]
    for buf, nbytes in enumerate(want):
        assert N.lib().nkt_attn_cache_bytes(h, buf, ctypes.byref(sz), eb, 256) == 0
        assert sz.value == nbytes
    assert N.lib().nkt_attn_cache_bytes(h, 5, ctypes.byref(sz), eb, 256) == -1
    N.lib().nkt_attn_destroy(h)


@pytest.fixture
def bound():
    """A handle bound to addresses that nothing reads: every call below is refused before a launch."""
    h, err = _create()
    assert h, err
    ptrs = (ctypes.c_void_p * 5)(0x1000, 0x2000, None, None, 0x3000)
    eb = ctypes.create_string_buffer(256)
    assert N.lib().nkt_attn_bind_cache(h, ptrs, eb, 256) == 0
    yield h
    N.lib().nkt_attn_destroy(h)


def test_calls_need_a_bound_cache():
    L, eb = N.lib(), ctypes.create_string_buffer(256)
    h, _ = _create()
    assert L.nkt_attn_read(h, None, 0, None, None, None, eb, 256) == -1 and b"no cache bound" in eb.value
    assert L.nkt_attn_read(None, None, 0, None, None, None, eb, 256) == -1 and b"null handle" in eb.value
    for bad in ((None, 0x1000, None, None, 0x1000), (0x1000, 0x1008, None, None, 0x1000),
                (0x1000, 0x1000, None, None, None)):
        assert L.nkt_attn_bind_cache(h, (ctypes.c_void_p * 5)(*bad), eb, 256) == -1 and b"buffer" in eb.value
    L.nkt_attn_destroy(h)
    h, _ = _create(fmt=N.CACHE_INT8)
    assert L.nkt_attn_bind_cache(h, (ctypes.c_void_p * 5)(0x1000, 0x1000, None, 0x1000, 0x1000), eb, 256) == -1
    L.nkt_attn_destroy(h)


# one argument of a good call at a time, and what the message names
WRITE = [0x1000, 640, 0x1000, 640, 0x1000, 640, 0x1000, 0x1000, 0x1000, 16, None, None, 1e-6, 4, 0x1000]


@pytest.mark.parametrize("at,value,msg", [
    (0, None, b"null"), (2, None, b"null"), (4, None, b"null"), (6, None, b"null"), (7, None, b"null"),
    (8, None, b"null"), (14, None, b"null"), (0, 0x1002, b"aligned"), (1, 641, b"aligned"), (3, 2, b"aligned"),
    (5, 1, b"aligned"), (8, 0x1008, b"aligned"), (10, 0x1004, b"aligned"), (9, 0, b"rope_rows"),
    (13, -1, b"num_tokens"), (13, 1 << 28, b"num_tokens"),
])
def test_write_rejects(bound, at, value, msg):
    args = list(WRITE)
    args[at] = value
    eb = ctypes.create_string_buffer(256)
    assert N.lib().nkt_attn_write(bound, *args, None, eb, 256) == -1
    assert msg in eb.value


@pytest.mark.parametrize("args,msg", [
    ((None, 4, 0x1000, 0x1000), b"slots"), ((0x1000, 4, 0x1008, 0x1000), b"aligned"),
    ((0x1000, 4, 0x1000, None), b"v_out"), ((0x1000, -1, 0x1000, 0x1000), b"num_slots"),
    ((0x1000, 1 << 30, 0x1000, 0x1000), b"num_slots"),
])
def test_read_rejects(bound, args, msg):
    eb = ctypes.create_string_buffer(256)
    assert N.lib().nkt_attn_read(bound, *args, None, eb, 256) == -1
    assert msg in eb.value


@pytest.mark.parametrize("args,msg", [
    ((None, 4, 0x1000, 0x1000, 4, 0x1000, 2), b"null"), ((0x1000, 4, 0x1000, None, 4, 0x1000, 2), b"null"),
    ((0x1000, -1, 0x1000, 0x1000, 4, 0x1000, 2), b"table_width"), ((0x1000, 4, 0x1000, 0x1000, -1, 0x1000, 2), b"kept_width"),
    ((0x1000, 4, 0x1000, 0x1000, 4, 0x1000, -2), b"num_seqs"), ((0x1000, 1 << 25, 0x1000, 0x1000, 4, 0x1000, 2), b"2^30"),
])
def test_keep_rejects(bound, args, msg):
    eb = ctypes.create_string_buffer(256)
    assert N.lib().nkt_attn_keep(bound, *args, None, eb, 256) == -1
    assert msg in eb.value


#           q       table  width lens   starts  T  B  mq  max_len  scale out     ws    bytes
FORWARD = [0x1000, 0x1000, 4, 0x1000, 0x1000, 4, 2, 3, 200, 1.0, 0x1000, None, 0]


@pytest.mark.parametrize("at,value,msg", [
    (0, None, b"null"), (1, None, b"null"), (3, None, b"null"), (10, None, b"null"), (0, 0x1008, b"aligned"),
    (10, 0x1004, b"aligned"), (2, -1, b"table_width"), (2, 1 << 25, b"table_width"), (4, None, b"query_starts"),
    (5, -1, b"num_tokens"), (6, -1, b"num_seqs"), (5, 1 << 28, b"2^27"), (7, -1, b"max_queries"),
    (8, -1, b"max_seq_len"), (9, 0.0, b"scale"), (9, -1.0, b"scale"), (9, float("nan"), b"scale"), (9, float("inf"), b"scale"),
])
def test_forward_rejects(bound, at, value, msg):
    L, eb = N.lib(), ctypes.create_string_buffer(256)
    args = list(FORWARD)
    args[at] = value
    assert L.nkt_attn_forward(bound, *args, None, eb, 256) == -1
    assert msg in eb.value
    assert L.nkt_attn_forward_tree(bound, args[0], 0x1000, 1, *args[1:], None, eb, 256) == -1
    assert msg in eb.value


def test_forward_rejects_more_workgroups_than_a_launch_holds(bound):
    """Many sequences of a long bound: 2^23 sequences x 2 heads x 512 chunks."""
    L, eb, sz = N.lib(), ctypes.create_string_buffer(256), ctypes.c_size_t()
    assert L.nkt_attn_workspace_bytes(bound, 1 << 23, 1 << 23, 1, 1 << 20, ctypes.byref(sz), eb, 256) == -1
    assert b"workgroups" in eb.value
    assert L.nkt_attn_workspace_bytes(bound, 64, 64, 1, 1 << 20, ctypes.byref(sz), eb, 256) == 0 and sz.value > 0
    assert L.nkt_attn_workspace_bytes(bound, 0, 0, 0, 1 << 20, ctypes.byref(sz), eb, 256) == 0


@pytest.mark.parametrize("mask,words", [(None, 1), (0x1000, 0), (0x1000, -1), (0x1000, 1 << 29)])
def test_tree_rejects_masks(bound, mask, words):
    eb = ctypes.create_string_buffer(256)
    assert N.lib().nkt_attn_forward_tree(bound, FORWARD[0], mask, words, *FORWARD[1:], None, eb, 256) == -1
    assert b"tree_mask" in eb.value


def test_empty_calls_launch_nothing(bound):
    L, eb = N.lib(), ctypes.create_string_buffer(256)
    write = list(WRITE)
    write[13] = 0
    assert L.nkt_attn_write(bound, *write, None, eb, 256) == 0
    assert L.nkt_attn_read(bound, None, 0, None, None, None, eb, 256) == 0
    assert L.nkt_attn_keep(bound, None, 4, None, None, 4, None, 0, None, eb, 256) == 0
    assert L.nkt_attn_forward(bound, None, None, 4, None, 0x1000, 0, 2, 0, 200, 1.0, None, None, 0, None, eb, 256) == 0


def test_no_cpu_fallback():
    from nano_ktrans_amd import NativeAttention

    with pytest.raises(N.NativeError):
        NativeAttention(num_heads=8, num_kv_heads=2, head_dim=128, num_pages=4, device="cpu")


def test_rope_table():
    t = rope_table(5000, 8, theta=100.0)
    assert t.shape == (5000, 8) and t.dtype == torch.float32
    angle = torch.tensor(4999.0, dtype=torch.float64) * 100.0 ** -0.25
    assert abs(float(t[4999, 1]) - float(torch.cos(angle))) <= 2.0 ** -24
    assert abs(float(t[4999, 5]) - float(torch.sin(angle))) <= 2.0 ** -24


def test_tree_mask_from_parents():
    m = tree_mask_from_parents([[-1, 0, 0, 1, -1], [-1]])
    assert m.tolist() == [[0b1], [0b11], [0b101], [0b1011], [0b10000], [0b1]]
    chain = tree_mask_from_parents([list(range(-1, 129))])
    assert chain.shape == (130, 3)
    assert chain[63].tolist() == [-1, 0, 0] and chain[129].tolist() == [-1, -1, 3] and chain[62].tolist()[0] == (1 << 63) - 1
    assert tree_mask_from_parents([]).shape == (0, 1)
    for bad in ([[0]], [[-1, 1]], [[-2]]):
        with pytest.raises(ValueError):
            tree_mask_from_parents(bad)
