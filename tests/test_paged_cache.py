"""The paged cache's refusals that need no GPU, and its host's argument checks through the C ABI."""

import ctypes

import pytest
import torch

from anna_amd import _lib
from anna_amd.paged_cache import PagedInt4Cache


def handle(**over):
    f = dict(dtype=0, num_layers=1, num_pages=8, kv_heads=2, q_heads=4, head_dim=64, max_sequences=4, max_pages=4, pool=64,
             table=64)
    f.update(over)
    h = ctypes.c_void_p()
    _lib.call("anna_mi_paged_create", ctypes.byref(_lib.PagedDesc(**f)), ctypes.byref(h))
    return h


def i32(*v):
    return (ctypes.c_int32 * len(v))(*v)


def i64(*v):
    return (ctypes.c_int64 * len(v))(*v)


def test_struct_sizes():
    assert _lib.load().anna_mi_sizeof_paged_desc() == ctypes.sizeof(_lib.PagedDesc)
    assert _lib.load().anna_mi_sizeof_paged_span() == ctypes.sizeof(_lib.PagedSpan)


@pytest.mark.parametrize("over,match", [
    (dict(dtype=2), "dtype"), (dict(head_dim=96), "head_dim"), (dict(q_heads=5), "multiple"), (dict(kv_heads=0), "multiple"),
    (dict(num_layers=0), "num_layers"), (dict(num_pages=0), "num_pages"), (dict(max_sequences=0), "max_sequences"),
    (dict(max_pages=1 << 40), "max_pages"), (dict(max_sequences=1 << 20, max_pages=1 << 20), "max_"),
    (dict(pool=None), "null"), (dict(pool=24), "aligned"),
])
def test_create_refuses(over, match):
    with pytest.raises(RuntimeError, match=match):
        handle(**over)


def test_calls_are_checked_before_anything_is_launched():
    h = handle()
    seqs = i32(0, 0)
    _lib.call("anna_mi_paged_add", h, 2, seqs)
    assert list(seqs) == [0, 1]
    for name, args, match in [
        ("anna_mi_paged_add", (3, i32(0, 0, 0)), "2 of 4 are free"),
        ("anna_mi_paged_add", (1, None), "bad arguments"),
        ("anna_mi_paged_fork", (1, i32(3), i32(0), None), "not in use"),
        ("anna_mi_paged_fork", (3, i32(0, 0, 0), i32(0, 0, 0), None), "free"),
        ("anna_mi_paged_extend", (1, i32(5), i64(1), None, None), "not in use"),
        ("anna_mi_paged_extend", (2, i32(1, 1), i64(1, 1), None, None), "twice"),
        ("anna_mi_paged_extend", (1, i32(1), i64(-1), None, None), "count"),
        ("anna_mi_paged_extend", (1, i32(1), i64(257), None, None), "at most 256 fit"),
        ("anna_mi_paged_extend", (1, i32(1), i64((1 << 63) - 1), None, None), "at most 256 fit"),
        ("anna_mi_paged_extend", (1, None, i64(1), None, None), "bad arguments"),
        ("anna_mi_paged_truncate", (0, 1, None), "length 1 of a sequence of 0"),
        ("anna_mi_paged_truncate", (3, 0, None), "not in use"),
        ("anna_mi_paged_free", (1, i32(-1), None), "not in use"),
        ("anna_mi_paged_resize", (0, 64, None), "pages"),
        ("anna_mi_paged_resize", (8, 64, None), "another"),
        ("anna_mi_paged_resize", (8, 72, None), "aligned"),
        ("anna_mi_paged_span_plan", (1, i32(0), i64(0), i64(1), ctypes.byref(_lib.PagedSpan())), "holds 0"),
        ("anna_mi_paged_span_plan", (1, i32(0), i64(0), i64(0), None), "null span"),
        ("anna_mi_paged_span_fill", (0, None, None, None, ctypes.byref(_lib.PagedSpan()), None), "null or unaligned"),
        ("anna_mi_paged_store", (0, ctypes.byref(_lib.PagedSpan()), 16, 0, 0, 16, 0, 0, 0, None), "null span"),
        ("anna_mi_paged_attend", (0, None, 16, 0, 0, None, 0, 0, 16, 1.0, 0, None), "null span"),
    ]:
        with pytest.raises(RuntimeError, match=match):
            _lib.call(name, h, *args)
    with pytest.raises(RuntimeError, match="pages needed, 8 of 8"):
        big = handle(max_pages=64)
        _lib.call("anna_mi_paged_add", big, 1, seqs)
        _lib.call("anna_mi_paged_extend", big, 1, i32(0), i64(64 * 9), None, None)
    with pytest.raises(RuntimeError, match="null handle"):
        _lib.call("anna_mi_paged_add", None, 1, seqs)
    lengths = i64(7, 7, 7)
    live = ctypes.c_int64(-1)
    _lib.call("anna_mi_paged_lengths", h, 3, i32(0, 3, 99), lengths, ctypes.byref(live))
    assert list(lengths) == [0, -1, -1] and live.value == 0
    span = _lib.PagedSpan(buf=64)
    span.tokens = 1
    for args, match in [((5, ctypes.byref(span), 16, 0, 0, None, 0, 0, 16, 1.0, 0, None), "layer 5 of 1"),
                        ((0, ctypes.byref(span), 16, 0, 0, None, 0, 0, 16, 0.0, 0, None), "scaling"),
                        ((0, ctypes.byref(span), 16, 4, 0, None, 0, 0, 16, 1.0, 0, None), "16-byte"),
                        ((0, ctypes.byref(span), 16, 0, 0, 8, 0, 0, 16, 1.0, 0, None), "16-byte"),
                        ((0, ctypes.byref(span), None, 0, 0, None, 0, 0, 16, 1.0, 0, None), "null query")]:
        with pytest.raises(RuntimeError, match=match):
            _lib.call("anna_mi_paged_attend", h, *args)
    _lib.call("anna_mi_paged_destroy", h)


@pytest.mark.parametrize("over,error,match", [
    (dict(head_dim=96), ValueError, "head_dim"), (dict(dtype=torch.float32), ValueError, "float16"),
    (dict(q_heads=3), ValueError, "multiple"), (dict(num_pages=0), ValueError, "positive"),
    (dict(device="cpu"), RuntimeError, "ROCm device"),
])
def test_constructor_refuses(over, error, match):
    kw = dict(num_layers=1, num_pages=4, kv_heads=2, q_heads=4, head_dim=64, max_sequences=2, max_length=100)
    kw.update(over)
    with pytest.raises(error, match=match):
        PagedInt4Cache(**kw)
