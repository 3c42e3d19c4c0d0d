"""Host-side checks of the append, selection and sparse attention entry points (no GPU): refusals
before any CUDA call."""

from __future__ import annotations

import ctypes

import pytest
import torch


def test_c_entry_points_refuse_bad_arguments() -> None:
    from faquant_b200 import _lib

    lib = _lib.load()
    p = ctypes.c_void_p(256)
    pool = (p, 4, 1 << 20)

    def append(dtype=0, heads=4, d=128, page=16, q=p, cos=p, sin=p, ld=64, rows=9, eps=1e-6, norm=0, rope=1, ss=0, out=p,
               levels=123, total=4):
        return lib.faq_hif4_kv_append(q, p, p, dtype, total, heads, 2, d, 512, 128, 256, 128, 256, 128, p, p, norm, eps, cos,
                                      sin, rope, ld, rows, None, None, ss, 1, out, 512, 128, *pool, page, p, 3, 3, p, p, 1,
                                      levels, 123, None)

    assert append(q=None) == 1 and "null" in _lib.last_error()
    assert append(out=None) == 1
    assert append(heads=3) == 1 and "multiple" in _lib.last_error()
    assert append(heads=0) == 1
    assert append(d=96) == 3 and append(page=24) == 3
    assert append(dtype=7) == 1 and append(norm=5) == 1 and append(rope=5) == 1
    assert append(sin=None) == 1 and "go together" in _lib.last_error()
    assert append(ld=63) == 1 and append(rows=0) == 1
    assert append(eps=-1.0) == 1 and append(eps=float("nan")) == 1
    assert append(ss=64) == 1
    assert append(levels=5) == 1
    assert append(total=-1) == 1 and append(total=1 << 31) == 1
    assert append(total=0) == 0

    def bounds(d=128, total=4, out=p, page=16):
        return lib.faq_hif4_key_bounds(*pool, page, 2, d, p, 3, 3, p, p, 1, total, out, None)

    assert bounds(out=None) == 1 and bounds(out=ctypes.c_void_p(8)) == 1 and bounds(d=32) == 3 and bounds(page=8) == 3
    assert bounds(total=-1) == 1 and bounds(total=0) == 0

    def select(q=p, heads=4, count=5, first=1, last=2, columns=3, bounds=p, out=p, total=4):
        return lib.faq_hif4_select_pages(q, total, heads, 512, 128, bounds, 4, 16, 2, 128, p, columns, columns, p, p, 1, count,
                                         first, last, out, None, None)

    assert select(q=None) == 1 and select(bounds=None) == 1 and select(out=None) == 1
    assert select(heads=5) == 1 and select(heads=258) == 3 and "128 query heads" in _lib.last_error()
    assert select(columns=32769) == 3 and "columns" in _lib.last_error()
    assert select(count=2) == 1 and select(last=0) == 1 and select(first=-1) == 1 and select(count=0, first=0) == 1
    assert select(total=0) == 0 and select(total=-2) == 1

    def attend(q=p, heads=4, count=5, scale=1.0, qs=512, out=p, lists=p, total=4):
        return lib.faq_hif4_sparse_attention(q, total, heads, qs, 128, *pool, 16, 2, 128, p, 3, 3, p, p, 1, lists, count,
                                             ctypes.c_float(scale), out, 512, 128, None)

    assert attend(q=None) == 1 and attend(out=None) == 1 and attend(lists=None) == 1
    assert attend(heads=3) == 1 and attend(count=0) == 1 and attend(qs=12) == 1 and "strides" in _lib.last_error()
    assert attend(count=32769) == 3 and "32768" in _lib.last_error()
    assert attend(scale=0.0) == 1 and attend(scale=float("nan")) == 1 and attend(scale=float("inf")) == 1
    assert attend(q=ctypes.c_void_p(264)) == 1 and "aligned" in _lib.last_error()
    assert attend(total=0) == 0


def test_operators_refuse_cpu_tensors() -> None:
    from faquant_b200 import ops

    x = torch.zeros(2, 1, 64, dtype=torch.bfloat16)
    pages = torch.zeros(1, 1184, dtype=torch.uint8)
    bounds = torch.zeros(1, 1, 144, dtype=torch.uint8)
    table, cu, lens = (torch.zeros(*s, dtype=torch.int32) for s in ((1, 1), (2,), (1,)))
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.hif4_kv_append(x, x, x, pages, table, cu, lens, page_size=16)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.hif4_key_bounds(pages, bounds, table, cu, lens, page_size=16, total=2)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.hif4_select_pages(x, bounds, table, cu, lens, page_size=16, count=3)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.hif4_sparse_attention(x, pages, table, cu, lens, torch.zeros(2, 1, 3, dtype=torch.int32), page_size=16)
    assert ops.hif4_bounds_bytes(128) == 272 and ops.hif4_bounds_bytes(64) == 144
    with pytest.raises(ValueError):
        ops.hif4_bounds_bytes(96)


def test_sparse_caches_are_checked_when_made() -> None:
    from faquant_b200.kv_cache import PagedKVCache

    for bad in (dict(sparse_pages=2, sparse_first=1, sparse_last=2), dict(sparse_pages=3, sparse_last=0),
                dict(sparse_pages=3, sparse_first=-1)):
        with pytest.raises(ValueError, match="sparse_pages"):
            PagedKVCache(1, 1, 64, max_length=100, page_size=16, device="cpu", **bad)
    with pytest.raises(ValueError, match="32768 pages"):
        PagedKVCache(1, 1, 64, max_length=1 << 20, num_pages=4, page_size=16, device="cpu", sparse_pages=4)
    cache = PagedKVCache(2, 3, 64, max_length=100, page_size=16, device="cpu", sparse_pages=4)
    assert cache.bounds.shape == (2, 7, 3, 144)
    assert PagedKVCache(2, 3, 64, max_length=100, page_size=16, device="cpu").bounds is None
