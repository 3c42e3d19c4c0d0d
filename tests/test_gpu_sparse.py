"""Appending to the paged HiF4 cache (faq_hif4_kv_append), the bounds and the selection of pages
(faq_hif4_key_bounds, faq_hif4_select_pages) and the attention over listed pages
(faq_hif4_sparse_attention), against 64-bit references.

Tolerances, derived. Keys are computed in fp64 and rounded once, bounds and scores are exact: all
of these are compared bit for bit. q: one bf16 rounding, at most 2^-8 of the value, of an
fp32 result. Its errors, in units of 2^-24 of the row's 2-norm: the norm's factor 16 (a sum of 16
squares per lane and three joins, the reciprocal root, two products), the rotation 2 sqrt(2), the
smoothing 1, seven stages of the transform 7 and its factor 2: below 2^5, and where channels are
smoothed times the ratio of the greatest factor to the least; 2^-18 of the norm is taken.
The attention is held to the bound of the dense one (test_gpu_paged.py): (2^-8 + 2^-8 + 2^-12) A."""

from __future__ import annotations

import math

import pytest
import torch

import sparse_reference as ref
from paged_reference import Pool, quantized

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
BOUND = 2.0**-8 + 2.0**-8 + 2.0**-12


def _randn(*shape, seed, dtype=torch.bfloat16, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).to(DEV)


def _int32(*values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _no_status():
    assert _status() == 0


def _status():
    from faquant_b200 import _lib

    torch.cuda.synchronize()
    return _lib.device_status(reset=True)


def _tables(rows, d, dtype=torch.float32, wide=False):
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    if wide:
        angle = torch.cat((angle, angle), 1)
    return angle.cos().to(dtype).to(DEV), angle.sin().to(dtype).to(DEV)


def _pos(lens, new):
    return torch.tensor([p for _, p in ref.positions(lens, new)], dtype=torch.long)


def _bounds(pool):
    from faquant_b200 import ops

    return torch.full((pool.pages.shape[0], pool.kv_heads, ops.hif4_bounds_bytes(pool.d)), 0x5A, dtype=torch.uint8, device=DEV)


# ------------------------------------------------------------------ append
OPTIONS = {
    "nothing": {},
    "rope": dict(rope=torch.float32),
    "norm": dict(norm=torch.bfloat16),
    "qwen3": dict(norm=torch.bfloat16, rope=torch.float32),
    "hadamard": dict(rotate=True),
    "deployed": dict(norm=torch.float32, rope=torch.bfloat16, wide=True, smooth=1, offset=True, rotate=True),
    "per head": dict(rope=torch.float32, smooth=2, rotate=True),
}


def _append(pool, q, k, v, new, lens, options, seed=90, **kw):
    """Calls the operator and the reference: ``(q', reference q, its error bound, reference keys)``."""
    from faquant_b200 import ops

    d, h, heads = pool.d, pool.kv_heads, q.shape[1]
    q_norm, k_norm = ((1 + 0.3 * torch.randn(d, generator=torch.Generator().manual_seed(seed + i))).to(
        options.get("norm", torch.float32)).to(DEV) if "norm" in options else None for i in range(2))
    cos, sin = _tables(max(lens, default=0) + 1, d, options["rope"], options.get("wide", False)) if "rope" in options else (None, None)
    smooth = None
    if "smooth" in options:
        smooth = torch.exp(0.5 * _randn(*((d,) if options["smooth"] == 1 else (h, d)), seed=seed + 2, dtype=torch.float32).clamp(-1, 1))
    offset = _randn(h, d, seed=seed + 3, dtype=torch.float32) if "offset" in options else None
    rotate = options.get("rotate", False)
    out = ops.hif4_kv_append(q, k, v, pool.pages, pool.table, pool.cu(new), _int32(*lens), page_size=pool.page_size, cos=cos,
                             sin=sin, q_norm=q_norm, k_norm=k_norm, eps=1e-5, rotate=rotate, smooth_scale=smooth,
                             key_offset=offset, **kw)
    pos = _pos(lens, new).clamp(min=0)
    n = len(pos)
    per_head = None if smooth is None else smooth.expand(h, d)
    kw = dict(eps=1e-5, cos=cos, sin=sin, rotate=rotate)
    want_q = ref.turned(q[:n], pos, norm=q_norm, smooth=None if smooth is None else per_head.repeat_interleave(heads // h, 0), **kw)
    want_k = ref.turned(k[:n], pos, norm=k_norm, offset=offset, smooth=per_head, divide=True, **kw)
    ratio = 1.0 if smooth is None else float(smooth.max() / smooth.min())
    return out, want_q, 2.0**-8 * want_q.abs() + 2.0**-18 * ratio * want_q.norm(dim=-1, keepdim=True) + 2.0**-126, want_k


@pytest.mark.parametrize("options", OPTIONS.values(), ids=OPTIONS.keys())
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("d", [64, 128])
def test_append_matches_fp64(d, dtype, options) -> None:
    lens, new, h, heads = [1, 40, 17, 0, 63, 200, 33], [1, 3, 17, 0, 1, 130, 0], 3, 15
    pool = Pool(lens, h, d, 32, DEV)
    before = pool.store.clone()
    n = sum(new)
    q, k, v = (_randn(n, x, d, seed=1 + i, dtype=dtype, scale=s) for i, (x, s) in enumerate(((heads, 1.0), (h, 3.0), (h, 0.1))))
    k[::7] *= 1e3
    out, want, bound, want_k = _append(pool, q, k, v, new, lens, options, levels=("123", "13"))
    assert out.dtype is torch.bfloat16 and bool(((out.double().cpu() - want).abs() <= bound).all())
    rk, rv = pool.read(new)
    assert torch.equal(rk.float().cpu(), quantized(want_k.float())) and torch.equal(rv.float().cpu(), quantized(v, "13"))
    assert int((pool.store != before).sum()) <= n * 2 * h * 37 * d // 64  # no other token's bytes
    _no_status()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_append_without_steps_is_a_write(dtype) -> None:
    lens = [70, 5]
    written, appended = (Pool(lens, 2, 128, 16, DEV) for _ in range(2))
    q, k, v = (_randn(75, x, 128, seed=4 + i, dtype=dtype) for i, x in enumerate((4, 2, 2)))
    written.write(k, v)
    out = _append(appended, q, k, v, lens, lens, {})[0]
    assert torch.equal(written.store, appended.store) and torch.equal(out, q.to(torch.bfloat16))


@pytest.mark.parametrize("d", [64, 128])
def test_a_keys_bits_do_not_depend_on_the_step(d) -> None:
    lens, options = [90], OPTIONS["deployed"]
    q, k, v = (_randn(90, x, d, seed=7 + i) for i, x in enumerate((2, 1, 1)))
    whole, steps = (Pool(lens, 1, d, 32, DEV) for _ in range(2))
    full = _append(whole, q, k, v, [90], [90], options)[0]
    # the same tables and weights: those of the last length
    from faquant_b200 import ops

    for begin, end in ((0, 1), (1, 18), (18, 19), (19, 90)):
        part = slice(begin, end)
        cos, sin = _tables(91, d, torch.bfloat16, True)
        norms = [(1 + 0.3 * torch.randn(d, generator=torch.Generator().manual_seed(90 + i))).to(DEV) for i in range(2)]
        smooth = torch.exp(0.5 * _randn(d, seed=92, dtype=torch.float32).clamp(-1, 1))
        out = ops.hif4_kv_append(q[part], k[part], v[part], steps.pages, steps.table, steps.cu([end - begin]), _int32(end),
                                 page_size=32, cos=cos, sin=sin, q_norm=norms[0], k_norm=norms[1], eps=1e-5, rotate=True,
                                 smooth_scale=smooth, key_offset=_randn(1, d, seed=93, dtype=torch.float32))
        assert torch.equal(out, full[part])
    assert torch.equal(whole.store, steps.store)


def test_append_strides_and_in_place() -> None:
    lens, h, heads, d = [21, 40], 2, 6, 128
    n = sum(lens)
    for shift in (0, 1):  # a fused projection, 16-byte aligned or not
        fused = _randn(n, (heads + 2 * h) * d + 8, seed=10)[:, shift:]
        parts = fused[:, : (heads + 2 * h) * d].unflatten(1, (heads + 2 * h, d))
        q, k, v = parts[:, :heads], parts[:, heads : heads + h], parts[:, heads + h :]
        dense, strided = (Pool(lens, h, d, 16, DEV) for _ in range(2))
        want = _append(dense, q.contiguous(), k.contiguous(), v.contiguous(), lens, lens, OPTIONS["qwen3"])[0]
        rest = parts[:, heads:].clone()
        out = _append(strided, q, k, v, lens, lens, OPTIONS["qwen3"], out=q)[0]
        assert out.data_ptr() == q.data_ptr() and torch.equal(out, want) and torch.equal(parts[:, heads:], rest)
        assert torch.equal(dense.store, strided.store)
    turned = _randn(d, heads, n, seed=11).permute(2, 1, 0)  # channels outermost
    pool = Pool(lens, h, d, 16, DEV)
    out, want, bound, _ = _append(pool, turned, turned[:, :h], turned[:, :h], lens, lens, OPTIONS["rope"],
                                  out=torch.empty(heads, n, d, dtype=torch.bfloat16, device=DEV).transpose(0, 1))
    assert bool(((out.double().cpu() - want).abs() <= bound).all())
    _no_status()


def test_append_tokens_without_a_place() -> None:
    from faquant_b200 import _lib, ops

    h, d = 1, 64
    pool = Pool([40, 20], h, d, 16, DEV)
    q, k, v = (_randn(14, x, d, seed=13 + i) for i, x in enumerate((2, 1, 1)))
    before = pool.store.clone()
    out = torch.full((14, 2, d), 7.0, dtype=torch.bfloat16, device=DEV)
    args = dict(page_size=16, rotate=True, out=out)
    # six new tokens of four, four of an idle sequence's none; four rows behind the batch
    ops.hif4_kv_append(q, k, v, pool.pages, pool.table, _int32(0, 6, 10), _int32(4, 0), **args)
    assert not out[:2].any() and bool(out[2:6].any(-1).all()) and not out[6:10].any() and bool((out[10:] == 7.0).all())
    pool.lens.copy_(_int32(4, 0))
    assert torch.equal(pool.read([4, 0])[0].float().cpu(), quantized(ref.hadamard(k[2:6].double().cpu()).float()))
    _no_status()
    # positions beyond the tables
    pool.store.copy_(before)
    cos, sin = _tables(18, d)
    out.fill_(7.0)
    ops.hif4_kv_append(q, k, v, pool.pages, pool.table, _int32(0, 14, 14), _int32(24, 0), cos=cos, sin=sin, page_size=16, out=out)
    assert _status() == _lib.FAQ_STATUS_BAD_BOUND
    assert bool(out[:8].any(-1).all()) and not out[8:].any()
    pool.lens.copy_(_int32(24, 0))
    rk, _ = pool.read([14, 0])
    want = ref.turned(k[:8], torch.arange(10, 18), cos=cos, sin=sin)
    assert torch.equal(rk[:8].float().cpu(), quantized(want.float()))
    assert int((pool.store != before).sum()) <= 8 * 2 * 37
    # a sequence beyond the rows given, one that falls; a page that is missing
    for bounds in ((0, 4, 15), (0, 4, 2)):
        pool.store.copy_(before)
        out.fill_(7.0)
        ops.hif4_kv_append(q, k, v, pool.pages, pool.table, _int32(*bounds), _int32(40, 20), **args)
        assert _status() == _lib.FAQ_STATUS_BAD_BOUND
        assert bool(out[:4].any(-1).all()) and bool((out[4:] == 7.0).all()) and int((pool.store != before).sum()) <= 4 * 2 * 37
    pool.table[0, 2] = -1
    pool.store.copy_(before)
    ops.hif4_kv_append(q, k, v, pool.pages, pool.table, _int32(0, 4, 14), _int32(40, 20), **args)
    assert _status() == _lib.FAQ_STATUS_BAD_PAGE and int((pool.store != before).sum()) <= 10 * 2 * 37


def test_append_not_a_number_stays_in_its_row() -> None:
    pools = [Pool([20], 2, 128, 16, DEV) for _ in range(2)]
    q, k, v = (_randn(20, x, 128, seed=16 + i) for i, x in enumerate((4, 2, 2)))
    good = _append(pools[0], q, k, v, [20], [20], OPTIONS["deployed"])[0]
    q[3, 1, 5], q[4, 0, 0], k[7, 1, 9] = math.nan, math.inf, math.nan
    out = _append(pools[1], q, k, v, [20], [20], OPTIONS["deployed"])[0]
    assert out[3, 1].isnan().all() and not out[4, 0].isfinite().any()
    out[3, 1], out[4, 0] = good[3, 1], good[4, 0]
    assert torch.equal(out, good)
    a, b = (p.read()[0] for p in pools)
    assert torch.equal(a[torch.arange(20) != 7], b[torch.arange(20) != 7]) and torch.equal(a[7, 0], b[7, 0])


def test_append_infinite_keys_scale_their_group() -> None:
    """Where no step mixes the channels, an infinite key divided by its smoothing is infinite, as it would
    be written without the step; its group of 64 channels takes the greatest scale, the others keep their bits."""
    from faquant_b200 import ops

    pools = [Pool([3], 2, 128, 16, DEV, fill=0) for _ in range(2)]
    q, k, v = (_randn(3, x, 128, seed=19 + i, dtype=torch.float32) for i, x in enumerate((2, 2, 2)))
    k[0, 0, 3], k[1, 1, 70], k[2, 0, 127] = math.inf, -math.inf, math.inf
    smooth = torch.full((128,), 2.0, device=DEV)  # the division is exact
    ops.hif4_kv_append(q, k, v, pools[0].pages, pools[0].table, pools[0].cu([3]), _int32(3), page_size=16, smooth_scale=smooth)
    ops.hif4_kv_write(k / 2, v, pools[1].pages, pools[1].table, pools[1].cu([3]), _int32(3), page_size=16)
    assert torch.equal(pools[0].store, pools[1].store)
    _no_status()


def test_steps_without_a_token_and_two_streams_at_once() -> None:
    from faquant_b200 import ops

    pools = [Pool([1500], 2, 128, 16, DEV, fill=0) for _ in range(2)]
    k, v, q = (_randn(1500, x, 128, seed=23 + i) for i, x in enumerate((2, 2, 8)))
    bounds = [_bounds(p) for p in pools]

    def step(pool, bounds, lens, new):
        args = (pool.table, pool.cu([new]), _int32(lens))
        part = slice(lens - new, lens)
        x = ops.hif4_kv_append(q[part], k[part], v[part], pool.pages, *args, page_size=16, rotate=True)
        ops.hif4_key_bounds(pool.pages, bounds, *args, page_size=16, total=new)
        lists = ops.hif4_select_pages(x, bounds, *args, page_size=16, count=9)
        return x, lists, ops.hif4_sparse_attention(x, pool.pages, *args, lists, page_size=16)

    before = [p.store.clone() for p in pools]
    x, lists, out = step(pools[0], bounds[0], 0, 0)
    assert x.shape == out.shape == (0, 8, 128) and lists.shape == (0, 2, 9) and torch.equal(pools[0].store, before[0])
    cuts = [(1200, 1200), (1203, 3), (1500, 297)]
    want = [step(pools[0], bounds[0], *c) for c in cuts]
    torch.cuda.synchronize()
    # the same on another stream, while this one repeats its last step
    other = torch.cuda.Stream(DEV)
    got = []
    for c in cuts:
        with torch.cuda.stream(other):
            got.append(step(pools[1], bounds[1], *c))
        again = step(pools[0], bounds[0], *cuts[-1])
        assert all(torch.equal(a, b) for a, b in zip(again, want[-1]))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))
    assert torch.equal(pools[0].store, pools[1].store) and torch.equal(bounds[0], bounds[1])
    _no_status()


# ------------------------------------------------------------------ bounds
def _refresh(pool, bounds, new=None, lens=None):
    from faquant_b200 import ops

    new = pool.lens_host if new is None else new
    lens = pool.lens if lens is None else _int32(*lens)
    ops.hif4_key_bounds(pool.pages, bounds, pool.table, pool.cu(new), lens, page_size=pool.page_size, total=sum(new))


def _check_bounds(pool, bounds, keys, lens):
    """Every page's bytes against the reference, from the packed keys of all tokens."""
    keys, d, table, at = quantized(keys), pool.d, pool.table.cpu(), 0
    got = bounds.cpu().view(torch.int8).double()
    for b, length in enumerate(lens):
        for c in range(-(-length // pool.page_size)):
            for j in range(pool.kv_heads):
                lo, hi, e = ref.page_bounds(keys[at + c * pool.page_size : at + min(length, (c + 1) * pool.page_size), j])
                row = got[table[b, c], j]
                assert torch.equal(row[:d], lo) and torch.equal(row[d : 2 * d], hi) and row[2 * d] == e and not row[2 * d + 1 :].any()
        at += length


@pytest.mark.parametrize("page", [16, 64, 512])
@pytest.mark.parametrize("d", [64, 128])
def test_bounds_of_pages(d, page) -> None:
    lens = [1, 16, 17, 0, 130, 700]
    pool = Pool(lens, 2, d, page, DEV, fill=0xFF)
    k = _randn(sum(lens), 2, d, seed=20)
    k[5:9] *= 1e6
    k[20:30] *= 1e-12
    k[0] = 0
    pool.write(k, k)
    bounds = _bounds(pool)
    _refresh(pool, bounds)
    _check_bounds(pool, bounds, k, lens)
    held = {int(x) for x in pool.table.flatten() if x >= 0}
    for other in set(range(pool.pages.shape[0])) - held:
        assert bool((bounds[other] == 0x5A).all())
    _no_status()


def test_bounds_follow_steps_and_forget_what_was_taken_back() -> None:
    pool = Pool([50, 20], 1, 128, 16, DEV)
    k = _randn(70, 1, 128, seed=21)
    k[18:30] *= 100.0  # drafts that will be rejected
    bounds = _bounds(pool)
    pool.write(k[:30], k[:30], new=[30, 0], lens=[30, 0])
    _refresh(pool, bounds, [30, 0], [30, 0])
    before = bounds.clone()
    again = _randn(2, 1, 128, seed=22)
    pool.write(again, again, new=[2, 0], lens=[20, 0])  # positions 18 and 19
    _refresh(pool, bounds, [2, 0], [20, 0])
    keys = torch.cat((k[:18], again))
    pool.lens_host = [20, 0]
    _check_bounds(pool, bounds, keys, [20, 0])
    first = pool.table[0, 0]
    assert torch.equal(bounds[first], before[first])
    # steps of one token end at the bounds of the whole
    for i in range(20, 50):
        pool.write(k[i : i + 1], k[i : i + 1], new=[1, 0], lens=[i + 1, 0])
        _refresh(pool, bounds, [1, 0], [i + 1, 0])
    _check_bounds(pool, bounds, torch.cat((keys, k[20:50])), [50, 0])
    _no_status()


# ------------------------------------------------------------------ selection
SELECTIONS = [  # heads, kv_heads, d, page, lens, new, count, first, last
    (4, 1, 128, 16, [1], [1], 1, 0, 1),
    (8, 2, 128, 16, [500, 17, 0, 90], [1, 3, 0, 1], 6, 1, 2),
    (32, 8, 128, 64, [3000], [1], 8, 1, 1),
    (6, 2, 64, 32, [700, 1, 64], [5, 1, 64], 4, 2, 2),
    (5, 1, 128, 16, [2000], [2], 100, 0, 3),
    (3, 3, 64, 16, [5000], [1], 300, 1, 1),
    (16, 1, 128, 128, [900, 128, 129], [1, 1, 2], 3, 1, 1),
    (2, 1, 64, 16, [300], [300], 7, 1, 2),
    (20, 2, 64, 16, [700, 90], [1, 2], 9, 1, 2),
    (128, 1, 128, 32, [1500], [2], 20, 1, 2),
    (2, 2, 128, 16, [20000], [2], 700, 2, 2),
    # many rows, one to eight tokens of a warp, at sequences' ends and starts
    (16, 2, 128, 16, [700, 30, 500, 3], [690, 3, 500, 3], 9, 1, 2),
    (50, 5, 64, 32, [330, 100], [300, 50], 4, 1, 1),
    (24, 8, 64, 16, [200, 150, 7], [150, 150, 7], 5, 2, 1),
    (16, 8, 64, 16, [9, 9, 9, 600, 20], [9, 1, 1, 570, 20], 6, 0, 1),
    (8, 8, 128, 16, [8, 1, 2, 1190, 5], [8, 1, 2, 1170, 5], 3, 1, 2),
    (40, 5, 64, 16, [17000], [300], 80, 1, 2),
]


@pytest.mark.parametrize("shape", SELECTIONS, ids=lambda s: f"h{s[0]}_{s[1]}_d{s[2]}_p{s[3]}_b{len(s[4])}_c{s[6]}")
def test_selection_matches_the_definition(shape) -> None:
    from faquant_b200 import ops

    heads, h, d, page, lens, new, count, first, last = shape
    pool = Pool(lens, h, d, page, DEV, fill=0xFF)
    k = _randn(sum(lens), h, d, seed=30)
    pool.write(k, k)
    bounds = _bounds(pool)
    _refresh(pool, bounds)
    q = _randn(sum(new) + 2, heads, d, seed=31, scale=2.0)  # two rows behind the batch
    out = torch.full((sum(new) + 2, h, count), -7, dtype=torch.int32, device=DEV)
    got, scores = ops.hif4_select_pages(q, bounds, pool.table, pool.cu(new), pool.lens, page_size=page, count=count,
                                        first=first, last=last, want_scores=True, out=out)
    n = sum(new)
    want, want_scores = ref.select(q[:n], k, lens, new, page, count, first, last)
    assert got.data_ptr() == out.data_ptr() and torch.equal(got[:n].cpu(), want)
    assert torch.equal(scores[:n].double().cpu(), want_scores) and bool((got[n:] == -7).all())
    assert torch.equal(ops.hif4_select_pages(q, bounds, pool.table, pool.cu(new), pool.lens, page_size=page, count=count,
                                             first=first, last=last)[:n], got[:n])
    _no_status()


def test_selection_of_strided_and_unaligned_operands() -> None:
    from faquant_b200 import ops

    lens, new = [300, 90, 1200], [1, 2, 1]
    pool = Pool(lens, 2, 64, 16, DEV)
    k = _randn(sum(lens), 2, 64, seed=41)
    pool.write(k, k)
    bounds = _bounds(pool)
    _refresh(pool, bounds)
    wide = _randn(4, 6 * 64 + 8, seed=42)[:, 3 : 3 + 6 * 64].unflatten(1, (6, 64))  # not 16-byte aligned
    turned = _randn(64, 6, 4, seed=43).permute(2, 1, 0)                            # channels outermost
    table = torch.full((3, pool.table.shape[1] + 5), -1, dtype=torch.int32, device=DEV)[:, 2:-3]
    table.copy_(pool.table)
    for q in (wide, turned):
        got = ops.hif4_select_pages(q, bounds, table, pool.cu(new), pool.lens, page_size=16, count=9)
        assert torch.equal(got.cpu(), ref.select(q, k, lens, new, 16, 9, 1, 2)[0])
        lists = torch.empty(4, 2, 12, dtype=torch.int32, device=DEV)[..., :9]
        lists.copy_(got)  # a list that is a slice
        out = ops.hif4_sparse_attention(q, pool.pages, table, pool.cu(new), pool.lens, lists, page_size=16)
        want, size = ref.attention(q, quantized(k), quantized(k), lens, new, 16, got.cpu())
        assert bool(((out.double().cpu() - want).abs() <= BOUND * size).all())
    _no_status()


def test_scores_bound_the_products() -> None:
    """A page's score is at least the product of the 8-bit query with every key of the page."""
    from faquant_b200 import ops

    pool = Pool([640], 1, 128, 64, DEV)
    k = _randn(640, 1, 128, seed=32)
    pool.write(k, k)
    bounds = _bounds(pool)
    _refresh(pool, bounds)
    q = _randn(1, 4, 128, seed=33)
    got, scores = ops.hif4_select_pages(q, bounds, pool.table, pool.cu([1]), pool.lens, page_size=64, count=10, want_scores=True)
    f = ref.exponent(float(q.abs().max()))
    rounded = torch.round(q[0].double().cpu() * 2.0**-f) * 2.0**f
    products = (rounded @ quantized(k)[:, 0].double().T).amax(0).reshape(10, 64).amax(1)
    assert got[0, 0].tolist() == list(range(10)) and bool((scores[0, 0].double().cpu() >= products).all())


def test_ties_missing_pages_and_what_is_not_finite() -> None:
    from faquant_b200 import _lib, ops

    lens, new, page, count = [640], [3], 16, 7
    pool = Pool(lens, 2, 64, page, DEV)
    k = _randn(16, 2, 64, seed=34).repeat(40, 1, 1)  # every full page alike
    pool.write(k, k)
    bounds = _bounds(pool)
    _refresh(pool, bounds)
    q = _randn(3, 4, 64, seed=35)
    args = (bounds, pool.table, pool.cu(new), pool.lens)
    kw = dict(page_size=page, count=count, first=1, last=2)
    assert ops.hif4_select_pages(q, *args, **kw)[2, 1].tolist() == [0, 1, 2, 3, 4, 38, 39]
    _no_status()
    missing = [(0, 0), (0, 2), (0, 38), (0, 20)]
    for b, c in missing:
        pool.table[b, c] = -1 if c else 10**6
    q[1, 0, 3], q[1, 1, 4], q[2, 2, 0] = math.nan, math.inf, -math.inf
    got, scores = ops.hif4_select_pages(q, *args, want_scores=True, **kw)
    want, want_scores = ref.select(q, k, lens, new, page, count, 1, 2, set(missing))
    assert torch.equal(got.cpu(), want) and torch.equal(scores.double().cpu(), want_scores)
    assert _status() == _lib.FAQ_STATUS_BAD_PAGE
    pool.table.fill_(-1)
    assert bool((ops.hif4_select_pages(q, *args, **kw) == -1).all()) and _status() == _lib.FAQ_STATUS_BAD_PAGE


@pytest.mark.parametrize("behind", [0, 3])
@pytest.mark.parametrize("heads, h, d", [(24, 12, 64), (99, 9, 128), (12, 12, 128)])
def test_many_rows_missing_pages_and_what_is_not_finite(heads, h, d, behind) -> None:
    """Tokens of one sequence taken together and others, pages that are not there, tokens below position zero."""
    from faquant_b200 import _lib, ops

    lens, new, count = [900, 50, 333], [200, 80, 70], 6
    pool = Pool(lens, h, d, 16, DEV)
    k = _randn(sum(lens), h, d, seed=44)
    pool.write(k, k)
    bounds = _bounds(pool)
    _refresh(pool, bounds)
    q = _randn(sum(new) + behind, heads, d, seed=45, scale=2.0)
    q[5, 0, 3], q[6, 1, 4], q[270, heads - 1, 0], q[340] = math.nan, math.inf, -math.inf, 0.0
    missing = [(0, 0), (0, 17), (0, 55), (1, 1), (2, 20)]
    for b, c in missing:
        pool.table[b, c] = -1 if c else 10**6
    out = torch.full((sum(new) + behind, h, count), -7, dtype=torch.int32, device=DEV)
    _, scores = ops.hif4_select_pages(q, bounds, pool.table, pool.cu(new), pool.lens, page_size=16, count=count, want_scores=True,
                                      out=out)
    n = sum(new)
    want, want_scores = ref.select(q[:n], k, lens, new, 16, count, 1, 2, set(missing))
    assert torch.equal(out[:n].cpu(), want) and torch.equal(scores[:n].double().cpu(), want_scores) and bool((out[n:] == -7).all())
    assert _status() == _lib.FAQ_STATUS_BAD_PAGE


def test_selection_of_tokens_without_a_place_and_bad_batches() -> None:
    from faquant_b200 import _lib, ops

    pool = Pool([100, 100], 1, 64, 16, DEV)
    k = _randn(200, 1, 64, seed=36)
    pool.write(k, k)
    bounds = _bounds(pool)
    _refresh(pool, bounds)
    q = _randn(8, 2, 64, seed=37)
    kw = dict(page_size=16, count=3)
    got = ops.hif4_select_pages(q, bounds, pool.table, _int32(0, 4, 8), _int32(2, 0), **kw)
    assert got[:, 0].tolist() == [[-1, -1, -1]] * 2 + [[0, -1, -1]] * 2 + [[-1, -1, -1]] * 4
    _no_status()
    for bounds_of in ((0, 4, 9), (0, 4, 2), (0, 8, 7)):
        out = torch.full((8, 1, 3), -7, dtype=torch.int32, device=DEV)
        ops.hif4_select_pages(q, bounds, pool.table, _int32(*bounds_of), pool.lens, out=out, **kw)
        assert _status() == _lib.FAQ_STATUS_BAD_BOUND
        n = bounds_of[1]
        assert bool((out[:n] >= 0).all()) and bool((out[n:] == -7).all())


def test_selection_among_the_most_columns() -> None:
    from faquant_b200 import ops

    columns, page = 32768, 16
    pages = torch.zeros(columns, ops.hif4_page_bytes(1, 64, page), dtype=torch.uint8, device=DEV)
    table = torch.randperm(columns, generator=torch.Generator().manual_seed(38)).to(torch.int32)[None].to(DEV)
    lens, cu = _int32(columns * page), _int32(0, columns * page)
    k = torch.randn(columns * page, 1, 64, generator=torch.Generator(DEV).manual_seed(39), device=DEV).to(torch.bfloat16)
    ops.hif4_kv_write(k, k, pages, table, cu, lens, page_size=page)
    bounds = torch.zeros(columns, 1, ops.hif4_bounds_bytes(64), dtype=torch.uint8, device=DEV)
    ops.hif4_key_bounds(pages, bounds, table, cu, lens, page_size=page, total=columns * page)
    q = _randn(1, 128, 64, seed=40)
    got, scores = ops.hif4_select_pages(q, bounds, table, _int32(0, 1), lens, page_size=page, count=500, first=3, last=4,
                                        want_scores=True)
    rows = bounds[table[0].long(), 0].view(torch.int8).double()
    f = ref.exponent(float(q.abs().max()))
    q8 = torch.round(q[0].double() * 2.0**-f)
    every = (q8.clamp(min=0) @ rows[:, 64:128].T + q8.clamp(max=0) @ rows[:, :64].T).amax(0) * torch.exp2(rows[:, 128])
    ranked = every.clone()
    ranked[:3] = ranked[-4:] = math.inf
    want = torch.sort(ranked, dim=0, descending=True, stable=True).indices[:500].sort().values
    assert torch.equal(got[0, 0].long(), want) and torch.equal(scores[0, 0].double(), every[want] * 2.0**f)
    _no_status()


# ------------------------------------------------------------------ attention
def _lists(lens, new, h, page, count, seed):
    """Random columns per token and kv head: in any order, some twice, some behind the token, some -1."""
    g = torch.Generator().manual_seed(seed)
    out = torch.full((sum(new), h, count), -1, dtype=torch.int32)
    for t, (_, pos) in enumerate(ref.positions(lens, new)):
        for j in range(h):
            columns = max(pos, 0) // page + 1
            row = torch.randperm(columns + 2, generator=g)[:count].to(torch.int32)  # up to two behind the token
            row[torch.rand(len(row), generator=g) < 0.2] = -1
            if len(row) > 3 and j % 2:
                row[3] = row[1]  # twice
            at = torch.randperm(count, generator=g)[: len(row)]
            out[t, j, at] = row
    return out


def _attend(pool, q, new, selected, lens=None, **kw):
    from faquant_b200 import ops

    return ops.hif4_sparse_attention(q, pool.pages, pool.table, pool.cu(new), pool.lens if lens is None else _int32(*lens),
                                     selected.to(DEV), page_size=pool.page_size, **kw)


SHAPES = [  # heads, kv_heads, d, page, lens, new, count
    (4, 1, 128, 16, [1], [1], 1),
    (8, 2, 128, 16, [1, 2, 15, 16, 17, 127, 129, 500], [1] * 8, 9),
    (32, 8, 128, 64, [3000], [1], 16),
    (5, 1, 128, 32, [100, 31], [1, 3], 2),
    (2, 2, 64, 128, [40, 700, 0, 3], [1, 8, 0, 3], 4),
    (16, 4, 64, 32, [5, 70, 64, 900], [5, 0, 8, 100], 12),
    (9, 1, 128, 16, [300], [2], 7),
    (24, 1, 64, 16, [90], [3], 5),
    (128, 1, 128, 64, [1300], [3], 8),
    (8, 1, 128, 256, [2000], [40], 3),
    (16, 8, 128, 16, [600], [300], 6),
    (7, 7, 64, 4096, [5000], [1], 2),
    (1, 1, 128, 16, [4000], [1], 250),
    (33, 1, 64, 32, [200], [20], 3),
    (100, 1, 128, 16, [150], [9], 5),
    (8, 1, 128, 16, [3500], [16], 100),
    # more units than the SMs hold at once
    (16, 8, 64, 16, [50 + 37 * i for i in range(60)], [1] * 60, 12),
    (20, 4, 128, 32, [90 + 31 * i for i in range(40)], [3] * 40, 5),
    (16, 16, 128, 64, [4 + 19 * i for i in range(33)], [0, 1, 2] * 11, 4),
    # enough of them to be taken together: tiles of one to 32 tokens, all ratios of heads, one CTA or a cluster
    (8, 8, 128, 16, [700], [200], 41),
    (6, 2, 64, 64, [900, 5, 300], [400, 5, 200], 27),
    (20, 4, 128, 32, [2000, 100], [180, 60], 36),
    (132, 4, 64, 32, [400], [150], 13),
    (100, 1, 128, 16, [600], [150], 38),
    (64, 8, 128, 64, [1500], [130], 16),
    (8, 1, 64, 4096, [9000], [100], 3),
    (16, 2, 128, 16, [400] * 10, [200] * 10, 17),
    (8, 1, 128, 1024, [33000], [32], 32),
    (4, 4, 64, 32, [3000, 2, 700], [150, 2, 1], 60),
    (128, 1, 128, 64, [1300], [60], 21),
    (16, 16, 64, 16, [460], [460], 9),
]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"h{s[0]}_{s[1]}_d{s[2]}_p{s[3]}_b{len(s[4])}_n{max(s[5])}_c{s[6]}")
def test_attention_over_listed_pages_matches_fp64(shape) -> None:
    heads, h, d, page, lens, new, count = shape
    pool = Pool(lens, h, d, page, DEV, fill=0xFF)
    k, v = _randn(sum(lens), h, d, seed=50), _randn(sum(lens), h, d, seed=51, scale=0.5)
    pool.write(k, v)
    q = _randn(sum(new), heads, d, seed=52, scale=2.0)
    lists = _lists(lens, new, h, page, count, 53)
    out = _attend(pool, q, new, lists)
    want, size = ref.attention(q, quantized(k), quantized(v), lens, new, page, lists)
    assert out.shape == q.shape and bool(((out.double().cpu() - want).abs() <= BOUND * size + 2.0**-126).all())
    # the same bits again, and on strided q and out
    wide = torch.zeros(heads, sum(new), d + 8, dtype=torch.bfloat16, device=DEV).transpose(0, 1)
    wide[..., :d] = q
    into = torch.empty_like(wide)[..., :d]
    assert torch.equal(_attend(pool, wide[..., :d], new, lists, out=into), out)
    # columns beyond the table set the status, others do not
    assert _status() in (0, 2)


@pytest.mark.parametrize("heads", [4, 9])
def test_long_lists_in_any_order(heads) -> None:
    """Entries that repeat an earlier one far before them are dropped: the list once through, in its order."""
    pool = Pool([9000], 1, 128, 16, DEV, fill=0xFF)
    k, v = _randn(9000, 1, 128, seed=61), _randn(9000, 1, 128, seed=62, scale=0.5)
    pool.write(k, v)
    q = _randn(1, heads, 128, seed=63, scale=2.0)
    g = torch.Generator().manual_seed(64)
    once = torch.randperm(563, generator=g)[:400]
    lists = torch.cat((once, once[torch.randint(400, (900,), generator=g)]))[torch.randperm(1300, generator=g)].to(torch.int32)
    want, size = ref.attention(q, quantized(k), quantized(v), [9000], [1], 16, lists.reshape(1, 1, -1))
    out = _attend(pool, q, [1], lists.reshape(1, 1, -1))
    assert bool(((out.double().cpu() - want).abs() <= BOUND * size + 2.0**-126).all())
    _no_status()


@pytest.mark.parametrize("n", [1, 5, 90, 300])
def test_every_page_listed_is_the_dense_attention(n) -> None:
    lens, page = [1000, 300], 32
    pool = Pool(lens, 2, 128, page, DEV)
    k, v = _randn(1300, 2, 128, seed=54), _randn(1300, 2, 128, seed=55)
    pool.write(k, v)
    q = _randn(2 * n, 8, 128, seed=56, scale=2.0)
    lists = torch.arange(33, dtype=torch.int32).expand(2 * n, 2, 33)  # up to one behind the table
    dense, sparse = pool.attend(q, [n, n]), _attend(pool, q, [n, n], lists)
    _, size = ref.attention(q, quantized(k), quantized(v), lens, [n, n], page, lists)
    assert bool(((dense - sparse).double().abs().cpu() <= 2 * BOUND * size).all())
    _no_status()


@pytest.mark.parametrize("heads", [3, 17])
def test_rows_without_a_key_and_rows_left_alone(heads) -> None:
    from faquant_b200 import _lib

    pool = Pool([4, 30], 1, 64, 16, DEV)
    k = _randn(34, 1, 64, seed=57)
    pool.write(k, k)
    q = _randn(12, heads, 64, seed=58)
    lists = torch.zeros(12, 1, 2, dtype=torch.int32)
    lists[:, :, 1] = -5
    lists[8] = -1      # a token without a list
    lists[9, 0, 0] = 1  # a page behind the token
    out = torch.full_like(q, 7.0)
    _attend(pool, q, [6, 4], lists, lens=[4, 12], out=out)
    want, size = ref.attention(q[:10], quantized(k[:16]), quantized(k[:16]), [4, 12], [6, 4], 16, lists)
    assert not out[:2].any() and not out[8:10].any() and bool((out[10:] == 7.0).all())
    assert bool(((out[:10].double().cpu() - want).abs() <= BOUND * size + 2.0**-126).all())
    _no_status()
    for bounds in ((0, 6, 13), (0, 6, 5), (0, 12, 7)):
        out = torch.full_like(q, 7.0)
        from faquant_b200 import ops

        ops.hif4_sparse_attention(q, pool.pages, pool.table, _int32(*bounds), pool.lens, lists.to(DEV), page_size=16, out=out)
        assert _status() == _lib.FAQ_STATUS_BAD_BOUND
        assert bool((out[bounds[1] :] == 7.0).all()) and not bool((out[: bounds[1]] == 7.0).any())
    # a page that is missing is left out and reported
    pool.table[1, 0] = 10**6
    lists = torch.tensor([0, 1], dtype=torch.int32).expand(12, 1, 2)
    out = _attend(pool, q, [0, 12], lists)
    want, size = ref.attention(q, quantized(k), quantized(k), [4, 30], [0, 12], 16, lists, missing={(1, 0)})
    assert _status() == _lib.FAQ_STATUS_BAD_PAGE and bool(((out.double().cpu() - want).abs() <= BOUND * size + 2.0**-126).all())


def test_tiles_of_rows_without_a_key_and_rows_left_alone() -> None:
    from faquant_b200 import _lib, ops

    lens, new, count = [100, 900], [300, 400], 50
    pool = Pool(lens, 2, 64, 16, DEV)
    k, v = _randn(1000, 2, 64, seed=65), _randn(1000, 2, 64, seed=66)
    pool.write(k, v)
    q = _randn(720, 8, 64, seed=67)
    lists = torch.full((720, 2, count), -1, dtype=torch.int32)
    lists[:700] = _lists(lens, new, 2, 16, count, 68)
    lists[300:310] = -1  # tokens without a list
    args = (pool.pages, pool.table)
    kw = dict(page_size=16)
    out = torch.full_like(q, 7.0)
    ops.hif4_sparse_attention(q, *args, pool.cu(new), pool.lens, lists.to(DEV), out=out, **kw)
    want, size = ref.attention(q[:700], quantized(k), quantized(v), lens, new, 16, lists)
    assert not out[:200].any() and not out[300:310].any() and bool((out[700:] == 7.0).all())
    assert bool(((out[:700].double().cpu() - want).abs() <= BOUND * size + 2.0**-126).all())
    _status()
    for bounds in ((0, 300, 721), (0, 300, 299)):
        out = torch.full_like(q, 7.0)
        ops.hif4_sparse_attention(q, *args, _int32(*bounds), pool.lens, lists.to(DEV), out=out, **kw)
        assert _status() == _lib.FAQ_STATUS_BAD_BOUND and bool((out[300:] == 7.0).all())
        assert bool(((out[:300].double().cpu() - want[:300]).abs() <= BOUND * size[:300] + 2.0**-126).all())
    pool.table[1, 2], pool.table[1, 40] = -1, 10**6
    out = ops.hif4_sparse_attention(q, *args, pool.cu(new), pool.lens, lists.to(DEV), **kw)
    want, size = ref.attention(q[:700], quantized(k), quantized(v), lens, new, 16, lists, missing={(1, 2), (1, 40)})
    assert _status() == _lib.FAQ_STATUS_BAD_PAGE
    assert bool(((out[:700].double().cpu() - want).abs() <= BOUND * size + 2.0**-126).all())


@pytest.mark.parametrize("n, length", [(6, 900), (530, 2000)])
def test_peaked_scores_ranges_and_not_a_number(n, length) -> None:
    lens, new, page = [length], [n], 16
    pool = Pool(lens, 1, 128, page, DEV)
    k, v = _randn(length, 1, 128, seed=59), _randn(length, 1, 128, seed=60)
    k[700] *= 30.0  # one key far above the others, found late
    v[3] *= 1e6     # and a value row of another magnitude
    v[600:] *= 1e-20
    pool.write(k, v)
    q = _randn(n, 4, 128, seed=61)
    q[1] = 0
    pages = -(-length // page)
    lists = torch.arange(pages, dtype=torch.int32).expand(n, 1, pages)
    for scale in (None, 0.002, 0.5):
        out = _attend(pool, q, new, lists, scale=scale)
        want, size = ref.attention(q, quantized(k), quantized(v), lens, new, page, lists, scale)
        assert bool(((out.double().cpu() - want).abs() <= BOUND * size + 2.0**-126).all())
    good = _attend(pool, q, new, lists)
    q[2, 1, 17], q[4, 0, 0] = math.nan, math.inf
    out = _attend(pool, q, new, lists)
    assert out[2, 1].isnan().all() and out[4, 0].isnan().any()
    out[2, 1], out[4, 0] = good[2, 1], good[4, 0]
    assert torch.equal(out, good)


def test_offsets_past_32_bits() -> None:
    from faquant_b200 import ops

    size = ops.hif4_page_bytes(8, 128, 1024)
    count = (1 << 32) // size + 4
    pages = torch.empty(count, size, dtype=torch.uint8, device=DEV)
    far = (1 << 31) // size + 1
    table = torch.tensor([[far, count - 1], [count - 2, 0]], dtype=torch.int32, device=DEV)
    lens, cu = _int32(1050, 33), _int32(0, 1050, 1083)
    q, k, v = (_randn(1083, x, 128, seed=62 + i) for i, x in enumerate((16, 8, 8)))
    turned = ops.hif4_kv_append(q, k, v, pages, table, cu, lens, page_size=1024)
    rk, rv = ops.hif4_kv_read(pages, table, cu, lens, page_size=1024, head_dim=128, total=1083)
    assert torch.equal(rk.float().cpu(), quantized(k)) and torch.equal(rv.float().cpu(), quantized(v))
    bounds = torch.zeros(count, 8, ops.hif4_bounds_bytes(128), dtype=torch.uint8, device=DEV)
    ops.hif4_key_bounds(pages, bounds, table, cu, lens, page_size=1024, total=1083)
    one = _int32(0, 1, 2)
    last = turned[[1049, 1082]]
    lists = ops.hif4_select_pages(last, bounds, table, one, lens, page_size=1024, count=2, first=0, last=1)
    assert lists[0].tolist() == [[0, 1]] * 8 and lists[1].tolist() == [[0, -1]] * 8
    out = ops.hif4_sparse_attention(last, pages, table, one, lens, lists, page_size=1024)
    want, size = ref.attention(last, quantized(k), quantized(v), [1050, 33], [1, 1], 1024, lists.cpu())
    assert bool(((out.double().cpu() - want).abs() <= BOUND * size).all())
    _no_status()


# ------------------------------------------------------------------ a step of all of them
def _step(pool, bounds, q, k, v, cu, lens, total, count, cos, sin, norms):
    from faquant_b200 import ops

    batch = (pool.table, cu, lens)
    turned = ops.hif4_kv_append(q, k, v, pool.pages, *batch, page_size=pool.page_size, cos=cos, sin=sin, q_norm=norms[0],
                                k_norm=norms[1])
    ops.hif4_key_bounds(pool.pages, bounds, *batch, page_size=pool.page_size, total=total)
    lists = ops.hif4_select_pages(turned, bounds, *batch, page_size=pool.page_size, count=count)
    return turned, lists, ops.hif4_sparse_attention(turned, pool.pages, *batch, lists, page_size=pool.page_size)


def _steps(d=128, h=2, heads=8, page=16, count=5):
    """A prompt, a step of drafts, a step of one: inputs and the reference's answers."""
    steps = [([200, 31], [200, 31]), ([204, 32], [4, 1]), ([205, 33], [1, 1])]
    pool = Pool([205, 33], h, d, page, DEV)
    cos, sin = _tables(300, d)
    norms = [(1 + 0.2 * _randn(d, seed=70 + i, dtype=torch.float32)).to(torch.bfloat16) for i in range(2)]
    inputs, want = [], []
    keys = values = [torch.zeros(0, h, d, dtype=torch.float64)] * 2
    for i, (lens, new) in enumerate(steps):
        q, k, v = (_randn(sum(new), x, d, seed=72 + 3 * i + j) for j, x in enumerate((heads, h, h)))
        inputs.append((q, k, v, lens, new))
        fresh = ref.turned(k, _pos(lens, new), norm=norms[1], cos=cos, sin=sin).float()
        keys = [torch.cat((a, b)) for a, b in zip(keys, fresh.split(new))]
        values = [torch.cat((a, b)) for a, b in zip(values, v.cpu().split(new))]
        want.append((torch.cat(keys), torch.cat(values)))
    return pool, inputs, want, cos, sin, norms, count


def _check_step(got, inputs, want, page, count):
    turned, lists, out = got
    _, _, _, lens, new = inputs
    want_lists, _ = ref.select(turned, want[0], lens, new, page, count, 1, 2)
    assert torch.equal(lists.cpu(), want_lists)
    value, size = ref.attention(turned, quantized(want[0]), quantized(want[1]), lens, new, page, want_lists)
    assert bool(((out.double().cpu() - value).abs() <= BOUND * size + 2.0**-126).all())


def test_steps_of_a_batch_on_another_stream() -> None:
    pool, inputs, want, cos, sin, norms, count = _steps()
    bounds = _bounds(pool)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    got = []
    with torch.cuda.stream(stream):
        for q, k, v, lens, new in inputs:
            got.append(_step(pool, bounds, q, k, v, pool.cu(new), _int32(*lens), sum(new), count, cos, sin, norms))
    torch.cuda.current_stream().wait_stream(stream)
    for g, i, w in zip(got, inputs, want):
        _check_step(g, i, w, pool.page_size, count)
    _no_status()


def test_two_graphs_of_a_step_replayed_in_turn() -> None:
    """Decode steps captured once per buffer set and replayed as the lengths grow."""
    pool, inputs, want, cos, sin, norms, count = _steps()
    bounds = _bounds(pool)
    q, k, v, lens, new = inputs[0]
    _step(pool, bounds, q, k, v, pool.cu(new), _int32(*lens), sum(new), count, cos, sin, norms)
    graphs = []
    for q, k, v, lens, new in inputs[1:]:
        held = dict(q=torch.zeros_like(q), k=torch.zeros_like(k), v=torch.zeros_like(v), cu=pool.cu(new), lens=_int32(0, 0))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        keep = pool.store.clone(), bounds.clone()
        with torch.cuda.stream(side):  # warm-up
            _step(pool, bounds, *held.values(), sum(new), count, cos, sin, norms)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _step(pool, bounds, *held.values(), sum(new), count, cos, sin, norms)
        pool.store.copy_(keep[0])
        bounds.copy_(keep[1])
        graphs.append((graph, held, out))
    for _ in range(2):  # the second time over the same positions: the same answers
        for (graph, held, out), (q, k, v, lens, new), w in zip(graphs, inputs[1:], want[1:]):
            for name, x in (("q", q), ("k", k), ("v", v), ("lens", _int32(*lens))):
                held[name].copy_(x)
            graph.replay()
            torch.cuda.synchronize()
            _check_step(out, (q, k, v, lens, new), w, pool.page_size, count)
    _no_status()
