"""The paged operators at the ends of their arguments' ranges: keys near the largest and the smallest numbers, lists in
any order with many entries, tables and unions as large as the kernels of tiles take. Against 64-bit references."""

from __future__ import annotations

import pytest
import torch

import sparse_reference as ref
from paged_reference import Pool, quantized
from test_gpu_sparse import DEV, _int32, _no_status, _pos, _randn, _status, _tables

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ append
@pytest.mark.parametrize("power, low", [(126, 0), (-126, -20)], ids=["largest", "smallest"])
@pytest.mark.parametrize("rotate", [False, True])
@pytest.mark.parametrize("d", [64, 128])
def test_append_of_keys_at_the_ends_of_the_range(d, rotate, power, low) -> None:
    """Keys whose products with the norm's weights leave fp32's range: the norm brings them back into it."""
    from faquant_b200 import ops

    lens, h = [37], 2
    pool = Pool(lens, h, d, 16, DEV)
    q, v = _randn(37, 4, d, seed=101), _randn(37, h, d, seed=102)
    k = _randn(37, h, d, seed=103, dtype=torch.float32).clamp(-3.5, 3.5)
    k[::2] *= 2.0**power
    k = k.to(torch.bfloat16)
    norm = (torch.exp2(torch.linspace(low, low + 6, d)) * 1.1).to(torch.bfloat16).to(DEV)
    cos, sin = _tables(40, d)
    ops.hif4_kv_append(q, k, v, pool.pages, pool.table, pool.cu(lens), pool.lens, page_size=16, cos=cos, sin=sin, k_norm=norm,
                       eps=0.0, rotate=rotate)
    want = ref.turned(k, _pos(lens, lens), norm=norm, eps=0.0, cos=cos, sin=sin, rotate=rotate).float()
    assert bool(want.isfinite().all()) and torch.equal(pool.read()[0].float().cpu(), quantized(want))
    _no_status()


# ------------------------------------------------------------------ lists in any order
BOUND = 2.0**-8 + 2.0**-8 + 2.0**-12  # of test_gpu_sparse.py


def _microseconds(call):
    times = []
    for _ in range(6):
        begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        begin.record()
        call()
        end.record()
        torch.cuda.synchronize()
        times.append(1e3 * begin.elapsed_time(end))
    return min(times)


def test_a_long_list_in_any_order_costs_about_what_an_ascending_one_does() -> None:
    """Most entries lie behind the token, as a list of fixed size for a short context has them."""
    from faquant_b200 import ops

    page, count = 512, 8192
    pool = Pool([2100], 1, 64, page, DEV)
    k, v = _randn(2100, 1, 64, seed=110), _randn(2100, 1, 64, seed=111)
    pool.write(k, v)
    q = _randn(1, 4, 64, seed=112)
    order = torch.randperm(count, generator=torch.Generator().manual_seed(113)).to(torch.int32)
    order[order > 8000] = 3  # some of them again
    times = []
    for lists in (torch.arange(count, dtype=torch.int32), order):
        lists = lists.reshape(1, 1, -1).to(DEV)

        def call():
            return ops.hif4_sparse_attention(q, pool.pages, pool.table, pool.cu([1]), pool.lens, lists, page_size=page)

        want, size = ref.attention(q, quantized(k), quantized(v), [2100], [1], page, lists.cpu())
        assert bool(((call().double().cpu() - want).abs() <= BOUND * size + 2.0**-126).all())
        times.append(_microseconds(call))
    assert times[1] < 4 * times[0], times
    _no_status()


@pytest.mark.parametrize("heads, h, d, tokens", [(8, 1, 128, 1), (2, 2, 64, 3), (8, 8, 64, 70)])
def test_repeated_columns_of_a_context_of_many(heads, h, d, tokens) -> None:
    """Columns far apart (more than 131072 of them), holes and repeats at any distance; a page may stand in several columns."""
    from faquant_b200 import ops

    columns, page, held = 270001, 16, 50
    pool = Pool([held * page], h, d, page, DEV, fill=0xFF)
    k, v = _randn(held * page, h, d, seed=114), _randn(held * page, h, d, seed=115, scale=0.5)
    pool.write(k, v)
    k, v = (quantized(x).double().reshape(held, page, h, d) for x in (k, v))
    g = torch.Generator().manual_seed(116)
    at = torch.randint(held, (columns,), generator=g)
    table = pool.table[0][at.to(DEV)][None].contiguous()
    lens, cu = _int32(columns * page), _int32(0, tokens)
    q = _randn(tokens, heads, d, seed=117, scale=2.0)
    once = torch.cat((torch.randint(columns - tokens // page - 1, (150,), generator=g), torch.tensor([0, 31, 32, 131071, 131072, 262144])))
    lists = torch.full((tokens, h, 700), -1, dtype=torch.int32)
    for row in lists.view(-1, 700):
        row[:500] = once[torch.randint(len(once), (500,), generator=g)].to(torch.int32)
        row[:] = row[torch.randperm(700, generator=g)]
    out = ops.hif4_sparse_attention(q, pool.pages, table, cu, lens, lists.to(DEV), page_size=page)
    _check(out, q, k, v, at, lists)
    _no_status()


def _check(out, q, k, v, at, lists):
    """Of whole pages, all visible: ``k``, ``v`` fp64 ``[pages, page, H, D]``, ``at`` the page of each column."""
    out, q, (h, d) = out.double().cpu(), q.double().cpu(), k.shape[2:]
    for t in range(q.shape[0]):
        for j, heads in enumerate(torch.arange(q.shape[1]).chunk(h)):
            mine = at[torch.tensor(sorted(set(lists[t, j].tolist()) - {-1}))]
            keys, values = (x[mine, :, j].reshape(-1, d) for x in (k, v))
            p = torch.softmax(q[t, heads] @ keys.T * d**-0.5, -1)
            assert bool(((out[t, heads] - p @ values).abs() <= BOUND * (p @ values.abs()) + 2.0**-126).all())


# ------------------------------------------------------------------ both kernels at their ends
def _tokens_of_tiles(h, blocks):
    """New tokens of a call that the kernel of tiles takes for certain: half as many again as its rule asks for."""
    sms = torch.cuda.get_device_properties(DEV).multi_processor_count
    return -(-3 * 440 * sms // (2 * h * blocks))


@pytest.mark.parametrize("heads, h, d, columns, apart", [
    (8, 2, 64, 1875, True),     # a tile's union holds the most columns that there may be
    (8, 2, 64, 1875, False),    # more columns than a tile has threads
    (12, 4, 64, 16384, False),  # the most columns whose marks fit
    (12, 4, 64, 16385, False),  # and one more, which single tokens take
    (10, 2, 128, 32768, False),
    (10, 2, 128, 32769, False),
])
def test_tiles_among_many_columns(heads, h, d, columns, apart) -> None:
    from faquant_b200 import ops

    page, held = 16, 40
    tile = min(32, 128 // (heads // h))
    count = 1536 // tile
    tokens = _tokens_of_tiles(h, count)
    pool = Pool([held * page], h, d, page, DEV, fill=0xFF)
    k, v = _randn(held * page, h, d, seed=120), _randn(held * page, h, d, seed=121, scale=0.5)
    pool.write(k, v)
    k, v = (quantized(x).double().reshape(held, page, h, d) for x in (k, v))
    g = torch.Generator().manual_seed(122)
    at = torch.randint(held, (columns,), generator=g)
    table = pool.table[0][at.to(DEV)][None].contiguous()
    seen = columns - -(-tokens // page)
    q = _randn(tokens, heads, d, seed=123, scale=2.0)
    if apart:
        order = torch.stack([torch.randperm(seen, generator=g)[:1536] for _ in range(-(-tokens // tile) * h)])
        lists = order.reshape(-1, h, tile, count).transpose(1, 2).reshape(-1, h, count)[:tokens]
    else:
        lists = torch.randint(seen, (tokens, h, count), generator=g)
        lists[:, :, 0], lists[:, :, 1] = 0, seen - 1
    lists = lists.to(torch.int32).contiguous()
    out = ops.hif4_sparse_attention(q, pool.pages, table, _int32(0, tokens), _int32(columns * page), lists.to(DEV), page_size=page)
    _check(out, q, k, v, at, lists)
    _no_status()


@pytest.mark.parametrize("tiles", [False, True])
def test_columns_behind_the_token_set_no_status_and_those_beyond_the_table_do(tiles) -> None:
    from faquant_b200 import _lib, ops

    heads, h, d, page, count = 8, 2, 128, 64, 24
    tokens = _tokens_of_tiles(h, count * page // 16) if tiles else 5
    length = 60 * page
    pool = Pool([length], h, d, page, DEV, fill=0xFF)  # a table of 61 columns, the last one without a page
    k, v = _randn(length, h, d, seed=124), _randn(length, h, d, seed=125)
    pool.write(k, v)
    q = _randn(tokens, heads, d, seed=126, scale=2.0)
    g = torch.Generator().manual_seed(127)
    lists = torch.stack([torch.randperm(90, generator=g)[:count] for _ in range(tokens * h)]).reshape(tokens, h, count).to(torch.int32)
    args = (pool.pages, pool.table, pool.cu([tokens]))
    # all of a column's tokens behind the queries, or no column at all
    out = ops.hif4_sparse_attention(q, *args, pool.lens, lists.to(DEV), page_size=page)
    want, size = ref.attention(q, quantized(k), quantized(v), [length], [tokens], page, lists)
    assert bool(((out.double().cpu() - want).abs() <= BOUND * size + 2.0**-126).all())
    _no_status()
    # a sequence that is longer than its row of the table: columns that the tokens see, and no page for them
    longer = length + 12 * page + tokens
    out = ops.hif4_sparse_attention(q, *args, _int32(longer), lists.to(DEV), page_size=page)
    assert _status() == _lib.FAQ_STATUS_BAD_PAGE
    want, size = ref.attention(q, quantized(k), quantized(v), [longer], [tokens], page, lists, missing={(0, c) for c in range(60, 90)})
    assert bool(((out.double().cpu() - want).abs() <= BOUND * size + 2.0**-126).all())


@pytest.mark.parametrize("heads, h, d, lens, new", [(32, 8, 128, [3000], [700]), (8, 8, 64, [2000, 900], [400, 500]), (8, 2, 128, [700], [3])])
def test_selection_with_a_table_far_wider_than_the_lengths(heads, h, d, lens, new) -> None:
    """The kernel and its split are chosen by the table's columns; the lists are the same."""
    from faquant_b200 import ops

    pool = Pool(lens, h, d, 16, DEV)
    k = _randn(sum(lens), h, d, seed=130)
    pool.write(k, k)
    bounds = torch.zeros(pool.pages.shape[0], h, ops.hif4_bounds_bytes(d), dtype=torch.uint8, device=DEV)
    wide = torch.full((len(lens), 8192), -1, dtype=torch.int32, device=DEV)
    wide[:, : pool.table.shape[1]] = pool.table
    ops.hif4_key_bounds(pool.pages, bounds, wide, pool.cu(lens), pool.lens, page_size=16, total=sum(lens))
    q = _randn(sum(new), heads, d, seed=131)
    lists = [ops.hif4_select_pages(q, bounds, table, pool.cu(new), pool.lens, page_size=16, count=20, want_scores=True)
             for table in (pool.table, wide, wide[:, : pool.table.shape[1]])]
    for other in lists[1:]:
        assert all(torch.equal(a, b) for a, b in zip(lists[0], other))
    out = [ops.hif4_sparse_attention(q, pool.pages, table, pool.cu(new), pool.lens, lists[0][0], page_size=16)
           for table in (pool.table, wide)]
    assert torch.equal(*out)
    _no_status()
