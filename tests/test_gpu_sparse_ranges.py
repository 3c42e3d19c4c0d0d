"""The paged operators at the ends of their arguments' ranges: keys near the largest and the smallest numbers, lists in
any order with many entries, tables and unions as large as the kernels of tiles take. Against 64-bit references."""

from __future__ import annotations

import pytest
import torch

import sparse_reference as ref
from paged_reference import Pool, quantized
from test_gpu_sparse import DEV, _int32, _no_status, _pos, _randn, _tables

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
    out = ops.hif4_sparse_attention(q, pool.pages, table, cu, lens, lists.to(DEV), page_size=page).double().cpu()
    group = heads // h
    for t in range(tokens):
        for j in range(h):
            mine = at[torch.tensor(sorted(set(lists[t, j].tolist()) - {-1}))]
            keys, values = (x[mine, :, j].reshape(-1, d) for x in (k, v))
            p = torch.softmax(q[t, j * group : (j + 1) * group].double().cpu() @ keys.T * d**-0.5, -1)
            error = (out[t, j * group : (j + 1) * group] - p @ values).abs()
            assert bool((error <= BOUND * (p @ values.abs()) + 2.0**-126).all())
    _no_status()
