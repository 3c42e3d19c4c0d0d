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
