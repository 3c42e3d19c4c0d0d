"""The paged HiF4 K/V cache (faq_hif4_kv_write / _read) and the attention of new tokens over it
(faq_hif4_paged_attention), against the oracle's quantizer and a 64-bit softmax.

Tolerance of the attention, derived: bf16 has 8 significant bits, so its rounding errs by at
most 2^-8 of the value. P is rounded to bf16 after its product with V's scale, the output to
bf16 (|O| <= A, A = sum p |v|); scores are fp32 sums of 128 exact products, which moves p by
less than 2^-13 relative for the |scores| used here. So every value is within
(2^-8 + 2^-8 + 2^-12) A of the fp64 result, plus the smallest normal number."""

from __future__ import annotations

import pytest
import torch

from paged_reference import Pool, attention, quantized

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
BOUND = 2.0**-8 + 2.0**-8 + 2.0**-12


def _randn(*shape, seed, dtype=torch.bfloat16, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).to(DEV)


def _close(got, lens, new, q, k, v, scale=None):
    ref, size = attention(q, k, v, lens, new, scale)
    err = (got.double().cpu() - ref).abs()
    assert bool((err <= BOUND * size + 2.0**-126).all()), float((err / size.clamp(min=1e-30)).max())


def _no_status():
    from faquant_b200 import _lib

    torch.cuda.synchronize()
    assert _lib.device_status(reset=True) == 0


# ------------------------------------------------------------------ write, read
@pytest.mark.parametrize("levels", ["123", "12", "13"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("d", [64, 128])
def test_write_then_read_gives_the_oracles_values(d, dtype, levels) -> None:
    lens = [1, 2, 15, 16, 17, 0, 63, 200]
    pool = Pool(lens, 3, d, 32, DEV)
    k = _randn(sum(lens), 3, d, seed=1, dtype=dtype, scale=3.0)
    v = _randn(sum(lens), 3, d, seed=2, dtype=dtype, scale=0.01)
    k[::7] *= 1e4
    v[::5] = 0
    pool.write(k, v, levels=(levels, "123"))
    for out_dtype in (torch.bfloat16, torch.float32):
        rk, rv = pool.read(dtype=out_dtype)
        assert torch.equal(rk.float().cpu(), quantized(k, levels)) and torch.equal(rv.float().cpu(), quantized(v))
    _no_status()


def test_the_cache_holds_the_operand_preparations_values() -> None:
    from faquant_b200 import ops

    pool = Pool([70], 2, 128, 16, DEV)
    k, v = _randn(70, 2, 128, seed=3), _randn(70, 2, 128, seed=4)
    pool.write(k, v)
    rk, rv = pool.read()
    for x, r in ((k, rk), (v, rv)):
        prep = ops.qk_prep(x.transpose(0, 1)[None], levels="123", rotate=False)[0]
        assert torch.equal(prep[0].transpose(0, 1), r)


@pytest.mark.parametrize("page_size", [16, 64, 256])
def test_tokens_written_one_by_one_or_in_chunks_give_the_same_pages(page_size) -> None:
    lens, h, d = [37, 5], 2, 128
    k, v = _randn(42, h, d, seed=5), _randn(42, h, d, seed=6)
    whole, steps = (Pool(lens, h, d, page_size, DEV, seed=9) for _ in range(2))
    whole.write(k, v)
    for begin, end in [(0, 1), (1, 2), (2, 19), (19, 20), (20, 37)]:  # the other sequence idle, then in the last step
        new = [end - begin, 5 if end == 37 else 0]
        parts = [torch.cat((x[begin:end], x[37:] if end == 37 else x[:0])) for x in (k, v)]
        steps.write(*parts, new=new, lens=[end, 5 if end == 37 else 0])
    assert torch.equal(whole.store, steps.store)


def test_write_touches_only_its_tokens_bytes() -> None:
    from faquant_b200 import ops

    pool = Pool([40], 2, 64, 16, DEV, gap=16)
    before = pool.store.clone()
    k = _randn(3, 2, 64, seed=7)
    pool.write(k, k, new=[3])
    changed = (pool.store != before).sum().item()
    assert 0 < changed <= 3 * 2 * 2 * 37  # three tokens, K and V, two heads, 37 bytes each
    assert torch.equal(pool.store[:, -16:], before[:, -16:])
    rk, _ = pool.read(new=[3])
    assert torch.equal(rk.float().cpu(), quantized(k))
    assert ops.hif4_page_bytes(2, 64, 16) == 2 * 2 * 592


def test_strides_alignment_and_outputs() -> None:
    lens, h, d = [21, 40], 2, 128
    total = sum(lens)
    pool = Pool(lens, h, d, 16, DEV)
    wide = _randn(total, 3 * h * d + 8, seed=8)  # a fused projection: heads strided, a slice not 16-byte aligned
    k = wide[:, 1 : 1 + h * d].unflatten(1, (h, d))
    v = _randn(h, total, d, seed=9).transpose(0, 1)  # heads outermost
    assert k.data_ptr() % 16
    pool.write(k, v)
    want_k, want_v = quantized(k), quantized(v)
    rk, rv = pool.read()
    assert torch.equal(rk.float().cpu(), want_k) and torch.equal(rv.float().cpu(), want_v)
    out_k = torch.empty(total, h, d + 1, device=DEV)[..., 1:]  # unaligned rows
    out_v = torch.empty(h, total, d, device=DEV).transpose(0, 1)
    pool.read(out=(out_k, out_v))
    assert torch.equal(out_k.cpu(), want_k) and torch.equal(out_v.cpu(), want_v)


def test_offsets_past_32_bits() -> None:
    """Pages beyond 2^31 and 2^32 bytes of a pool, written, read and attended to."""
    from faquant_b200 import ops

    size = ops.hif4_page_bytes(8, 128, 4096)
    count = (1 << 32) // size + 4
    pages = torch.empty(count, size, dtype=torch.uint8, device=DEV)
    table = torch.tensor([[(1 << 31) // size + 1], [count - 1]], dtype=torch.int32, device=DEV)
    lens, new = [50, 33], [50, 33]
    cu = torch.tensor([0, 50, 83], dtype=torch.int32, device=DEV)
    lens_d = torch.tensor(lens, dtype=torch.int32, device=DEV)
    k, v = _randn(83, 8, 128, seed=10), _randn(83, 8, 128, seed=11)
    q = _randn(83, 8, 128, seed=12)
    ops.hif4_kv_write(k, v, pages, table, cu, lens_d, page_size=4096)
    rk, rv = ops.hif4_kv_read(pages, table, cu, lens_d, page_size=4096, head_dim=128, total=83)
    assert torch.equal(rk.float().cpu(), quantized(k)) and torch.equal(rv.float().cpu(), quantized(v))
    out = ops.hif4_paged_attention(q, pages, table, cu, lens_d, page_size=4096, max_new=50)
    _close(out, lens, new, q, rk, rv)
    _no_status()


def test_a_page_of_more_than_8_gib() -> None:
    """V stands more than 2^32 bytes behind K in a page of very many heads: for the kernels of few
    rows, of up to 128 and of more."""
    from faquant_b200 import ops

    h, d, ps = 14400, 128, 4096
    pages = torch.zeros(1, ops.hif4_page_bytes(h, d, ps), dtype=torch.uint8, device=DEV)
    assert pages.shape[1] // 2 > 1 << 32
    table = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    length = 140
    g = torch.Generator(DEV).manual_seed(15)
    k, v = (torch.randn(length, h, d, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
    some = torch.tensor([0, 1, 7000, 14168, 14169, 14170, 14171, h - 1], device=DEV)
    kq, vq = quantized(k[:, some]), quantized(v[:, some])
    cu, lens = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([0, length], [length]))
    ops.hif4_kv_write(k, v, pages, table, cu, lens, page_size=ps)
    for n, most in ((1, 1), (20, 20), (140, 140), (135, 140)):  # the last: q has rows beyond the batch
        cu = torch.tensor([0, n], dtype=torch.int32, device=DEV)
        q = torch.randn(most, h, d, generator=g, device=DEV).to(torch.bfloat16)
        out = ops.hif4_paged_attention(q, pages, table, cu, lens, page_size=ps, max_new=n, max_len=4096, total_len=length)
        _close(out[:n, some], [length], [n], q[:n, some], kq, vq)
    _no_status()


def test_tokens_without_a_place() -> None:
    """Positions below zero are skipped; bad table entries and lengths are reported."""
    from faquant_b200 import _lib, ops

    pool = Pool([20], 1, 64, 16, DEV)
    k = _randn(20, 1, 64, seed=13)
    pool.write(k, k, new=[20])
    keep = pool.store.clone()
    ops.hif4_kv_write(k, k, pool.pages, pool.table, pool.cu([20]), torch.tensor([4], dtype=torch.int32, device=DEV),
                      page_size=16)  # only the last four tokens have a place
    pool.lens.fill_(4)
    assert torch.equal(pool.read(new=[4])[0].float().cpu(), quantized(k[16:]))
    rk, _ = pool.read(new=[6])
    assert not rk[:2].any() and torch.equal(rk[2:].float().cpu(), quantized(k[16:]))
    _no_status()
    pool.store.copy_(keep)
    pool.lens.fill_(20)
    pool.table[0, 1] = 10**6
    rk, _ = pool.read(new=[20])
    assert torch.equal(rk[:16].float().cpu(), quantized(k[:16])) and not rk[16:].any()
    assert _lib.device_status(reset=True) == _lib.FAQ_STATUS_BAD_PAGE
    pool.write(k, k, new=[20])
    assert _lib.device_status(reset=True) == _lib.FAQ_STATUS_BAD_PAGE
    # the attention leaves that page's keys out
    q = _randn(1, 2, 64, seed=14)
    out = pool.attend(q, [1])
    ref, size = attention(q, quantized(k[:16]), quantized(k[:16]), [16], [1])
    assert bool(((out.double().cpu() - ref).abs() <= BOUND * size).all())
    assert _lib.device_status(reset=True) == _lib.FAQ_STATUS_BAD_PAGE


# ------------------------------------------------------------------ attention
# Short sequences of any number of rows may be one kernel's; a higher bound on their lengths
# gives the same batches to the kernels of long ones.
MAX_LEN = [0, 5000]
SHAPES = [  # heads, kv_heads, d, page_size, lens, new
    (4, 1, 128, 16, [1], [1]),
    (8, 2, 128, 16, [1, 2, 15, 16, 17, 127, 129, 500], [1] * 8),
    (32, 8, 128, 64, [3000], [1]),
    (5, 1, 128, 32, [100, 31], [1, 3]),
    (7, 1, 64, 16, [90, 300], [2, 1]),
    (2, 2, 64, 128, [40, 700, 0, 3], [1, 8, 0, 3]),
    (16, 4, 128, 32, [5, 70, 64, 200], [5, 0, 8, 1]),
    (16, 2, 64, 16, [33, 260], [33, 17]),
    (12, 4, 128, 16, [130], [130]),
    (24, 2, 128, 256, [700, 20], [40, 20]),
    (3, 3, 128, 16, [0, 0, 9], [0, 0, 1]),
    # more rows (tokens x query heads of a kv head): up to 128, beyond
    (4, 1, 128, 16, [17], [17]),
    (4, 1, 128, 16, [200, 16, 17], [17, 16, 16]),
    (8, 8, 128, 64, [65, 128, 129, 300], [65, 128, 129, 256]),
    (10, 2, 128, 16, [400, 1, 90], [150, 1, 90]),
    (14, 2, 64, 32, [300, 80], [60, 11]),
    (32, 2, 64, 16, [513, 0, 40], [9, 0, 40]),
    (128, 1, 128, 16, [70], [3]),
    (48, 2, 128, 128, [1300], [45]),
]


@pytest.mark.parametrize("max_len", MAX_LEN)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"h{s[0]}_{s[1]}_d{s[2]}_p{s[3]}_b{len(s[4])}_n{max(s[5])}")
def test_attention_matches_fp64(shape, max_len) -> None:
    heads, h, d, page, lens, new = shape
    pool = Pool(lens, h, d, page, DEV, fill=0xFF)  # unwritten slots hold the largest scales and codes
    k, v = _randn(sum(lens), h, d, seed=20), _randn(sum(lens), h, d, seed=21, scale=0.5)
    pool.write(k, v)
    q = _randn(sum(new), heads, d, seed=22, scale=2.0)
    out = pool.attend(q, new, max_len)
    assert out.shape == q.shape and out.dtype == torch.bfloat16
    _close(out, lens, new, q, quantized(k), quantized(v))
    _no_status()


@pytest.mark.parametrize("max_len", MAX_LEN)
@pytest.mark.parametrize("n", [1, 2, 4, 7, 9, 14, 30, 40, 150])
def test_rows_without_a_key_are_zero(n, max_len) -> None:
    """More new tokens than the sequence holds: the first have no position."""
    lens, new = [max(1, n // 2), 0, 300], [n, n, n]
    pool = Pool(lens, 2, 128, 16, DEV)
    k, v = _randn(sum(lens), 2, 128, seed=23), _randn(sum(lens), 2, 128, seed=24)
    pool.write(k, v)
    q = _randn(3 * n, 8, 128, seed=25)
    out = torch.full_like(q, float("nan"))
    pool.attend(q, new, max_len, out=out)
    none = n - lens[0]
    assert not out[:none].any() and not out[n : 2 * n].any()
    _close(out, lens, new, q, quantized(k), quantized(v))


def test_a_step_of_queries_equals_each_alone() -> None:
    """Chunk invariance: the drafts' rows, attended together, are the rows of one-token calls
    within the bound of both."""
    pool = Pool([1500], 2, 128, 64, DEV)
    k, v = _randn(1500, 2, 128, seed=26), _randn(1500, 2, 128, seed=27)
    pool.write(k, v)
    q = _randn(8, 16, 128, seed=28, scale=2.0)
    out = pool.attend(q, [8])
    _, size = attention(q, quantized(k), quantized(v), [1500], [8])
    for i in range(8):
        pool.lens.fill_(1500 - 7 + i)
        one = pool.attend(q[i : i + 1], [1])
        assert bool(((one[0] - out[i]).double().abs().cpu() <= 2 * BOUND * size[i]).all())


@pytest.mark.parametrize("n", [1, 7, 20, 70, 200])
def test_sequences_beyond_the_rows_given_are_reported(n) -> None:
    """cu says more tokens than k, v, q or `total` have rows, or falls: such a sequence is left out and
    recorded, the others are served."""
    from faquant_b200 import _lib, ops

    lens = [300, 300]
    pool = Pool(lens, 1, 64, 16, DEV)
    k, v = _randn(600, 1, 64, seed=45), _randn(600, 1, 64, seed=46)
    pool.write(k, v)
    _no_status()
    before = pool.store.clone()
    q = _randn(2 * n, 2, 64, seed=47)
    kw = dict(page_size=16)
    for bounds in ([0, n, 2 * n + 1], [0, n, n - 1]):
        cu = torch.tensor(bounds, dtype=torch.int32, device=DEV)
        args = (pool.pages, pool.table, cu, pool.lens)
        for max_len in (300, 5000):
            out = torch.full_like(q, 7.0)
            ops.hif4_paged_attention(q, *args, max_new=n, max_len=max_len, out=out, **kw)
            assert _lib.device_status(reset=True) == _lib.FAQ_STATUS_BAD_BOUND
            _close(out[:n], [300], [n], q[:n], quantized(k[:300]), quantized(v[:300]))
            assert bool((out[n:] == 7.0).all())
        back = [torch.full((2 * n, 1, 64), 7.0, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
        ops.hif4_kv_read(*args, head_dim=64, total=2 * n, out=tuple(back), **kw)
        assert _lib.device_status(reset=True) == _lib.FAQ_STATUS_BAD_BOUND
        assert torch.equal(back[0][:n].float().cpu(), quantized(k[300 - n : 300])) and bool((back[0][n:] == 7.0).all())
        new = torch.cat((k[300 - n : 300], k[:n]))  # the first sequence's tokens once more
        ops.hif4_kv_write(new, torch.cat((v[300 - n : 300], v[:n])), *args, **kw)
        assert _lib.device_status(reset=True) == _lib.FAQ_STATUS_BAD_BOUND
        assert torch.equal(pool.store, before)


@pytest.mark.parametrize("n", [4, 7, 14, 30, 40])
def test_peaked_and_flat_scores_scale_and_ranges(n) -> None:
    lens, new = [900], [n]
    pool = Pool(lens, 1, 128, 16, DEV)
    k, v = _randn(900, 1, 128, seed=29), _randn(900, 1, 128, seed=30)
    k[700] *= 30.0  # one key far above the others, found late
    v[3] *= 1e6     # and a value row of another magnitude
    v[600:] *= 1e-20
    pool.write(k, v)
    q = _randn(n, 4, 128, seed=31)
    q[1] = 0
    for scale in (None, 0.002, 0.5):
        _close(pool.attend(q, new, 5000, scale=scale), lens, new, q, quantized(k), quantized(v), scale)


@pytest.mark.parametrize("max_len", MAX_LEN)
@pytest.mark.parametrize("n", [6, 12, 30])
def test_not_a_number_stays_in_its_row(n, max_len) -> None:
    pool = Pool([300], 2, 128, 16, DEV)
    k, v = _randn(300, 2, 128, seed=32), _randn(300, 2, 128, seed=33)
    pool.write(k, v)
    q = _randn(n, 8, 128, seed=34)
    good = pool.attend(q, [n], max_len)
    q[2, 5, 17] = float("nan")
    q[4, 0, 0] = float("inf")
    out = pool.attend(q, [n], max_len)
    assert out[2, 5].isnan().all() and out[4, 0].isnan().any()
    out[2, 5], out[4, 0] = good[2, 5], good[4, 0]
    assert torch.equal(out, good)


def test_shared_pages_strides_streams_and_repetition() -> None:
    """Two sequences share a prefix's pages; q and out strided; another stream; the same bits
    on every call, with one workspace and back to back."""
    from faquant_b200 import ops

    pool = Pool([64, 0], 2, 128, 16, DEV, spare=4)
    k, v = _randn(64, 2, 128, seed=35), _randn(64, 2, 128, seed=36)
    pool.write(k, v)
    pool.table[1] = pool.table[0]
    pool.lens_host = [64, 64]
    pool.lens.fill_(64)
    wide = _randn(4, 3, 8, 136, seed=37)
    q = wide[:, 1, :, :128]
    out = torch.empty(8, 4, 128, dtype=torch.bfloat16, device=DEV).transpose(0, 1)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        pool.attend(q, [2, 2], out=out)
    stream.synchronize()
    kk, vv = torch.cat((quantized(k),) * 2), torch.cat((quantized(v),) * 2)
    _close(out, [64, 64], [2, 2], q, kk, vv)
    big = Pool([4000, 77, 2500], 2, 128, 32, DEV)
    k, v = _randn(6577, 2, 128, seed=38), _randn(6577, 2, 128, seed=39)
    big.write(k, v)
    new = [1, 1, 1]
    q = _randn(3, 16, 128, seed=40)
    first = big.attend(q, new)
    ws = torch.empty(64 << 20, dtype=torch.uint8, device=DEV)
    again = [big.attend(q, new, workspace=ws) for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(first, x) for x in again)
    assert ops.hif4_page_bytes(2, 128, 32) == 2 * 2 * 2 * 1184


def test_captured_in_a_graph_with_growing_lengths() -> None:
    """A captured step replays with the device's lengths of the moment."""
    pool = Pool([400], 2, 128, 64, DEV)
    k, v = _randn(400, 2, 128, seed=41), _randn(400, 2, 128, seed=42)
    pool.write(k, v)
    q = _randn(1, 8, 128, seed=43)
    out, ws = torch.empty_like(q), torch.empty(8 << 20, dtype=torch.uint8, device=DEV)
    cu = pool.cu([1])
    from faquant_b200 import ops

    def step():
        ops.hif4_paged_attention(q, pool.pages, pool.table, cu, pool.lens, page_size=64, max_new=1, max_len=400, out=out,
                                 workspace=ws)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for n in (1, 63, 64, 65, 399, 400):
        pool.lens.fill_(n)
        graph.replay()
        torch.cuda.synchronize()
        _close(out, [n], [1], q, quantized(k[:n]), quantized(v[:n]))


def test_prompt_kernel_over_many_runs_and_its_ranges() -> None:
    """A chunk whose units are cut over many CTAs, one query row far above the others, values
    of very different sizes; strided q; the same bits again."""
    lens, new = [5000, 260], [70, 200]
    pool = Pool(lens, 1, 128, 64, DEV)
    k, v = _randn(sum(lens), 1, 128, seed=60), _randn(sum(lens), 1, 128, seed=61)
    k[4000] *= 30.0
    v[3] *= 1e6
    pool.write(k, v)
    wide = _randn(sum(new), 3, 2, 136, seed=62)
    q = wide[:, 1, :, :128]
    q[20] *= 8.0
    q[21] = 0
    out = pool.attend(q, new)
    _close(out, lens, new, q, quantized(k), quantized(v))
    assert all(torch.equal(out, pool.attend(q, new, total_len=sum(lens))) for _ in range(3))
    _no_status()


def test_prompt_kernel_keeps_not_a_number_in_its_row() -> None:
    pool = Pool([300], 2, 128, 16, DEV, fill=0xFF)
    k, v = _randn(300, 2, 128, seed=63), _randn(300, 2, 128, seed=64)
    pool.write(k, v)
    q = _randn(90, 4, 128, seed=65)
    good = pool.attend(q, [90], 5000)
    q[12, 3, 17] = float("nan")
    q[40, 0, 0] = float("inf")
    out = pool.attend(q, [90], 5000)
    assert out[12, 3].isnan().all() and out[40, 0].isnan().any()
    out[12, 3], out[40, 0] = good[12, 3], good[40, 0]
    assert torch.equal(out, good)


def test_batches_beyond_their_bounds_are_reported() -> None:
    from faquant_b200 import _lib, ops

    lens, new = [400, 400], [50, 50]
    pool = Pool(lens, 2, 128, 16, DEV)
    k, v = _randn(800, 2, 128, seed=66), _randn(800, 2, 128, seed=67)
    pool.write(k, v)
    q = _randn(100, 8, 128, seed=68)
    out = torch.zeros_like(q)
    ops.hif4_paged_attention(q, pool.pages, pool.table, pool.cu(new), pool.lens, page_size=16, max_new=50, max_len=2000,
                             total_len=300, out=out)
    assert _lib.device_status(reset=True) == _lib.FAQ_STATUS_BAD_BOUND
    ref, size = attention(q, quantized(k), quantized(v), lens, new)  # the first one fits
    assert bool(((out.double().cpu() - ref).abs() <= BOUND * size)[:50].all()) and not out[50:].any()


def test_a_sequence_beyond_max_new_is_reported() -> None:
    from faquant_b200 import _lib, ops

    lens, new = [300, 300], [5, 60]
    pool = Pool(lens, 2, 128, 16, DEV)
    k, v = _randn(600, 2, 128, seed=69), _randn(600, 2, 128, seed=70)
    pool.write(k, v)
    q = _randn(65, 8, 128, seed=71)
    out = torch.zeros_like(q)
    ops.hif4_paged_attention(q, pool.pages, pool.table, pool.cu(new), pool.lens, page_size=16, max_new=30, max_len=2000,
                             out=out)
    assert _lib.device_status(reset=True) == _lib.FAQ_STATUS_BAD_BOUND
    ref, size = attention(q, quantized(k), quantized(v), lens, new)
    assert bool(((out.double().cpu() - ref).abs() <= BOUND * size)[:5].all()) and not out[5:].any()


@pytest.mark.parametrize("max_len", [0, 20000])
@pytest.mark.parametrize("new", [[200, 1, 1, 30, 0, 2], [130, 64, 64, 64, 0, 300], [0, 1, 0, 0, 1, 129]])
def test_prompts_and_steps_in_one_batch(new, max_len) -> None:
    """One kernel for all, or one for the long chunks and one for the others, as the bound on
    the lengths has it."""
    lens = [700, 64, 1, 300, 0, 350]
    pool = Pool(lens, 8, 64, 32, DEV, fill=0xFF)
    k, v = _randn(sum(lens), 8, 64, seed=75), _randn(sum(lens), 8, 64, seed=76)
    pool.write(k, v)
    q = _randn(sum(new), 16, 64, seed=77)
    out = torch.full_like(q, float("nan"))
    pool.attend(q, new, max_len, out=out)
    _close(out, lens, new, q, quantized(k), quantized(v))
    _no_status()


@pytest.mark.parametrize("max_len", [400, 2000])
@pytest.mark.parametrize("new", [[60, 7, 1, 0], [60, 60, 60, 60], [1, 1, 0, 1], [8, 2, 0, 0], [12, 9, 3, 1]])
def test_rows_beyond_the_batch_stay_as_they_are(new, max_len) -> None:
    """A q of a fixed size (batch x max_new rows), of which the batch uses the first."""
    from faquant_b200 import ops

    lens = [400, 90, 33, 200]
    pool = Pool(lens, 2, 128, 16, DEV)
    k, v = _randn(sum(lens), 2, 128, seed=72), _randn(sum(lens), 2, 128, seed=73)
    pool.write(k, v)
    used, most = sum(new), max(new)
    q = _randn(4 * most, 8, 128, seed=74)
    q[used:] = float("nan")
    out = torch.full_like(q, 7.0)
    ops.hif4_paged_attention(q, pool.pages, pool.table, pool.cu(new), pool.lens, page_size=16, max_new=most, max_len=max_len,
                             out=out)
    _close(out[:used], lens, new, q[:used], quantized(k), quantized(v))
    assert bool((out[used:] == 7.0).all())
    _no_status()


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("n", [1, 4, 8, 16, 30, 60, 150])
def test_keys_without_a_page_are_left_out(n, page) -> None:
    """Table entries outside the pool: their tokens are read as zeros and leave the softmax, in every
    kernel, whatever stood in the keys' place before; a sequence without pages gives zeros."""
    from faquant_b200 import _lib

    lens, new = [3000, 700, 200, 900], [n, n, n, n]
    pool = Pool(lens, 2, 64, page, DEV, seed=n)
    k, v = _randn(sum(lens), 2, 64, seed=83), _randn(sum(lens), 2, 64, seed=84)
    v[:3000] += 100.0  # the first sequence's values would show in another's output
    pool.write(k, v)
    holes = [[2, 700 // page], [0, 699 // page], list(range(-(-200 // page))), []]
    for b, cols in enumerate(holes):
        for i, col in enumerate(cols):
            pool.table[b, col] = (-1, 10**6, -(2**31), 2**31 - 1)[i % 4]
    q = _randn(4 * n, 8, 64, seed=85)
    out = torch.full_like(q, float("nan"))
    pool.attend(q, new, 5000, out=out)
    assert _lib.device_status(reset=True) == _lib.FAQ_STATUS_BAD_PAGE
    rk, rv = pool.read()
    assert _lib.device_status(reset=True) == _lib.FAQ_STATUS_BAD_PAGE
    kq, vq, begin = quantized(k).double(), quantized(v).double(), 0
    for b, length in enumerate(lens):
        here = torch.tensor([i // page not in holes[b] for i in range(length)])
        key, value = kq[begin : begin + length], vq[begin : begin + length]
        for got, want in ((rk, key), (rv, value)):
            assert torch.equal(got[begin : begin + length].double().cpu(), want * here[:, None, None])
        seen = here & (torch.arange(length) <= torch.arange(length - n, length)[:, None])
        s = torch.einsum("nhd,khd->hnk", q[b * n : b * n + n].double().cpu(), key.repeat_interleave(4, 1)) / 8.0
        p = torch.softmax(s.masked_fill(~seen, float("-inf")), -1).nan_to_num(0.0)  # no key: 0 / 0
        ref, size = (torch.einsum("hnk,khd->nhd", p, x.repeat_interleave(4, 1)) for x in (value, value.abs()))
        assert bool(((out[b * n : b * n + n].double().cpu() - ref).abs() <= BOUND * size + 2.0**-126).all()), b
        begin += length
    assert not out[2 * n : 3 * n].any()


@pytest.mark.parametrize("group,new", [(4, 5), (3, 21), (12, 10), (5, 25), (4, 9), (3, 200), (7, 90), (14, 30)])
def test_the_bits_depend_on_a_sequences_own_queries_only(group, new) -> None:
    """Neither the next sequence's queries, nor rows of q beyond the batch, nor what a call before left in
    shared memory (rows of a tile that no box of whole tokens fills) may move a rounding."""
    lens, counts = [3000, 2500], [new, new]
    pool = Pool(lens, 2, 128, 32, DEV)
    k, v = _randn(sum(lens), 2, 128, seed=86), _randn(sum(lens), 2, 128, seed=87)
    pool.write(k, v)
    q = _randn(2 * new + 40, 2 * group, 128, seed=88)
    other = _randn(2 * new, 2 * 4 if 4 * new > 16 else 64, 128, seed=89, scale=200.0)
    used = slice(0, 2 * new)
    want = pool.attend(q, counts, 5000)
    _close(want[used], lens, counts, q[used], quantized(k), quantized(v))
    for scale in (0.0, 60.0, 200.0, float("nan")):
        pool.attend(other, counts, 5000)
        x = q.clone()
        x[2 * new :] *= scale
        assert torch.equal(pool.attend(x, counts, 5000)[used], want[used]), scale
        x[new:] *= scale
        assert torch.equal(pool.attend(x, counts, 5000)[:new], want[:new]), scale
    _no_status()


# ------------------------------------------------------------------ many sequences
@pytest.mark.parametrize("most", [2, 20, 70], ids=["few", "chunk", "prompt"])
@pytest.mark.parametrize("batch", [40, 600, 1300])
def test_many_sequences(batch, most) -> None:
    """More sequences than a warp's lanes (40), than the threads of the few rows' kernel (600) and
    of the chunks' kernel (1300): ragged, with idle ones, short and long ones, and tokens
    without a key in all of them. The prefix sums over the batch say whose keys a CTA reads."""
    g = torch.Generator().manual_seed(batch + most)
    lens = torch.randint(0, 40, (batch,), generator=g)
    lens[torch.randint(0, batch, (3,), generator=g)] = 1100
    new = torch.where(torch.rand(batch, generator=g) < 0.4, 0, torch.randint(1, most + 1, (batch,), generator=g))
    if most == 70:  # prompts and steps in one batch
        new = torch.where(torch.rand(batch, generator=g) < 0.9, new.clamp(max=2), new)
    new[batch - 3], lens[batch - 3] = most, max(0, most - 1)  # the first of them has no key
    new[5] = most
    lens, new = lens.tolist(), new.tolist()
    pool = Pool(lens, 1, 64, 16, DEV, fill=0xFF)
    k, v = _randn(sum(lens), 1, 64, seed=80), _randn(sum(lens), 1, 64, seed=81)
    pool.write(k, v)
    rk, rv = pool.read()
    kq, vq = quantized(k), quantized(v)
    assert torch.equal(rk.float().cpu(), kq) and torch.equal(rv.float().cpu(), vq)
    q = _randn(sum(new), 2, 64, seed=82)
    ref, size = attention(q, kq, vq, lens, new)
    for max_len in (0, 5000):
        for _ in range(3):
            out = torch.full_like(q, float("nan"))
            pool.attend(q, new, max_len, out=out)
            assert bool(((out.double().cpu() - ref).abs() <= BOUND * size + 2.0**-126).all())
    tail, _ = pool.read(new=[min(n, length) for n, length in zip(new, lens)])
    ends = torch.tensor(lens).cumsum(0).tolist()
    want = torch.cat([kq[e - min(n, length) : e] for e, n, length in zip(ends, new, lens)])
    assert torch.equal(tail.float().cpu(), want)
    _no_status()


# ------------------------------------------------------------------ refusals
def test_refusals() -> None:
    from faquant_b200 import ops

    pool = Pool([20, 20], 2, 128, 16, DEV)
    cu, kw = pool.cu([1, 1]), dict(page_size=16)
    k = _randn(2, 2, 128, seed=50)
    q = _randn(2, 4, 128, seed=51)
    args = (pool.pages, pool.table, cu, pool.lens)
    with pytest.raises(ValueError):  # another page size than the pages'
        ops.hif4_kv_write(k, k, *args, page_size=32)
    with pytest.raises(ValueError):  # not a power of two
        ops.hif4_kv_write(k, k, *args, page_size=24)
    with pytest.raises(ValueError):  # K and V differ
        ops.hif4_kv_write(k, k[:1], *args, **kw)
    with pytest.raises(TypeError):
        ops.hif4_kv_write(k.half(), k.half(), *args, **kw)
    with pytest.raises(ValueError):
        ops.hif4_kv_write(k, k, *args, levels=("123", "23"), **kw)
    with pytest.raises(TypeError):  # 64-bit lengths
        ops.hif4_kv_write(k, k, pool.pages, pool.table, cu, pool.lens.long(), **kw)
    with pytest.raises(ValueError):  # cu of another batch
        ops.hif4_paged_attention(q, pool.pages, pool.table, cu[:2], pool.lens, max_new=1, **kw)
    with pytest.raises(ValueError):  # heads not a multiple
        ops.hif4_paged_attention(q[:, :3], *args, max_new=1, **kw)
    with pytest.raises(TypeError):
        ops.hif4_paged_attention(q.float(), *args, max_new=1, **kw)
    with pytest.raises(ValueError):
        ops.hif4_paged_attention(q, *args, max_new=1, scale=-1.0, **kw)
    with pytest.raises(ValueError):  # head_dim the pages do not have
        ops.hif4_paged_attention(_randn(2, 4, 64, seed=52), *args, max_new=1, **kw, out=q)
    with pytest.raises(RuntimeError):  # host tensors
        ops.hif4_kv_read(pool.pages.cpu(), pool.table, cu, pool.lens, head_dim=128, total=2, **kw)
    with pytest.raises(ValueError):
        ops.hif4_kv_read(*args, head_dim=96, total=2, **kw)
    with pytest.raises(ValueError):
        ops.hif4_kv_read(*args, head_dim=128, total=2, out=(k, k[:1]), **kw)


def test_no_tokens_is_no_work() -> None:
    pool = Pool([20], 2, 128, 16, DEV)
    empty = torch.empty(0, 2, 128, dtype=torch.bfloat16, device=DEV)
    before = pool.store.clone()
    pool.write(empty, empty, new=[0])
    assert torch.equal(before, pool.store)
    assert pool.read(new=[0])[0].shape == (0, 2, 128)
    assert pool.attend(torch.empty(0, 4, 128, dtype=torch.bfloat16, device=DEV), [0]).shape == (0, 4, 128)
