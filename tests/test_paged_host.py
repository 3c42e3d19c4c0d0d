"""Host-side checks of the paged-cache and verification entry points (no GPU): refusals before
any CUDA call, and the size functions."""

from __future__ import annotations

import ctypes

import pytest
import torch


def test_page_bytes() -> None:
    from faquant_b200 import ops

    assert ops.hif4_page_bytes(8, 128, 64) == 2 * 8 * 64 * 74  # 74 bytes per token, head and K or V
    assert ops.hif4_page_bytes(1, 64, 16) == 2 * 592
    for bad in ((1, 96, 16), (1, 128, 8), (1, 128, 48)):
        with pytest.raises(ValueError):
            ops.hif4_page_bytes(*bad)


def test_c_entry_points_refuse_bad_arguments() -> None:
    from faquant_b200 import _lib

    lib = _lib.load()
    p = ctypes.c_void_p(256)

    def write(d=128, page=16, stride=1 << 20, pages=p, levels=123, dtype=0):
        return lib.faq_hif4_kv_write(p, p, dtype, 4, 2, d, 256, 128, 256, 128, pages, 4, stride, page, p, 3, 3, p, p, 1,
                                     levels, 123, None)

    assert write(pages=None) == 1 and "null" in _lib.last_error()
    assert write(d=96) == 3 and "head_dim" in _lib.last_error()
    assert write(page=24) == 3 and "page_size" in _lib.last_error()
    assert write(stride=1000) == 1 and "aligned" in _lib.last_error()
    assert write(stride=1024) == 1 and "page stride" in _lib.last_error()
    assert write(pages=ctypes.c_void_p(8)) == 1
    assert write(levels=1) == 1 and "levels" in _lib.last_error()
    assert write(dtype=7) == 1 and "dtype" in _lib.last_error()

    def attend(heads=4, scale=1.0, ws=1 << 30, qs=512, max_new=4):
        return lib.faq_hif4_paged_attention(p, 4, heads, qs, 128, p, 4, 1 << 20, 16, 2, 128, p, 3, 3, p, p, 1, max_new, 2000,
                                            2000, ctypes.c_float(scale), p, 512, 128, p, ws, None)

    assert attend(heads=3) == 1 and "divisible" in _lib.last_error()
    assert attend(scale=0.0) == 1 and "scale" in _lib.last_error()
    assert attend(scale=float("nan")) == 1
    assert attend(qs=12) == 1 and "strides" in _lib.last_error()
    assert attend(ws=16) == 1 and "workspace" in _lib.last_error()
    assert attend(max_new=-1) == 1
    # one kernel without joins needs no workspace: eight rows, short sequences
    assert lib.faq_hif4_paged_attention_workspace_bytes(4, 4, 2, 1, 4, 1024, 1024, 128) == 0
    assert lib.faq_hif4_paged_attention_workspace_bytes(4, 4, 2, 1, 4, 1025, 1025, 128) > 0
    assert lib.faq_hif4_paged_attention_workspace_bytes(4, 6, 4, 1, 1, 48, 48, 128) == 0

    def verify(batch=1, k=2, vocab=10, dtype=1, target=p):
        return lib.faq_verify_drafts(p, target, None, dtype, batch, k, vocab, 30, 10, 0, 0, p, p, None, p, p, None)

    assert verify(target=None) == 1 and verify(vocab=0) == 1 and verify(vocab=1 << 23) == 1
    assert verify(k=-1) == 1 and verify(dtype=3) == 1
    assert verify(batch=0) == 0


def test_operators_refuse_cpu_tensors() -> None:
    from faquant_b200 import ops

    x = torch.zeros(2, 1, 64, dtype=torch.bfloat16)
    pages = torch.zeros(1, 1184, dtype=torch.uint8)
    table, cu, lens = (torch.zeros(*s, dtype=torch.int32) for s in ((1, 1), (2,), (1,)))
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.hif4_kv_write(x, x, pages, table, cu, lens, page_size=16)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.hif4_paged_attention(x, pages, table, cu, lens, page_size=16, max_new=1)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.verify_drafts(torch.zeros(1, 1, dtype=torch.int64), torch.ones(1, 2, 4), None, torch.ones(1, 1), torch.ones(1))


def test_lookup_drafts() -> None:
    from faquant_b200.generate import lookup_drafts

    assert lookup_drafts([1, 2, 3, 9, 1, 2, 3], 3, 3) == [9, 1, 2]
    assert lookup_drafts([1, 2, 3, 9, 7, 2, 3], 2, 3) == [9, 7]  # the last three do not recur, the last two do
    assert lookup_drafts([5, 6, 5, 7, 5], 4, 1) == [7, 5]  # the latest occurrence
    assert lookup_drafts([1, 2, 3], 4, 3) == [] and lookup_drafts([1], 4, 3) == [] and lookup_drafts([1, 1], 0, 2) == []


def test_paged_attention_needs_its_cache_and_no_mask() -> None:
    import types

    from faquant_b200.generate import paged_speculative_generate
    from faquant_b200.kv_cache import PagedKVCache

    with pytest.raises(ValueError):
        paged_speculative_generate(types.SimpleNamespace(), input_ids=torch.zeros(2, 3, dtype=torch.int64), max_length=9)
    with pytest.raises(ValueError):
        paged_speculative_generate(types.SimpleNamespace(), input_ids=torch.zeros(1, 3, dtype=torch.int64), max_length=9,
                                   num_drafts=-1)
    out, stats = paged_speculative_generate(types.SimpleNamespace(), input_ids=torch.zeros(1, 3, dtype=torch.int64), max_length=3)
    assert out.shape == (1, 3) and stats["steps"] == 0
    with pytest.raises(ValueError):
        PagedKVCache(1, 2, 96, max_length=10, device="cpu")
    cache = PagedKVCache(2, 2, 64, max_length=100, page_size=16, device="cpu")  # host bookkeeping runs anywhere
    cache.extend([33])
    assert cache.get_seq_length() == 33 and cache.table[0, :4].tolist() == [0, 1, 2, -1]
    cache.truncate([16])
    cache.extend([1])
    assert cache.lengths == [17] and len(cache._held[0]) == 2 and cache.get_mask_sizes(5) == (22, 0)


def _paged_layer(**attributes):
    """A Qwen3 attention layer on the host that runs the adapter, and its cache."""
    from transformers import Qwen3Config
    from transformers.models.qwen3.modeling_qwen3 import Qwen3Attention

    from faquant_b200.kv_cache import PagedKVCache

    cfg = Qwen3Config(hidden_size=32, num_hidden_layers=2, num_attention_heads=2, num_key_value_heads=1, head_dim=64,
                      use_sliding_window=True, sliding_window=8, max_window_layers=1,
                      layer_types=["full_attention", "sliding_attention"])
    layer = Qwen3Attention(cfg, attributes.pop("layer_idx", 0)).to(torch.bfloat16)
    layer.faquant_attention_kernel = "paged"
    for name, value in attributes.items():
        setattr(layer, name, value)
    return layer, PagedKVCache(2, 1, 64, max_length=64, page_size=16, device="cpu")


def _forward(layer, cache, mask=None, **kwargs):
    from faquant_b200.qwen3 import attention_forward

    x = torch.zeros(1, 3, 32, dtype=torch.bfloat16)
    cos = torch.ones(1, 3, 64, dtype=torch.bfloat16)
    return attention_forward(layer, x, (cos, torch.zeros_like(cos)), mask, past_key_values=cache, **kwargs)


def test_paged_layer_refuses_what_it_does_not_do() -> None:
    layer, cache = _paged_layer()
    with pytest.raises(RuntimeError, match="CUDA tensors only"):  # nothing to refuse: it goes on to the kernels
        _forward(layer, cache)
    window = torch.tensor([0, 3], dtype=torch.int32)
    for kwargs, error in (({"cu_seq_lens_q": window}, NotImplementedError), ({"cu_seq_lens_k": window}, NotImplementedError),
                          ({"max_length_q": 3}, NotImplementedError), ({"is_causal": False}, NotImplementedError),
                          ({"softcap": 30.0}, NotImplementedError), ({"sliding_window": 4}, NotImplementedError),
                          ({"mask": torch.ones(1, 3)}, NotImplementedError), ({"dropout": 0.1}, ValueError),
                          ({"output_attentions": True}, ValueError)):
        layer, cache = _paged_layer()
        with pytest.raises(error):
            _forward(layer, cache, **kwargs)
        assert cache.lengths == [0]  # no step was opened
    for attributes in ({"layer_idx": 1}, {"sliding_window": 8}, {"is_causal": False}):
        layer, cache = _paged_layer(**attributes)
        with pytest.raises(NotImplementedError):
            _forward(layer, cache)
        assert cache.lengths == [0]


def test_paged_layer_reads_the_operand_recipe() -> None:
    hif4 = {"quant_format": "hif4", "bits": 4, "group_size": 64}
    integer = {"quant_format": "int", "bits": 4, "group_size": 64}
    for attributes in ({"faquant_qk_matmul_quant": False}, {"faquant_pv_matmul_quant": False},
                       {"faquant_qk_matmul_quant": True, "faquant_matmul_quant_kwargs": integer},
                       {"faquant_pv_matmul_quant": True, "faquant_matmul_quant_kwargs": hif4,
                        "faquant_pv_matmul_quant_kwargs": integer},
                       {"faquant_qk_matmul_quant_kwargs": hif4 | {"group_size": 32}},
                       {"faquant_qk_matmul_quant_kwargs": hif4 | {"bits": 8}}):
        layer, cache = _paged_layer(**attributes)
        with pytest.raises(NotImplementedError):
            _forward(layer, cache)
        assert cache.lengths == [0]
    for attributes in ({"faquant_qk_matmul_quant": True, "faquant_pv_matmul_quant": True,
                        "faquant_matmul_quant_kwargs": hif4},
                       {"faquant_matmul_quant_kwargs": integer, "faquant_qk_matmul_quant_kwargs": hif4,
                        "faquant_pv_matmul_quant_kwargs": hif4 | {"group_size": -1}}):
        layer, cache = _paged_layer(**attributes)
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            _forward(layer, cache)


@pytest.mark.parametrize("bad_call", [0, 1])
def test_generation_stops_when_there_is_no_token_to_sample(monkeypatch, bad_call) -> None:
    """NaN logits at a temperature leave no mass, which verification reports as token -1: it is raised and
    never fed to the model. (Verification itself runs on a GPU only; its reference stands in.)"""
    import types

    from faquant_b200 import ops
    from faquant_b200.generate import paged_speculative_generate
    from faquant_b200.kv_cache import PagedKVCache
    from paged_reference import verify

    def on_host(draft, target, drafter, accept_u, sample_u):
        tokens, accepted = verify(draft.numpy(), target.nan_to_num(0.0), drafter, accept_u.numpy(), sample_u.numpy(),
                                  [draft.shape[1]])
        return torch.from_numpy(tokens), torch.from_numpy(accepted)

    monkeypatch.setattr(ops, "verify_drafts", on_host)
    cache, calls = PagedKVCache(1, 1, 64, max_length=64, page_size=16, device="cpu"), []

    def model(input_ids, past_key_values, logits_to_keep, **_):
        assert int(input_ids.min()) >= 0
        past_key_values.extend([input_ids.shape[1]])
        logits = torch.zeros(1, logits_to_keep, 11)
        if len(calls) == bad_call:
            logits[:] = float("nan")
        calls.append(input_ids)
        return types.SimpleNamespace(logits=logits)

    with pytest.raises(RuntimeError, match="no mass"):
        paged_speculative_generate(model, input_ids=torch.tensor([[3, 4, 5]]), max_length=20, cache=cache, temperature=1.0)
    assert len(calls) == bad_call + 1


def test_idle_sequences_do_not_count_in_the_bounds(monkeypatch) -> None:
    """The bounds choose kernels and workspace: one long idle sequence must not make a short step dear."""
    from faquant_b200 import ops
    from faquant_b200.kv_cache import PagedKVCache

    given = []
    monkeypatch.setattr(ops, "hif4_paged_attention", lambda q, *_, **kw: given.append(kw) or q)
    cache = PagedKVCache(1, 1, 64, max_sequences=3, max_length=4096, page_size=64, device="cpu")
    for counts, bounds in (([4000, 0, 0], (4000, 4000, 4000)), ([0, 30, 7], (30, 30, 37)), ([0, 1, 0], (1, 31, 31)),
                           ([1, 0, 1], (1, 4001, 4009)), ([0, 0, 0], (0, 0, 0))):
        cache.extend(counts)
        cache.attend(0, torch.zeros(sum(counts), 2, 64, dtype=torch.bfloat16))
        assert tuple(given[-1][n] for n in ("max_new", "max_len", "total_len")) == bounds
