"""PagedKVCache's append and its sparse attention: ragged steps against 64-bit references, taken-back
tokens, and a small random Hugging Face Qwen3 on it."""

from __future__ import annotations

import pytest
import torch

import sparse_reference as ref
from paged_reference import attention, quantized
from test_gpu_paged_generate import _logits, _model, _prompt
from test_gpu_sparse import BOUND, _no_status, _randn, _tables

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


class _Held:
    """The keys and values of a cache's sequences, kept beside it."""

    def __init__(self, batch, h, d):
        self.rows = [[torch.zeros(0, h, d) for _ in range(batch)] for _ in range(2)]

    def add(self, counts, *kv):
        for packed, t in zip(self.rows, kv):
            for b, part in enumerate(t.float().cpu().split(counts)):
                packed[b] = torch.cat((packed[b], part))

    def truncate(self, lengths):
        self.rows = [[x[:n] for x, n in zip(packed, lengths)] for packed in self.rows]

    def packed(self):
        return [torch.cat(packed) for packed in self.rows]


@pytest.mark.parametrize("d", [64, 128])
def test_ragged_steps_attend_to_the_selected_pages(d) -> None:
    from faquant_b200.kv_cache import PagedKVCache

    h, heads, page, count = 2, 8, 16, 6
    cache = PagedKVCache(1, h, d, max_sequences=4, max_length=700, page_size=page, device=DEV, sparse_pages=count,
                         sparse_first=1, sparse_last=2)
    held = _Held(4, h, d)
    steps = [[500, 0, 40, 17], [1, 30, 1, 0], [5, 1, 4, 1], [1, 1, 1, 1], [1, 0, 0, 0]]
    for i, counts in enumerate(steps):
        n = sum(counts)
        q, k, v = (_randn(n, x, d, seed=100 + 3 * i + j) for j, x in enumerate((heads, h, h)))
        cache.extend(counts)
        cache.write(0, k, v)
        out = cache.attend(0, q)
        held.add(counts, k, v)
        keys, values = held.packed()
        lists, _ = ref.select(q, keys, cache.lengths, counts, page, count, 1, 2)
        want, size = ref.attention(q, quantized(keys), quantized(values), cache.lengths, counts, page, lists)
        assert bool(((out.double().cpu() - want).abs() <= BOUND * size + 2.0**-126).all()), i
        if i == 2:  # drafts taken back, in the middle of pages
            lengths = [a - min(2, c) for a, c in zip(cache.lengths, counts)]
            cache.truncate(lengths)
            held.truncate(lengths)
    _no_status()


def test_short_contexts_and_prompts_are_dense() -> None:
    """No context longer than the pages taken, or a chunk beyond sparse_max_new: the dense kernels' bits."""
    from faquant_b200.kv_cache import PagedKVCache

    def run(**kw):
        cache = PagedKVCache(1, 2, 128, max_sequences=2, max_length=400, page_size=16, device=DEV, **kw)
        out = []
        for i, counts in enumerate([[100, 60], [1, 1], [200, 1], [3, 1]]):
            n = sum(counts)
            cache.extend(counts)
            q, k, v = (_randn(n, x, 128, seed=120 + 3 * i + j) for j, x in enumerate((8, 2, 2)))
            cache.write(0, k, v)
            out.append(cache.attend(0, q))
        return out

    dense, short, prompts = run(), run(sparse_pages=7), run(sparse_pages=7, sparse_max_new=2)
    assert torch.equal(dense[0], short[0]) and torch.equal(dense[1], short[1])  # 101 tokens are seven pages
    assert not torch.equal(dense[2], short[2]) and not torch.equal(dense[3], short[3])
    assert all(torch.equal(a, b) for a, b in zip(dense, prompts))
    assert torch.equal(run(sparse_pages=25)[3], dense[3])
    _no_status()


def test_append_and_attend_over_layers() -> None:
    """Projections to attention in two layers with their own weights, in a prompt and decode steps."""
    from faquant_b200.kv_cache import PagedKVCache

    h, heads, d, layers = 2, 4, 64, 2
    cache = PagedKVCache(layers, h, d, max_sequences=2, max_length=300, page_size=32, device=DEV, sparse_pages=4)
    held = [_Held(2, h, d) for _ in range(layers)]
    cos, sin = _tables(300, d)
    weights = [[(1 + 0.2 * _randn(d, seed=140 + 2 * x + i, dtype=torch.float32)).to(torch.bfloat16) for i in range(2)]
               for x in range(layers)]
    for i, counts in enumerate([[200, 20], [1, 1], [4, 0]]):
        cache.extend(counts)
        n = sum(counts)
        pos = torch.tensor([p for _, p in ref.positions(cache.lengths, counts)])
        for layer in range(layers):
            q, k, v = (_randn(n, x, d, seed=150 + 10 * i + 3 * layer + j) for j, x in enumerate((heads, h, h)))
            turned = cache.append(layer, q, k, v, cos=cos, sin=sin, q_norm=weights[layer][0], k_norm=weights[layer][1],
                                  rotate=True)
            kw = dict(cos=cos, sin=sin, rotate=True)
            want_q = ref.turned(q, pos, norm=weights[layer][0], **kw)
            bound = 2.0**-8 * want_q.abs() + 2.0**-18 * want_q.norm(dim=-1, keepdim=True)
            assert bool(((turned.double().cpu() - want_q).abs() <= bound).all())
            held[layer].add(counts, ref.turned(k, pos, norm=weights[layer][1], **kw).float(), v)
            keys, values = held[layer].packed()
            out = cache.attend(layer, turned)
            lists, _ = ref.select(turned, keys, cache.lengths, counts, 32, 4, 1, 2)
            want, size = ref.attention(turned, quantized(keys), quantized(values), cache.lengths, counts, 32, lists)
            assert bool(((out.double().cpu() - want).abs() <= BOUND * size + 2.0**-126).all())
    with pytest.raises(ValueError, match="new tokens"):
        cache.append(0, *(torch.zeros(2, x, d, dtype=torch.bfloat16, device=DEV) for x in (heads, h, h)))
    _no_status()


@torch.inference_mode()
def test_a_model_on_a_sparse_cache() -> None:
    from faquant_b200.generate import paged_speculative_generate
    from faquant_b200.kv_cache import PagedKVCache

    model, ids = _model("paged"), _prompt(300)
    kw = dict(max_length=400, page_size=16, device=DEV)
    chunks = [250, 1, 1, 8, 40]
    dense = _logits(model, ids, PagedKVCache.for_model(model, **kw), chunks)
    # prompts dense: the first chunk's bits
    some = _logits(model, ids, PagedKVCache.for_model(model, sparse_pages=8, sparse_max_new=16, **kw), chunks)
    assert torch.equal(some[:, :250], dense[:, :250]) and bool(some.isfinite().all())
    # 18 of at most 19 pages: near the dense model
    most = _logits(model, ids, PagedKVCache.for_model(model, sparse_pages=18, **kw), chunks)
    assert torch.equal(most[:, :250], dense[:, :250]) and float((most - dense).norm() / dense.norm()) < 0.2
    cache = PagedKVCache.for_model(model, sparse_pages=6, **kw)
    out, stats = paged_speculative_generate(model, input_ids=ids[:, :200], max_length=240, cache=cache, num_drafts=3, chunk=64)
    assert out.shape == (1, 240) and torch.equal(out[:, :200], ids[:, :200]) and stats["steps"] >= 10
    _no_status()
