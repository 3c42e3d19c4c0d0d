"""The paged HiF4 K/V cache under a small random Hugging Face Qwen3: chunked prompts, drafted
tokens verified and taken back, hand-off of the cache in bf16."""

from __future__ import annotations

import types

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def _model(kernel: str):
    from transformers import Qwen3Config, Qwen3ForCausalLM

    from faquant_b200.attention import B200_ATTENTION_IMPLEMENTATION, register_simulated_attention_backend
    from faquant_b200.qwen3 import attention_forward

    register_simulated_attention_backend()
    cfg = Qwen3Config(vocab_size=512, hidden_size=256, intermediate_size=512, num_hidden_layers=2,
                      num_attention_heads=4, num_key_value_heads=2, head_dim=128, max_position_embeddings=4096,
                      tie_word_embeddings=False)
    torch.manual_seed(0)
    model = Qwen3ForCausalLM(cfg).to(device=DEV, dtype=torch.bfloat16).eval()
    model.set_attn_implementation(B200_ATTENTION_IMPLEMENTATION)
    for layer in model.model.layers:
        attn = layer.self_attn
        attn.faquant_attention_kernel = kernel
        attn.faquant_qk_rotation = True
        attn.forward = types.MethodType(attention_forward, attn)
    return model


def _prompt(n, seed=1):
    # a repeated phrase, so that looked-up drafts have something to find
    g = torch.Generator().manual_seed(seed)
    phrase = torch.randint(0, 512, (40,), generator=g)
    return phrase.repeat(-(-n // 40))[:n][None].to(DEV)


@torch.inference_mode()
def _logits(model, ids, cache, chunks):
    out, begin = [], 0
    for n in chunks:
        position = torch.arange(begin, begin + n, device=DEV)
        out.append(model(input_ids=ids[:, begin : begin + n], past_key_values=cache, position_ids=position[None],
                         cache_position=position, use_cache=True, return_dict=True).logits)
        begin += n
    return torch.cat(out, 1).float()


@torch.inference_mode()
def test_chunks_steps_and_one_pass_agree() -> None:
    """Whatever the chunks, the same cache and nearly the same logits (bf16 roundings apart: two
    layers of a few roundings of 2^-8 each); and near the unquantized model's."""
    from faquant_b200.kv_cache import PagedKVCache

    model, ids = _model("paged"), _prompt(300)
    caches = [PagedKVCache.for_model(model, max_length=400, page_size=ps, device=DEV) for ps in (64, 16)]
    one = _logits(model, ids, caches[0], [300])
    some = _logits(model, ids, caches[1], [1, 150, 33, 1, 1, 8, 106])
    assert float((one - some).norm() / one.norm()) < 2e-2
    for layer in range(2):
        (ka, va), (kb, vb) = caches[0].read(layer), caches[1].read(layer)
        assert ka.shape == (300, 2, 128)
        for a, b in ((ka, kb), (va, vb)):  # projections of other batch sizes: a rounding may move a code
            assert float((a - b).float().norm() / a.float().norm()) < 5e-2
    plain = _model("native")
    plain.set_attn_implementation("eager")
    ref = plain(input_ids=ids).logits.float()
    assert float((one - ref).norm() / ref.norm()) < 0.2  # HiF4 keys and values


@torch.inference_mode()
@pytest.mark.parametrize("drafts", [0, 4, 7])
def test_greedy_generation_takes_the_models_best_tokens(drafts) -> None:
    """Every generated token is, given the ones before it, the best of a one-pass run up to
    the roundings that differ between the runs."""
    from faquant_b200.generate import paged_speculative_generate
    from faquant_b200.kv_cache import PagedKVCache

    model, ids = _model("paged"), _prompt(150)
    cache = PagedKVCache.for_model(model, max_length=230, page_size=16, device=DEV)
    out, stats = paged_speculative_generate(model, input_ids=ids, max_length=200, cache=cache, num_drafts=drafts, chunk=64)
    assert out.shape == (1, 200) and torch.equal(out[:, :150], ids)
    assert stats["accepted"] <= stats["drafted"] <= drafts * stats["steps"]
    assert cache.lengths[0] in range(199, 200 + drafts) and stats["steps"] >= 49 // (drafts + 1)
    if drafts == 0:
        assert stats == {"steps": 49, "drafted": 0, "accepted": 0}
    logits = _logits(model, out, PagedKVCache.for_model(model, max_length=256, device=DEV), [200])[0, 149:199]
    best = logits.max(-1).values
    chosen = logits.gather(-1, out[0, 150:, None])[:, 0]
    assert bool((best - chosen <= 0.05 * logits.std()).all())


@torch.inference_mode()
def test_sampled_generation_repeats_with_its_seed_and_ends_at_eos() -> None:
    from faquant_b200.generate import paged_speculative_generate

    model, ids = _model("paged"), _prompt(90)
    runs = [paged_speculative_generate(model, input_ids=ids, max_length=140, temperature=0.8,
                                       generator=torch.Generator(DEV).manual_seed(7))[0] for _ in range(2)]
    assert torch.equal(*runs) and runs[0].shape == (1, 140)
    eos = int(runs[0][0, 100])
    first = (runs[0][0, 90:] == eos).nonzero()[0].item() + 90
    out, _ = paged_speculative_generate(model, input_ids=ids, max_length=140, temperature=0.8, eos_token_id=eos,
                                        generator=torch.Generator(DEV).manual_seed(7))
    assert torch.equal(out, runs[0][:, : first + 1])


def test_ragged_sequences_pages_and_refusals() -> None:
    from faquant_b200.kv_cache import PagedKVCache

    cache = PagedKVCache(1, 2, 64, max_sequences=3, max_length=100, num_pages=9, page_size=16, device=DEV)
    g = torch.Generator().manual_seed(3)

    def step(counts):
        cache.extend(counts)
        t = sum(counts)
        k, v = (torch.randn(t, 2, 64, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2))
        cache.write(0, k, v)
        return k, v, cache.attend(0, torch.randn(t, 4, 64, generator=g).to(torch.bfloat16).to(DEV))

    k, v, out = step([40, 0, 17])
    assert out.shape == (57, 4, 64) and cache.lengths == [40, 0, 17]
    before = cache.read(0)[0]
    k2, _, _ = step([1, 20, 0])
    cache.truncate([40, 0, 17])  # the step is taken back
    assert torch.equal(cache.read(0)[0], before)
    with pytest.raises(RuntimeError, match="no step"):
        cache.write(0, k, v)
    with pytest.raises(RuntimeError, match="exhausted"):
        cache.extend([60, 64, 0])
    assert cache.lengths == [40, 0, 17]
    with pytest.raises(ValueError, match="max_length"):
        cache.extend([61, 0, 0])
    with pytest.raises(ValueError):
        cache.extend([1, 1])
    with pytest.raises(ValueError):
        cache.truncate([41, 0, 0])
    with pytest.raises(ValueError, match="different lengths"):
        cache.get_seq_length()
    step([8, 64, 0])  # all nine pages
    cache.truncate([0, 0, 0])
    assert sorted(cache._free) == list(range(9))


@pytest.mark.parametrize("new", [[0, 1, 0], [0, 40, 2], [0, 200, 1], [1, 0, 70]])
def test_a_step_beside_a_long_idle_sequence(new) -> None:
    """Bounds of the sequences that take part only, on every kernel, against a 64-bit softmax."""
    from faquant_b200.kv_cache import PagedKVCache
    from paged_reference import attention, quantized

    held = [6000, 90, 300]
    cache = PagedKVCache(1, 2, 64, max_sequences=3, max_length=8192, page_size=32, device=DEV)
    g = torch.Generator().manual_seed(4)
    rows = [[torch.empty(0, 2, 64)] * 3 for _ in range(2)]

    def step(counts):
        cache.extend(counts)
        kv = [torch.randn(sum(counts), 2, 64, generator=g).to(torch.bfloat16) for _ in range(2)]
        for packed, t in zip(rows, kv):
            for b, part in enumerate(t.split(counts)):
                packed[b] = torch.cat((packed[b], part.float()))
        cache.write(0, *(t.to(DEV) for t in kv))
        q = torch.randn(sum(counts), 8, 64, generator=g).to(torch.bfloat16)
        return q, cache.attend(0, q.to(DEV))

    step(held)
    q, out = step(new)
    ref, size = attention(q, *(quantized(torch.cat(packed)) for packed in rows), cache.lengths, new)
    bound = 2.0**-7 + 2.0**-12  # P and O rounded to bf16, the scores' fp32 sums
    assert bool(((out.double().cpu() - ref).abs() <= bound * size + 2.0**-126).all())
