"""Quantized prefill, then BF16 greedy decode: the generation loop of the reference's
LongBench evaluation (``eval_longbench._prefill_quant_decode_bf16_generate``,
src/faquant/workflows/eval_longbench.py:495-576).

The prompt runs through the HiF4 model -- in chunks when the model carries
``_faquant_prefill_chunk_tokens`` (a multiple of the attention's 256-query tile keeps every
attention tile and every token-local quantizer exactly as in one pass; the attention
backend of this package runs chunked prefill bit-identically) -- keeping only the last
position's logits. The first token is the argmax of those logits; the K/V QDQ copies
kept for quantized decode appends (``faquant_k_matmul_qdq_cache`` /
``faquant_v_matmul_qdq_cache`` on each attention module) are then released, and the
remaining tokens come greedily from the BF16 model stored as
``_faquant_bf16_decode_model``, which continues on the same K/V cache.

Only batch 1, greedy, one beam, as in the reference; the others raise ``ValueError``.
Both models follow the Hugging Face calling convention (keyword ``input_ids``,
``past_key_values``, ``cache_position``, ``use_cache``, ``return_dict``; the prefill model
also ``logits_to_keep``) and return an object with ``logits`` and ``past_key_values``.

:func:`paged_speculative_generate` is this package's own loop on a paged HiF4 K/V cache: chunked
prompt, drafted tokens verified several per step, greedy or sampled.
"""

from __future__ import annotations

import torch


def _stopped(stopping_criteria, sequence: torch.Tensor, scores: torch.Tensor) -> bool:
    """eval_longbench.py:495-501: a criteria object may answer with a tensor (all rows
    must agree to stop) or a plain bool."""
    if stopping_criteria is None:
        return False
    verdict = stopping_criteria(sequence, scores)
    if isinstance(verdict, torch.Tensor):
        return bool(verdict.all().item())
    return bool(verdict)


def _eos_ids(model, generation_kwargs: dict) -> set[int]:
    eos = generation_kwargs.get("eos_token_id", model.generation_config.eos_token_id)
    if eos is None:
        return set()
    return {int(eos)} if isinstance(eos, int) else {int(token) for token in eos}


def release_decode_qdq_caches(model) -> None:
    """Drop every attention module's K/V HiF4 append cache (only quantized decode
    appends use them; BF16 decode would otherwise hold a second K/V cache)."""
    for layer in model.model.layers:
        layer.self_attn.faquant_k_matmul_qdq_cache = None
        layer.self_attn.faquant_v_matmul_qdq_cache = None


@torch.inference_mode()
def prefill_quant_decode_bf16_generate(
    model,
    *,
    input_ids: torch.Tensor,
    max_length: int,
    stopping_criteria=None,
    **generation_kwargs,
) -> torch.Tensor:
    """``input_ids [1, S]`` -> ``[1, S + generated]`` (see the module docstring)."""
    if input_ids.shape[0] != 1:
        raise ValueError("prefill-only quantization requires batch size 1")
    if generation_kwargs.get("do_sample", False):
        raise ValueError("prefill-only quantization currently supports greedy decode")
    if int(generation_kwargs.get("num_beams", 1)) != 1:
        raise ValueError("prefill-only quantization currently supports one beam")

    decode_model = model.__dict__["_faquant_bf16_decode_model"]
    length = input_ids.shape[-1]
    chunk = int(model.__dict__.get("_faquant_prefill_chunk_tokens") or length)
    device = input_ids.device

    cache, outputs = None, None
    for begin in range(0, length, chunk):
        end = min(begin + chunk, length)
        outputs = model(input_ids=input_ids[:, begin:end], past_key_values=cache,
                        cache_position=torch.arange(begin, end, device=device), use_cache=True,
                        return_dict=True, logits_to_keep=1)
        cache = outputs.past_key_values
    release_decode_qdq_caches(model)

    scores = outputs.logits[:, -1, :]
    next_token = scores.argmax(dim=-1, keepdim=True)
    sequence = torch.cat((input_ids, next_token), dim=-1)
    eos_ids = _eos_ids(model, generation_kwargs)
    while sequence.shape[-1] < max_length:
        if int(next_token.item()) in eos_ids or _stopped(stopping_criteria, sequence, scores):
            break
        position = torch.tensor([cache.get_seq_length()], device=device, dtype=torch.long)
        outputs = decode_model(input_ids=next_token, past_key_values=cache, cache_position=position,
                               use_cache=True, return_dict=True)
        cache = outputs.past_key_values
        scores = outputs.logits[:, -1, :]
        next_token = scores.argmax(dim=-1, keepdim=True)
        sequence = torch.cat((sequence, next_token), dim=-1)
    return sequence


def lookup_drafts(tokens: list[int], count: int, ngram: int) -> list[int]:
    """Up to ``count`` tokens that followed the latest earlier occurrence of the last ``ngram``
    (or fewer, down to 1) tokens: drafts without a draft model."""
    for size in range(min(ngram, len(tokens) - 1), 0, -1):
        tail = tokens[-size:]
        for at in range(len(tokens) - size - 1, -1, -1):
            if tokens[at : at + size] == tail:
                return tokens[at + size : at + size + count]
    return []


def _target_probs(logits: torch.Tensor, temperature: float) -> torch.Tensor:
    """fp32 probabilities of ``logits [B, n, V]``; temperature 0 is the argmax with probability 1."""
    if temperature > 0:
        return torch.softmax(logits.float() / temperature, dim=-1)
    best = logits.argmax(dim=-1, keepdim=True)
    return torch.zeros(logits.shape, dtype=torch.float32, device=logits.device).scatter_(-1, best, 1.0)


@torch.inference_mode()
def paged_speculative_generate(
    model,
    *,
    input_ids: torch.Tensor,
    max_length: int,
    cache=None,
    num_drafts: int = 4,
    ngram: int = 3,
    temperature: float = 0.0,
    chunk: int = 2048,
    generator: torch.Generator | None = None,
    eos_token_id: int | list[int] | None = None,
) -> tuple[torch.Tensor, dict[str, int]]:
    """Generate on a paged HiF4 K/V cache with drafted tokens: ``input_ids [1, S]`` -> ``([1, S +
    generated], {"steps", "drafted", "accepted"})``.

    The prompt goes through the model in chunks of ``chunk`` tokens; then every step runs the
    last token and up to ``num_drafts`` looked-up drafts (:func:`lookup_drafts`) in one
    forward call, verifies the drafts against the model's probabilities
    (``ops.verify_drafts``) and takes the rejected ones' keys and values back. The result is
    distributed as sampling token by token at ``temperature`` (0: greedy). ``model`` is a
    Hugging Face causal LM whose attention modules run ``qwen3.attention_forward`` with
    ``faquant_attention_kernel = "paged"``; no counterpart in the reference, whose loop decodes
    single tokens (``eval_longbench.py:495-576``)."""
    from . import ops
    from .kv_cache import PagedKVCache

    if input_ids.dim() != 2 or input_ids.shape[0] != 1 or input_ids.shape[1] < 1:
        raise ValueError("paged generation takes one prompt: input_ids [1, S]")
    if num_drafts < 0 or ngram < 1 or chunk < 1 or temperature < 0:
        raise ValueError("num_drafts and temperature must not be negative, ngram and chunk must be positive")
    device, length = input_ids.device, input_ids.shape[1]
    if max_length <= length:
        return input_ids, {"steps": 0, "drafted": 0, "accepted": 0}
    if cache is None:
        cache = PagedKVCache.for_model(model, max_length=max_length + num_drafts, device=device)
    eos = set() if eos_token_id is None else {eos_token_id} if isinstance(eos_token_id, int) else set(eos_token_id)

    def forward(ids: torch.Tensor, keep: int) -> torch.Tensor:
        begin = cache.lengths[0]
        position = torch.arange(begin, begin + ids.shape[1], device=device)
        return model(input_ids=ids, past_key_values=cache, position_ids=position[None], cache_position=position,
                     use_cache=True, return_dict=True, logits_to_keep=keep).logits

    def verify(drafts: list[int], logits: torch.Tensor) -> tuple[list[int], int]:
        u = torch.rand(1, len(drafts) + 1, generator=generator, device=device)
        tokens, accepted = ops.verify_drafts(torch.tensor([drafts], dtype=torch.int64, device=device).reshape(1, -1),
                                             _target_probs(logits, temperature), None, u[:, :-1], u[:, -1].contiguous())
        n = int(accepted.item())
        new = tokens[0, : n + 1].tolist()
        if new[-1] < 0:  # no token to go on with: the embedding must not see it
            raise RuntimeError("the model's probabilities of the next token have no mass (NaN logits?)")
        return new, n

    for begin in range(0, length, chunk):
        logits = forward(input_ids[:, begin : min(begin + chunk, length)], 1)
    tokens = input_ids[0].tolist()
    new, _ = verify([], logits)
    stats = {"steps": 0, "drafted": 0, "accepted": 0}
    while True:
        for i, token in enumerate(new):
            tokens.append(token)
            if token in eos or len(tokens) >= max_length:
                return torch.tensor([tokens], dtype=input_ids.dtype, device=device), stats
        drafts = lookup_drafts(tokens, min(num_drafts, max_length - len(tokens) - 1), ngram)
        known = cache.lengths[0]
        logits = forward(torch.tensor([tokens[-1:] + drafts], dtype=input_ids.dtype, device=device), len(drafts) + 1)
        new, accepted = verify(drafts, logits)
        cache.truncate([known + 1 + accepted])
        stats["steps"] += 1
        stats["drafted"] += len(drafts)
        stats["accepted"] += accepted
