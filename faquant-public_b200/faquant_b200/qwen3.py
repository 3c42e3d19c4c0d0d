"""Qwen3 attention adapter on B200: the post-RoPE Q/K transform and the patched forward.

Mirrors ``qwen3._attention_forward`` (``src/faquant/qwen3.py:56-172``) with the same
``module.faquant_*`` attribute contract (installed by the reference's
``install_qwen3_attention_adapter :175-279`` and ``apply_qwen3_qk_smooth_scales
:282-346``): q/k/v projections, q_norm/k_norm, RoPE, then one fp32 excursion for
``k - offset``, Smooth-QK ``q * s`` / ``k / s`` and the Hadamard over head_dim with a
single bf16 rounding -- here one K4 launch per operand -- then the HiF4 attention
backend (``faquant_b200.attention``) and ``o_proj``. With ``faquant_attention_kernel =
"paged"`` and a :class:`~faquant_b200.kv_cache.PagedKVCache` as ``past_key_values`` the keys and
values go to HiF4 pages instead and the paged attention runs on them: K and V are quantized, Q and
P are not, whatever ``faquant_qk_matmul_quant`` and ``faquant_pv_matmul_quant`` say of
those; a recipe that asks for other keys or values raises.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import ops
from .attention import _hif4_kwargs, simulated_flash_attention_forward
from .kv_cache import PagedKVCache


def qk_pretransform(module, query_states: torch.Tensor, key_states: torch.Tensor):
    """Post-RoPE Q/K transform of ``qwen3.py:92-130`` on ``[B, H, S, D]`` tensors."""
    smooth = getattr(module, "faquant_qk_smooth_scale", None)
    delta = getattr(module, "faquant_qk_smooth_delta", None)
    if delta is not None:
        if smooth is None:
            raise RuntimeError("Smooth-QK delta requires a frozen base scale")
        smooth = smooth * delta.float().exp()
    offset = getattr(module, "faquant_qk_key_offset", None)
    rotate = bool(getattr(module, "faquant_qk_rotation", False))
    if smooth is None and offset is None and not rotate:
        return query_states, key_states
    head_dim = query_states.shape[-1]
    block = getattr(module, "faquant_qk_rotation_block_size", None)
    if rotate and block not in (None, head_dim):
        raise NotImplementedError("a block Hadamard narrower than head_dim is not implemented by faquant_b200")
    if query_states.dtype != torch.bfloat16 or key_states.dtype != torch.bfloat16:
        raise NotImplementedError("the fused Q/K transform rounds to bf16; bf16 Q/K are required")
    if offset is not None:
        offset = offset.reshape(key_states.shape[1], head_dim)
    q, _, _ = ops.qk_prep(query_states, levels=None, rotate=rotate, smooth_scale=smooth,
                          smooth_mode=None if smooth is None else "mul")
    k, _, _ = ops.qk_prep(key_states, levels=None, rotate=rotate, smooth_scale=smooth,
                          smooth_mode=None if smooth is None else "div", key_offset=offset)
    return q, k


def attention_forward(
    self,
    hidden_states: torch.Tensor,
    position_embeddings: tuple[torch.Tensor, torch.Tensor],
    attention_mask: Optional[torch.Tensor],
    past_key_values=None,
    cache_position: Optional[torch.LongTensor] = None,
    **kwargs,
):
    """Drop-in for ``Qwen3Attention.forward`` as patched by the reference (``qwen3.py:56-172``)."""
    from transformers.models.qwen3.modeling_qwen3 import apply_rotary_pos_emb

    legacy = kwargs.pop("past_key_value", None)
    if past_key_values is None:
        past_key_values = legacy
    input_shape = hidden_states.shape[:-1]
    hidden_shape = (*input_shape, -1, self.head_dim)
    query_states = self.q_norm(self.q_proj(hidden_states).view(hidden_shape)).transpose(1, 2)
    key_states = self.k_norm(self.k_proj(hidden_states).view(hidden_shape)).transpose(1, 2)
    value_states = self.v_proj(hidden_states).view(hidden_shape).transpose(1, 2)
    cos, sin = position_embeddings
    query_states, key_states = apply_rotary_pos_emb(query_states, key_states, cos, sin)
    query_states, key_states = qk_pretransform(self, query_states, key_states)
    if getattr(self, "faquant_attention_input_quant", False):
        quant_kwargs = self.faquant_core_quant_kwargs
        if quant_kwargs.get("quant_format") != "hif4":
            raise NotImplementedError("faquant_b200 implements HiF4 attention-input quantization only")
        query_states = ops.qk_prep(query_states, levels=ops.default_levels("act"), rotate=False)[0]
        key_states = ops.qk_prep(key_states, levels=ops.default_levels("act"), rotate=False)[0]
        value_states = ops.qk_prep(value_states, levels=ops.default_levels("act"), rotate=False)[0]
    kernel = getattr(self, "faquant_attention_kernel", "simulated")
    if kernel == "paged":  # write to the HiF4 pages, attend over them (Q and P not quantized)
        if not isinstance(past_key_values, PagedKVCache):
            raise ValueError('faquant_attention_kernel "paged" needs a PagedKVCache as past_key_values')
        _refuse_unpaged(self, attention_mask, kwargs)
        attn_output = past_key_values.forward(self.layer_idx, query_states, key_states, value_states, self.scaling)
        return _project(self, attn_output, input_shape), None
    if past_key_values is not None:
        cache_kwargs = {"sin": sin, "cos": cos, "cache_position": cache_position}
        key_states, value_states = past_key_values.update(key_states, value_states, self.layer_idx, cache_kwargs)
    if kernel == "simulated":  # the HiF4 attention of this package
        kwargs["cache_position"] = cache_position
        interface = simulated_flash_attention_forward
    elif kernel == "native":  # the model's own attention on the transformed Q/K (qwen3.py:147-152)
        from transformers.modeling_utils import ALL_ATTENTION_FUNCTIONS
        from transformers.models.qwen3.modeling_qwen3 import eager_attention_forward

        impl = self.config._attn_implementation
        interface = eager_attention_forward if impl == "eager" else ALL_ATTENTION_FUNCTIONS[impl]
    else:
        raise NotImplementedError("the differentiable (training) attention kernel is not part of faquant_b200")
    attn_output, attn_weights = interface(
        self, query_states, key_states, value_states, attention_mask, dropout=0.0, scaling=self.scaling,
        sliding_window=getattr(self, "sliding_window", None), **kwargs)
    return _project(self, attn_output, input_shape), attn_weights


def _refuse_unpaged(module, attention_mask, kwargs) -> None:
    """What the paged attention does not do -- it is causal over each sequence's whole cache -- is
    refused, as ``simulated_flash_attention_forward`` refuses what it does not do."""
    if attention_mask is not None:
        raise NotImplementedError("attention masks are not implemented by the paged attention of faquant_b200")
    if getattr(module, "sliding_window", None) is not None or kwargs.get("sliding_window") is not None:
        raise NotImplementedError("sliding windows are not implemented by the paged attention of faquant_b200")
    if any(kwargs.get(n) is not None for n in ("cu_seq_lens_q", "cu_seq_lens_k", "max_length_q", "max_length_k")):
        raise NotImplementedError("packed cu_seqlens are not supported: give each sequence its place in the PagedKVCache")
    if kwargs.get("softcap") is not None:
        raise NotImplementedError("softcap is not implemented by faquant_b200")
    requested = kwargs.get("is_causal")
    if not (getattr(module, "is_causal", True) if requested is None else requested):
        raise NotImplementedError("the paged attention of faquant_b200 is causal")
    shared = getattr(module, "faquant_matmul_quant_kwargs", None)
    for operand, what in (("qk", "QK operands"), ("pv", "PV operands")):
        if not getattr(module, f"faquant_{operand}_matmul_quant", True):
            raise NotImplementedError(f"{what}: the paged cache holds HiF4 keys and values only")
        _hif4_kwargs(getattr(module, f"faquant_{operand}_matmul_quant_kwargs", shared), what)
    if kwargs.get("dropout"):
        raise ValueError("the paged attention only supports dropout=0 inference")
    if kwargs.get("output_attentions", False):
        raise ValueError("the paged attention does not materialize attention weights")


def _project(module, attn_output: torch.Tensor, input_shape) -> torch.Tensor:
    """The output projection, with its input quantized first where the adapter asks for it."""
    attn_output = attn_output.reshape(*input_shape, -1).contiguous()
    if getattr(module, "faquant_attention_output_quant", False) and not getattr(module.o_proj, "faquant_quantizes_input", False):
        attn_output = ops.hif4_quantize(attn_output, levels=ops.default_levels("act"))[0]
    return module.o_proj(attn_output)
