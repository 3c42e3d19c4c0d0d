"""Tensor-level entry points over the C ABI (device tensors in, device tensors out).

Each function validates its torch arguments, allocates the outputs with torch
(the library itself never allocates) and launches on the current CUDA stream.
"""

from __future__ import annotations

import functools
import os

import torch

from . import _lib

LEVELS = {"123": 123, "12": 12, "13": 13}


def levels_code(levels: str | int) -> int:
    key = str(levels)
    if key not in LEVELS:
        raise ValueError(f"HiF4 levels must be one of {tuple(LEVELS)}, got {levels!r}")
    return LEVELS[key]


def default_levels(kind: str) -> str:
    """The reference's process-wide level variants (``src/faquant/hif4.py:13-43``).

    ``kind`` is ``weight``, ``act`` or one of the attention operands ``q``, ``k``,
    ``p``, ``v``. Read from the same environment variables, at call time.
    """
    weight = os.environ.get("FAQUANT_HIF4_SCALE_LEVELS", "123")
    act = os.environ.get("FAQUANT_HIF4_ACT_SCALE_LEVELS", weight)
    attn = os.environ.get("FAQUANT_HIF4_ATTN_SCALE_LEVELS", act)
    if kind == "weight":
        value = weight
    elif kind == "act":
        value = act
    elif kind in ("q", "k", "p", "v"):
        value = attn
        for entry in filter(None, os.environ.get("FAQUANT_HIF4_ATTN_OPERAND_LEVELS", "").split(",")):
            operand, _, val = entry.partition("=")
            if operand == kind:
                value = val
    else:
        raise ValueError(f"unknown HiF4 operand kind {kind!r}")
    levels_code(value)
    return value


def _dtype_code(t: torch.Tensor) -> int:
    if t.dtype == torch.bfloat16:
        return _lib.FAQ_BF16
    if t.dtype == torch.float32:
        return _lib.FAQ_F32
    raise TypeError(f"unsupported dtype {t.dtype}; the HiF4 kernels take bfloat16 or float32")


def _require_cuda(*tensors: torch.Tensor | None) -> torch.device:
    device = None
    index = -1
    for t in tensors:
        if t is None:
            continue
        at = t.get_device()  # -1 for a host tensor
        if at < 0:
            raise RuntimeError("faquant_b200 operators run on CUDA tensors only (no CPU fallback)")
        if device is None:
            device, index = t.device, at
        elif at != index:
            raise RuntimeError("all tensors must be on the same CUDA device")
    if device is None:
        raise RuntimeError("no CUDA tensor given")
    return device


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


# the current stream's handle without making a Stream object (2 us less per call), where torch has it
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(device: torch.device) -> int:
    if _raw_stream is not None and device.index is not None:
        return _raw_stream(device.index)
    return torch.cuda.current_stream(device).cuda_stream


def _rows_view(x: torch.Tensor) -> tuple[torch.Tensor, int]:
    """``x [..., k]`` as a 2-D row view and its row stride (copies only when needed)."""
    k = x.shape[-1]
    if x.dim() == 2 and x.stride(1) == 1 and x.stride(0) >= k:
        return x, x.stride(0)
    return x.contiguous().reshape(-1, k), k


def hif4_quantize(
    x: torch.Tensor,
    *,
    levels: str | int = "123",
    input_scale: torch.Tensor | None = None,
    signs: torch.Tensor | None = None,
    permutation: torch.Tensor | None = None,
    rot_block: int | None = None,
    want_qdq: bool = True,
    want_codes: bool = False,
) -> tuple[torch.Tensor | None, torch.Tensor | None, torch.Tensor | None]:
    """Rotation (optional) + HiF4 quantization of ``x [..., k]`` along the last axis.

    Returns ``(qdq, codes, meta)``: the dequantized values in ``x.dtype`` (shape of
    ``x``) and the packed codes ``uint8 [rows, k64/2]`` / meta ``int32 [rows, k64/64]``.
    """
    device = _require_cuda(x, input_scale, signs, permutation)
    if x.shape[-1] == 0:
        raise ValueError("HiF4 does not support an empty axis")
    k = x.shape[-1]
    rows, ldx = _rows_view(x)
    n = rows.shape[0]
    k64 = (k + 63) // 64 * 64
    qdq = torch.empty((n, k), dtype=x.dtype, device=device) if want_qdq else None
    codes = torch.empty((n, k64 // 2), dtype=torch.uint8, device=device) if want_codes else None
    meta = torch.empty((n, k64 // 64), dtype=torch.int32, device=device) if want_codes else None
    if input_scale is not None:
        input_scale = input_scale.to(device=device, dtype=x.dtype).contiguous()
        if input_scale.numel() != k:
            raise ValueError("input_scale must have one entry per input channel")
    if signs is not None:
        signs = signs.to(device=device, dtype=torch.int8).contiguous()
        if permutation is not None:
            permutation = permutation.to(device=device, dtype=torch.int64).contiguous()
    block = 0 if rot_block is None else int(rot_block)
    _lib.call(
        "faq_hif4_quantize", rows.data_ptr(), _dtype_code(x), n, k, ldx, _ptr(input_scale), _ptr(signs),
        _ptr(permutation), block, levels_code(levels), _ptr(codes), _ptr(meta), _ptr(qdq), k, _stream(device),
    )
    if qdq is not None:
        qdq = qdq.reshape(x.shape)
    return qdq, codes, meta


ACTIVATIONS = {"swiglu": 1, "gelu_tanh": 2}  # FAQ_ACT_SWIGLU, FAQ_ACT_GELU_TANH


def hif4_quantize_act(
    x: torch.Tensor,
    act: str,
    *,
    levels: str | int = "123",
    input_scale: torch.Tensor | None = None,
    signs: torch.Tensor,
    rot_block: int,
    want_qdq: bool = True,
    want_codes: bool = False,
) -> tuple[torch.Tensor | None, torch.Tensor | None, torch.Tensor | None]:
    """:func:`hif4_quantize` of an activation's output, the activation fused into the load
    (``faq_hif4_quantize_act``): ``act="swiglu"`` takes the gate|up tensor ``x [rows, 2k]``
    and quantizes ``silu_mul(x)``; ``act="gelu_tanh"`` takes ``x [rows, k]`` and quantizes
    ``gelu_tanh(x)`` -- the same outputs as the activation followed by
    :func:`hif4_quantize`, without the activation's tensor. bf16, signs-only rotation
    (block 8..256); returns ``(qdq [rows, k], codes, meta)``."""
    if act not in ACTIVATIONS:
        raise ValueError(f"act must be one of {sorted(ACTIVATIONS)}")
    device = _require_cuda(x, input_scale, signs)
    if x.dtype != torch.bfloat16 or x.dim() != 2:
        raise TypeError("hif4_quantize_act takes a rank-2 bfloat16 tensor")
    rows = x.shape[0]
    k = x.shape[1] // 2 if act == "swiglu" else x.shape[1]
    if act == "swiglu" and x.shape[1] % 2:
        raise ValueError("the SwiGLU input holds gate and up halves: an even width")
    if x.stride(-1) != 1 or (rows > 1 and x.stride(0) % 8) or x.data_ptr() % 16:
        x = x.contiguous()
    ldx = x.stride(0) if rows > 1 else x.shape[1]
    qdq = torch.empty((rows, k), dtype=torch.bfloat16, device=device) if want_qdq else None
    codes = torch.empty((rows, k // 2), dtype=torch.uint8, device=device) if want_codes else None
    meta = torch.empty((rows, k // 64), dtype=torch.int32, device=device) if want_codes else None
    if input_scale is not None:
        input_scale = input_scale.to(device=device, dtype=torch.bfloat16).contiguous()
    signs = signs.to(device=device, dtype=torch.int8).contiguous()
    _lib.call("faq_hif4_quantize_act", x.data_ptr(), ACTIVATIONS[act], rows, k, ldx, _ptr(input_scale),
              signs.data_ptr(), int(rot_block), levels_code(levels), _ptr(codes), _ptr(meta), _ptr(qdq), k,
              _stream(device))
    return qdq, codes, meta


def rms_norm_quantize_supported(k: int, rot_block: int | None) -> bool:
    """Whether :func:`hif4_quantize_rms_norm` takes a row of ``k`` channels rotated in
    blocks of ``rot_block`` (the K1 v4 shapes: k % 1024 == 0, k <= 16384, 32..1024)."""
    return (rot_block is not None and k % 1024 == 0 and k <= 16384 and 32 <= rot_block <= 1024
            and rot_block & (rot_block - 1) == 0)


def hif4_quantize_rms_norm(
    x: torch.Tensor,
    norm_weight: torch.Tensor | None,
    eps: float,
    *,
    levels: str | int = "123",
    input_scale: torch.Tensor | None = None,
    signs: torch.Tensor,
    permutation: torch.Tensor | None = None,
    rot_block: int,
    want_meta: bool = False,
    want_qdq: bool = True,
    codes_out: torch.Tensor | None = None,
) -> tuple[torch.Tensor | None, torch.Tensor | None]:
    """:func:`hif4_quantize` of ``rms_norm(x, norm_weight, eps)`` in one pass
    (``faq_hif4_quantize_rms_norm``): the same bits as :func:`rms_norm` followed by
    :func:`hif4_quantize`, without the normalized tensor in memory. bf16 ``x [rows, k]``
    with ``rms_norm_quantize_supported(k, rot_block)``; returns ``(qdq, meta)``
    (``qdq`` None with ``want_qdq=False``). ``codes_out`` (``uint8 [rows, k/2]``,
    contiguous) receives the packed codes as well. ``norm_weight=None`` takes the
    affine-free LayerNorm instead (``faq_hif4_quantize_layer_norm``, the bits of
    :func:`layer_norm` then :func:`hif4_quantize`)."""
    device = _require_cuda(x, norm_weight, input_scale, signs, permutation)
    if x.dtype != torch.bfloat16 or x.dim() != 2:
        raise TypeError("hif4_quantize_rms_norm takes a rank-2 bfloat16 tensor")
    rows, k = x.shape
    if x.stride(-1) != 1 or (rows > 1 and x.stride(0) % 8) or x.data_ptr() % 16:
        x = x.contiguous()
    ldx = x.stride(0) if rows > 1 else k
    qdq = torch.empty((rows, k), dtype=torch.bfloat16, device=device) if want_qdq else None
    meta = torch.empty((rows, k // 64), dtype=torch.int32, device=device) if want_meta else None
    if codes_out is not None:
        if (codes_out.dtype != torch.uint8 or tuple(codes_out.shape) != (rows, k // 2)
                or not codes_out.is_contiguous() or codes_out.device != device):
            raise ValueError("codes_out must be a contiguous uint8 [rows, k/2] tensor on x's device")
    elif not want_qdq:
        raise ValueError("nothing to write: want_qdq=False without codes_out")
    if input_scale is not None:
        input_scale = input_scale.to(device=device, dtype=torch.bfloat16).contiguous()
    signs = signs.to(device=device, dtype=torch.int8).contiguous()
    if permutation is not None:
        permutation = permutation.to(device=device, dtype=torch.int64).contiguous()
    tail = (_ptr(input_scale), signs.data_ptr(), _ptr(permutation), int(rot_block), levels_code(levels),
            _ptr(codes_out), _ptr(meta), _ptr(qdq), k, _stream(device))
    if norm_weight is None:
        _lib.call("faq_hif4_quantize_layer_norm", x.data_ptr(), rows, k, ldx, float(eps), *tail)
    else:
        norm_weight = norm_weight.to(device=device, dtype=torch.bfloat16).contiguous()
        _lib.call("faq_hif4_quantize_rms_norm", x.data_ptr(), rows, k, ldx, norm_weight.data_ptr(), float(eps), *tail)
    return qdq, meta


def hif4_dequantize(codes: torch.Tensor, meta: torch.Tensor, k: int, dtype: torch.dtype = torch.bfloat16,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """Packed HiF4 ``codes [rows, k64/2]`` / ``meta [rows, k64/64]`` -> values ``[rows, k]``
    (into ``out`` when given: any row stride, unit column stride)."""
    device = _require_cuda(codes, meta, out)
    rows = codes.shape[0]
    if out is None:
        out = torch.empty((rows, k), dtype=dtype, device=device)
    elif out.shape != (rows, k) or out.stride(-1) != 1 or out.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError("out must be a bf16/fp32 [rows, k] tensor with unit column stride")
    ldo = out.stride(0) if rows > 1 else k
    _lib.call("faq_hif4_dequantize", codes.contiguous().data_ptr(), meta.contiguous().data_ptr(), rows, k,
              out.data_ptr(), _dtype_code(out), ldo, _stream(device))
    return out


def hif4_pack_weight(
    weight: torch.Tensor,
    *,
    levels: str | int = "123",
    scale: torch.Tensor | None = None,
    lv2: torch.Tensor | None = None,
    lv3: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor, int]:
    """Pack an ``[n, k]`` HiF4-grid weight; returns ``(codes, meta, mismatches)``."""
    device = _require_cuda(weight)
    n, k = weight.shape
    k64 = (k + 63) // 64 * 64
    w = weight if weight.stride(-1) == 1 else weight.contiguous()
    codes = torch.empty((n, k64 // 2), dtype=torch.uint8, device=device)
    meta = torch.empty((n, k64 // 64), dtype=torch.int32, device=device)
    counter = torch.zeros(1, dtype=torch.int64, device=device)
    if scale is not None:
        scale = scale.to(device=device, dtype=torch.float32).reshape(n, k // 64).contiguous()
        lv2 = lv2.to(device=device, dtype=torch.int8).reshape(n, k // 64, 8).contiguous()
        lv3 = lv3.to(device=device, dtype=torch.int8).reshape(n, k // 64, 16).contiguous()
    _lib.call("faq_hif4_pack_weight", w.data_ptr(), _dtype_code(w), n, k, w.stride(0), _ptr(scale), _ptr(lv2),
              _ptr(lv3), levels_code(levels), codes.data_ptr(), meta.data_ptr(), counter.data_ptr(), _stream(device))
    return codes, meta, int(counter.item())


def set_gemm_sm_target(sms: int) -> None:
    """Size the persistent GEMMs' grids for ``sms`` SMs from the next launch on (0: every
    SM; ``faq_set_gemm_sm_target``): leaves SMs free for collectives that run beside them."""
    _lib.call("faq_set_gemm_sm_target", int(sms))


def gemm_bf16(a: torch.Tensor, b: torch.Tensor, bias: torch.Tensor | None = None,
              out: torch.Tensor | None = None, residual: torch.Tensor | None = None) -> torch.Tensor:
    """``a [m, k] @ b [n, k]^T (+ bias)`` in bf16 with fp32 accumulation (tcgen05); with
    ``residual [m, n]`` (bf16) the result is ``residual + that`` with the eager bf16 add's
    rounding (the product rounded to bf16 first), added in the GEMM's epilogue."""
    device = _require_cuda(a, b, bias, residual)
    if a.dtype != torch.bfloat16 or b.dtype != torch.bfloat16:
        raise TypeError("gemm_bf16 takes bfloat16 operands")
    if a.stride(-1) != 1:
        a = a.contiguous()
    if b.stride(-1) != 1:
        b = b.contiguous()
    m, k = a.shape
    n = b.shape[0]
    if b.shape[1] != k:
        raise ValueError("inner dimensions differ")
    lda = a.stride(0) if m > 1 else k
    ldb = b.stride(0) if n > 1 else k
    if k % 8 or lda % 8 or ldb % 8 or a.data_ptr() % 16 or b.data_ptr() % 16:
        # TMA wants 16-byte aligned rows: pad k with zeros, which adds nothing to the sums
        k8 = (k + 7) // 8 * 8
        a = torch.nn.functional.pad(a, (0, k8 - k))
        b = torch.nn.functional.pad(b, (0, k8 - k))
        k, lda, ldb = k8, k8, k8
    if bias is not None:
        bias = bias.to(device=device, dtype=torch.bfloat16).contiguous()
    if out is None:
        out = torch.empty((m, n), dtype=torch.bfloat16, device=device)
    if residual is None:
        _lib.call("faq_gemm_bf16_tn", a.data_ptr(), lda, b.data_ptr(), ldb, m, n, k, _ptr(bias), out.data_ptr(),
                  out.stride(0) if m > 1 else n, _stream(device))
        return out
    if residual.dtype != torch.bfloat16 or residual.shape != (m, n):
        raise ValueError("residual must be bfloat16 [m, n]")
    if residual.stride(-1) != 1:
        residual = residual.contiguous()
    _lib.call("faq_gemm_bf16_tn_residual", a.data_ptr(), lda, b.data_ptr(), ldb, m, n, k, _ptr(bias),
              residual.data_ptr(), residual.stride(0) if m > 1 else n, out.data_ptr(),
              out.stride(0) if m > 1 else n, _stream(device))
    return out


def w4a4_gemm(a: torch.Tensor | tuple[torch.Tensor, torch.Tensor], b_codes: torch.Tensor, b_meta: torch.Tensor,
              bias: torch.Tensor | None = None, out: torch.Tensor | None = None,
              residual: torch.Tensor | None = None) -> torch.Tensor:
    """The W4A4 GEMM on a packed HiF4 weight ``(b_codes uint8 [n, k/2], b_meta int32
    [n, k/64])``: ``deq(a) @ deq(b)^T (+ bias) (+ residual)`` in bf16, bit-identical to
    ``gemm_bf16`` on the dequantized operands. ``a`` is the activation's packed form
    ``(codes, meta)`` (``hif4_quantize(..., want_codes=True)``) or its bf16 QDQ ``[m, k]``;
    a bf16 ``a`` of at most 16 rows runs the small-row kernel, whose sums run in another
    order (the same values up to fp32 rounding of the accumulation). ``k`` must be a
    multiple of 256 (``NotImplementedError`` otherwise)."""
    device = _require_cuda(b_codes, b_meta, bias, residual)
    if b_codes.dtype != torch.uint8 or b_meta.dtype not in (torch.int32, torch.uint32):
        raise TypeError("packed weight: codes uint8 [n, k/2], meta int32 [n, k/64]")
    n = b_codes.shape[0]
    k = b_codes.shape[1] * 2
    if b_meta.shape != (n, k // 64):
        raise ValueError("packed weight: meta must be [n, k/64]")
    b_codes, b_meta = b_codes.contiguous(), b_meta.contiguous()
    packed_a = isinstance(a, tuple)
    if packed_a:
        a_codes, a_meta = (t.contiguous() for t in a)
        _require_cuda(a_codes, a_meta)
        m = a_codes.shape[0]
        if a_codes.dtype != torch.uint8 or a_codes.shape[1] * 2 != k or a_meta.shape != (m, k // 64):
            raise ValueError("packed activation: codes uint8 [m, k/2] and meta [m, k/64] with the weight's k")
    else:
        _require_cuda(a)
        if a.dtype != torch.bfloat16 or a.shape[-1] != k:
            raise ValueError("the QDQ activation must be bfloat16 [m, k] with the weight's k")
        if a.stride(-1) != 1 or a.stride(0) % 8 or a.data_ptr() % 16:
            a = a.contiguous()
        m = a.shape[0]
    if bias is not None:
        bias = bias.to(device=device, dtype=torch.bfloat16).contiguous()
    if out is None:
        out = torch.empty((m, n), dtype=torch.bfloat16, device=device)
    ldr = 0
    if residual is not None:
        if residual.dtype != torch.bfloat16 or residual.shape != (m, n):
            raise ValueError("residual must be bfloat16 [m, n]")
        if residual.stride(-1) != 1:
            residual = residual.contiguous()
        ldr = residual.stride(0) if m > 1 else n
    ldy = out.stride(0) if m > 1 else n
    if packed_a:
        _lib.call("faq_w4a4_gemm", a_codes.data_ptr(), a_meta.data_ptr(), b_codes.data_ptr(), b_meta.data_ptr(),
                  m, n, k, _ptr(bias), _ptr(residual), ldr, out.data_ptr(), ldy, _stream(device))
    else:
        lda = a.stride(0) if m > 1 else k
        _lib.call("faq_w4a4_gemm_qdq_a", a.data_ptr(), lda, b_codes.data_ptr(), b_meta.data_ptr(), m, n, k,
                  _ptr(bias), _ptr(residual), ldr, out.data_ptr(), ldy, _stream(device))
    return out


def selftest_wait_timeout(limit_ns: int) -> None:
    device = torch.device("cuda", torch.cuda.current_device())
    _lib.call("faq_selftest_wait_timeout", int(limit_ns), _stream(device))


def qk_prep(
    x: torch.Tensor,
    *,
    levels: str | int | None = "123",
    rotate: bool = True,
    smooth_scale: torch.Tensor | None = None,
    smooth_mode: str | None = None,
    key_offset: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
    want_codes: bool = False,
) -> tuple[torch.Tensor, torch.Tensor | None, torch.Tensor | None]:
    """Attention operand preparation of ``x [B, H, S, D]`` (any strides, D contiguous).

    ``smooth_mode`` is ``"mul"`` (Q), ``"div"`` (K) or None; ``smooth_scale`` is
    ``[D]`` or ``[H, D]``; ``key_offset`` is ``[H, D]`` (K only). Returns the bf16
    operand ``[B, H, S, D]`` (``out`` if given) and optional packed codes/meta.
    """
    device = _require_cuda(x, smooth_scale, key_offset)
    if x.dim() != 4:
        raise ValueError("qk_prep expects [batch, heads, seq, head_dim]")
    b, h, s, d = x.shape
    if x.stride(-1) != 1:
        x = x.contiguous()
    if out is None:
        out = torch.empty((b, h, s, d), dtype=torch.bfloat16, device=device)
    mode = {None: 0, "mul": 1, "div": 2}[smooth_mode]
    head_stride = 0
    if smooth_scale is not None:
        smooth_scale = smooth_scale.to(device=device, dtype=torch.float32).contiguous()
        head_stride = d if smooth_scale.dim() == 2 else 0
    if key_offset is not None:
        key_offset = key_offset.to(device=device, dtype=torch.float32).reshape(h, d).contiguous()
    lv = 0 if levels is None else levels_code(levels)
    codes = meta = None
    if want_codes and lv:
        codes = torch.empty((b * h * s, d // 2), dtype=torch.uint8, device=device)
        meta = torch.empty((b * h * s, d // 64), dtype=torch.int32, device=device)
    _lib.call("faq_qk_prep", x.data_ptr(), _dtype_code(x), b, h, s, d, x.stride(0), x.stride(1), x.stride(2),
              _ptr(key_offset), _ptr(smooth_scale), head_stride, mode, int(rotate), lv, out.data_ptr(),
              out.stride(0), out.stride(1), out.stride(2), _ptr(codes), _ptr(meta), _stream(device))
    return out, codes, meta


def qk_norm_rope_prep(
    x: torch.Tensor,
    *,
    norm_weight: torch.Tensor | None,
    eps: float = 1e-6,
    cos: torch.Tensor | None = None,
    sin: torch.Tensor | None = None,
    levels: str | int | None = "123",
    rotate: bool = True,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Qwen3 attention operand in one pass: per-head RMSNorm (``norm_weight [D]`` bf16),
    RoPE (bf16 ``cos``/``sin`` ``[S, D]``, position = sequence index), Hadamard over D,
    bf16, HiF4. ``x [B, H, S, D]`` bf16, any strides with D contiguous."""
    device = _require_cuda(x, norm_weight, cos, sin)
    if x.dim() != 4 or x.dtype != torch.bfloat16:
        raise ValueError("qk_norm_rope_prep expects bf16 [batch, heads, seq, head_dim]")
    b, h, s, d = x.shape
    if x.stride(-1) != 1:
        x = x.contiguous()
    if out is None:
        out = torch.empty((b, h, s, d), dtype=torch.bfloat16, device=device)
    if norm_weight is not None:
        norm_weight = norm_weight.to(device=device, dtype=torch.bfloat16).contiguous()
    rope_ld = 0
    if cos is not None:
        cos = cos.to(device=device, dtype=torch.bfloat16).contiguous()
        sin = sin.to(device=device, dtype=torch.bfloat16).contiguous()
        if cos.shape[0] < s or cos.shape[-1] != d:
            raise ValueError("cos/sin must be [>= seq, head_dim]")
        rope_ld = cos.stride(0)
    lv = 0 if levels is None else levels_code(levels)
    _lib.call("faq_qk_norm_rope_prep", x.data_ptr(), _dtype_code(x), b, h, s, d, x.stride(0), x.stride(1),
              x.stride(2), _ptr(norm_weight), float(eps), _ptr(cos), _ptr(sin), rope_ld, None, None, 0, 0,
              int(rotate), lv, out.data_ptr(), out.stride(0), out.stride(1), out.stride(2), None, None,
              _stream(device))
    return out


def wan_qk_prep(
    x: torch.Tensor,
    head_sumsq: torch.Tensor,
    norm_weight: torch.Tensor,
    *,
    head_offset: int = 0,
    eps: float = 1e-6,
    cos: torch.Tensor | None = None,
    sin: torch.Tensor | None = None,
    smooth_scale: torch.Tensor | None = None,
    smooth_mode: str | None = None,
    levels: str | int | None = "123",
    rotate: bool = True,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Wan2.2 self-attention operand in one pass: WanRMSNorm over each token's whole row
    of all heads, the 3-D RoPE (fp64 ``cos``/``sin`` ``[S, D/2]``), optional Smooth-QK,
    Hadamard over D, bf16, HiF4. ``x [B, H, S, D]`` bf16, any strides with D contiguous.

    ``head_sumsq [ranks, B*S, C]`` fp32 holds per-head sums of squares (``row_sumsq``
    with one segment per head; ``ranks`` > 1 when gathered from a head-sharded layer):
    this tensor's heads of rank r are columns ``head_offset .. head_offset + H`` of
    block r, so the norm runs over ``ranks * H`` heads. ``norm_weight [H, D]`` or
    ``[H*D]`` is this shard's weight."""
    device = _require_cuda(x, head_sumsq, norm_weight, cos, sin, smooth_scale)
    if x.dim() != 4 or x.dtype != torch.bfloat16:
        raise ValueError("wan_qk_prep expects bf16 [batch, heads, seq, head_dim]")
    b, h, s, d = x.shape
    if x.stride(-1) != 1:
        x = x.contiguous()
    if out is None:
        out = torch.empty((b, h, s, d), dtype=torch.bfloat16, device=device)
    if head_sumsq.dtype != torch.float32 or head_sumsq.dim() != 3 or not head_sumsq.is_contiguous():
        raise TypeError("head_sumsq must be a contiguous fp32 [ranks, batch * seq, columns] tensor")
    ranks, tokens, cols = head_sumsq.shape
    if tokens != b * s or head_offset < 0 or head_offset + h > cols:
        raise ValueError("head_sumsq does not cover these heads and tokens")
    norm_weight = norm_weight.to(device=device, dtype=torch.float32).reshape(h, d).contiguous()
    if cos is not None:
        cos = cos.to(device=device, dtype=torch.float64).contiguous()
        sin = sin.to(device=device, dtype=torch.float64).contiguous()
        if cos.shape != (s, d // 2) or sin.shape != (s, d // 2):
            raise ValueError("cos/sin must be [seq, head_dim / 2]")
    mode = {None: 0, "mul": 1, "div": 2}[smooth_mode]
    head_stride = 0
    if smooth_scale is not None:
        smooth_scale = smooth_scale.to(device=device, dtype=torch.float32).contiguous()
        head_stride = d if smooth_scale.dim() == 2 else 0
    lv = 0 if levels is None else levels_code(levels)
    _lib.call("faq_wan_qk_prep", x.data_ptr(), b, h, s, d, x.stride(0), x.stride(1), x.stride(2),
              head_sumsq.data_ptr() + 4 * head_offset, ranks * h, h, cols, tokens * cols, norm_weight.data_ptr(),
              float(eps), _ptr(cos), _ptr(sin),
              _ptr(smooth_scale), head_stride, mode, int(rotate), lv, out.data_ptr(), out.stride(0), out.stride(1),
              out.stride(2), _stream(device))
    return out


def row_sumsq(x: torch.Tensor, segments: int = 1, out: torch.Tensor | None = None) -> torch.Tensor:
    """fp32 ``[rows, segments]`` sums of squares of the ``segments`` equal column blocks
    of bf16 ``x [rows, cols]`` (a column slice of a wider tensor is fine)."""
    device = _require_cuda(x)
    if x.dtype != torch.bfloat16 or x.dim() != 2 or x.stride(1) != 1:
        raise TypeError("row_sumsq takes a bf16 [rows, cols] tensor with contiguous rows")
    rows, cols = x.shape
    if cols % segments:
        raise ValueError("cols must divide into the segments")
    if out is None:
        out = torch.empty((rows, segments), dtype=torch.float32, device=device)
    _lib.call("faq_row_sumsq", x.data_ptr(), rows, segments, cols // segments, x.stride(0) if rows > 1 else cols,
              out.data_ptr(), _stream(device))
    return out


def layer_norm(x: torch.Tensor, eps: float, out: torch.Tensor | None = None) -> torch.Tensor:
    """LayerNorm without affine of bf16 ``x [..., k]`` (fp32 statistics), one pass."""
    device = _require_cuda(x)
    if x.dtype != torch.bfloat16:
        raise TypeError("layer_norm takes bfloat16")
    rows, ldx = _rows_view(x)
    k = x.shape[-1]
    if out is None:
        out = torch.empty(x.shape, dtype=torch.bfloat16, device=device)
    _lib.call("faq_layer_norm", rows.data_ptr(), rows.shape[0], k, ldx, float(eps), out.data_ptr(), k,
              _stream(device))
    return out


def gelu_tanh(x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """GELU (tanh approximation) of a bf16 ``[rows, cols]`` tensor, one pass."""
    device = _require_cuda(x)
    if x.dtype != torch.bfloat16 or x.dim() != 2 or x.stride(1) != 1:
        raise TypeError("gelu_tanh takes a bf16 [rows, cols] tensor with contiguous rows")
    rows, cols = x.shape
    if out is None:
        out = torch.empty((rows, cols), dtype=torch.bfloat16, device=device)
    _lib.call("faq_gelu_tanh", x.data_ptr(), rows, cols, x.stride(0) if rows > 1 else cols, out.data_ptr(),
              out.stride(0) if rows > 1 else cols, _stream(device))
    return out


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float, out: torch.Tensor | None = None) -> torch.Tensor:
    """Qwen3RMSNorm of bf16 ``x [..., k]`` in one pass."""
    device = _require_cuda(x, weight)
    if x.dtype != torch.bfloat16:
        raise TypeError("rms_norm takes bfloat16")
    rows, ldx = _rows_view(x)
    k = x.shape[-1]
    if out is None:
        out = torch.empty(x.shape, dtype=torch.bfloat16, device=device)
    weight = weight.to(device=device, dtype=torch.bfloat16).contiguous()
    _lib.call("faq_rms_norm", rows.data_ptr(), rows.shape[0], k, ldx, weight.data_ptr(), float(eps), out.data_ptr(),
              k, _stream(device))
    return out


def silu_mul(gate_up: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """``silu(gate) * up`` of a bf16 ``[rows, 2f]`` gate|up tensor, one pass."""
    device = _require_cuda(gate_up)
    if gate_up.dtype != torch.bfloat16 or gate_up.dim() != 2 or gate_up.stride(1) != 1:
        raise TypeError("silu_mul takes a bf16 [rows, 2f] tensor with contiguous rows")
    rows, two_f = gate_up.shape
    f = two_f // 2
    if out is None:
        out = torch.empty((rows, f), dtype=torch.bfloat16, device=device)
    _lib.call("faq_silu_mul", gate_up.data_ptr(), rows, f, gate_up.stride(0), out.data_ptr(), out.stride(0),
              _stream(device))
    return out


def hif4_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    *,
    scale: float | None = None,
    causal: bool = True,
    p_levels: str | int | None = "123",
    quantized_normalizer: bool = True,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """HiF4 QK/PV attention of pre-quantized bf16 operands.

    ``q [B, Hq, Sq, 128]``, ``k/v [B, Hkv, Sk, 128]`` (any strides with the head dim
    contiguous); returns ``[B, Sq, Hq, 128]`` bf16 (``out`` if given).
    """
    device = _require_cuda(q, k, v)
    for t in (q, k, v):
        if t.dtype != torch.bfloat16 or t.dim() != 4:
            raise TypeError("hif4_attention takes rank-4 bfloat16 Q/K/V")
    b, hq, sq, d = q.shape
    _, hkv, sk, _ = k.shape
    if v.shape != k.shape:
        raise ValueError("K and V shapes differ")

    def fix(t: torch.Tensor) -> torch.Tensor:
        ok = t.stride(-1) == 1 and all(st % 8 == 0 for st in t.stride()[:-1]) and t.data_ptr() % 16 == 0
        return t if ok else t.contiguous()

    q, k, v = fix(q), fix(k), fix(v)
    if out is None:
        out = torch.empty((b, sq, hq, d), dtype=torch.bfloat16, device=device)
    scale = float(scale if scale is not None else d**-0.5)
    lv = 0 if p_levels is None else levels_code(p_levels)
    _lib.call("faq_hif4_attention", q.data_ptr(), k.data_ptr(), v.data_ptr(), b, hq, hkv, sq, sk, d,
              q.stride(0), q.stride(1), q.stride(2), k.stride(0), k.stride(1), k.stride(2),
              v.stride(0), v.stride(1), v.stride(2), scale, int(causal), lv, int(quantized_normalizer),
              out.data_ptr(), out.stride(0), out.stride(1), out.stride(2), _stream(device))
    return out


def hif4_decode_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    *,
    scale: float | None = None,
    p_levels: str | int | None = "123",
    quantized_normalizer: bool = True,
    out: torch.Tensor | None = None,
    workspace: torch.Tensor | None = None,
) -> torch.Tensor:
    """Decode-step HiF4 attention: ``q [B, Hq, Sq, 128]`` (the last Sq positions, Sq small)
    against ``k/v [B, Hkv, Sk, 128]`` (the whole cache), pre-quantized bf16 operands;
    returns ``[B, Sq, Hq, 128]``. Same semantics as :func:`hif4_attention` with causal
    masking; the keys are split over the GPU (exact running max per tile)."""
    device = _require_cuda(q, k, v)
    for t in (q, k, v):
        if t.dtype != torch.bfloat16 or t.dim() != 4:
            raise TypeError("hif4_decode_attention takes rank-4 bfloat16 Q/K/V")
    b, hq, sq, d = q.shape
    _, hkv, sk, _ = k.shape
    if v.shape != k.shape:
        raise ValueError("K and V shapes differ")
    def fix(t: torch.Tensor) -> torch.Tensor:
        ok = t.stride(-1) == 1 and all(st % 8 == 0 for st in t.stride()[:-1]) and t.data_ptr() % 16 == 0
        return t if ok else t.contiguous()

    q, k, v = fix(q), fix(k), fix(v)
    need = int(_lib.load().faq_hif4_decode_workspace_bytes(b, hq, hkv, sq, sk, d))
    if need == 0:
        raise ValueError("unsupported decode shape")
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty(need, dtype=torch.uint8, device=device)
    if out is None:
        out = torch.empty((b, sq, hq, d), dtype=torch.bfloat16, device=device)
    scale = float(scale if scale is not None else d**-0.5)
    lv = 0 if p_levels is None else levels_code(p_levels)
    _lib.call("faq_hif4_decode_attention", q.data_ptr(), k.data_ptr(), v.data_ptr(), b, hq, hkv, sq, sk, d,
              q.stride(0), q.stride(1), q.stride(2), k.stride(0), k.stride(1), k.stride(2), v.stride(0), v.stride(1),
              v.stride(2), scale, lv, int(quantized_normalizer), out.data_ptr(), out.stride(0), out.stride(1),
              out.stride(2), workspace.data_ptr(), workspace.numel() * workspace.element_size(), _stream(device))
    return out


@functools.lru_cache(maxsize=64)
def hif4_page_bytes(kv_heads: int, head_dim: int, page_size: int) -> int:
    """Bytes of one page of the HiF4 K/V cache: K and V of ``page_size`` tokens, 4.625 bits
    per value (the page format is in ``include/faquant_b200.h``)."""
    if head_dim not in (64, 128) or page_size < 16 or page_size & (page_size - 1):
        raise ValueError("head_dim must be 64 or 128 and page_size a power of two from 16")
    return 2 * kv_heads * (page_size // 16) * 592 * (head_dim // 64)


def _ragged(pages: torch.Tensor, table: torch.Tensor, cu: torch.Tensor, lens: torch.Tensor, kv_heads: int,
            head_dim: int, page_size: int) -> tuple:
    """Checks of a pool and the arrays that describe a ragged batch on it. Returns the C
    calls' arguments for them: ``(pages, num_pages, page_stride, page_size)`` and ``(table, row
    stride, columns, cu, lens, batch)``."""
    size = hif4_page_bytes(kv_heads, head_dim, page_size)
    shape = pages.shape
    if pages.dtype is not torch.uint8 or len(shape) < 2:
        raise TypeError("pages must be a uint8 tensor [num_pages, ...]")
    if len(shape) == 4 and (shape[1] != 2 or shape[2] != kv_heads):
        raise ValueError("pages of four dimensions are [num_pages, 2, kv_heads, bytes]")
    if pages.is_contiguous():
        page_stride = size
        whole = pages.numel() == shape[0] * size
    else:
        stride = pages.stride()
        page_stride = stride[0] if shape[0] > 1 else size
        whole, inner = True, 1
        for n, st in zip(reversed(shape[1:]), reversed(stride[1:])):
            whole = whole and (st == inner or n == 1)
            inner *= n
        whole = whole and inner == size
    if not whole:
        raise ValueError("a page must be hif4_page_bytes(kv_heads, head_dim, page_size) contiguous bytes")
    return ((pages.data_ptr(), shape[0], page_stride, page_size), _batch(table, cu, lens))


def _batch(table: torch.Tensor, cu: torch.Tensor, lens: torch.Tensor) -> tuple:
    """Checks of the arrays that describe a ragged batch. Returns the C calls' ``(table, row
    stride, columns, cu, lens, batch)``."""
    int32 = torch.int32
    if table.dtype is not int32 or cu.dtype is not int32 or lens.dtype is not int32:
        raise TypeError("table, cu and lens must be int32")
    shape, rows = table.shape, lens.shape
    if len(rows) != 1 or len(shape) != 2 or shape[0] != rows[0] or cu.shape != (rows[0] + 1,):
        raise ValueError("table must be [batch, columns], cu [batch + 1] and lens [batch]")
    batch, columns = shape
    ld = columns
    if not table.is_contiguous():
        ld, unit = table.stride()
        if unit != 1 and columns > 1:
            raise ValueError("table must have unit column stride")
        if batch == 1:
            ld = columns  # a single row may have any stride
    if not (cu.is_contiguous() and lens.is_contiguous()):
        raise ValueError("cu and lens must be contiguous")
    return table.data_ptr(), ld, columns, cu.data_ptr(), lens.data_ptr(), batch


def _kv_heads(pages: torch.Tensor, head_dim: int, page_size: int) -> int:
    """The kv heads that a pool of such pages holds."""
    shape = pages.shape
    if len(shape) == 4:
        return shape[2]
    size = 1
    for n in shape[1:]:
        size *= n
    return max(1, size // hif4_page_bytes(1, head_dim, page_size))


@functools.lru_cache(maxsize=256)
def _attention_workspace(device: int, *sizes: int) -> int:
    with torch.cuda.device(device):
        return int(_lib.load().faq_hif4_paged_attention_workspace_bytes(*sizes))


def hif4_kv_write(
    k: torch.Tensor,
    v: torch.Tensor,
    pages: torch.Tensor,
    table: torch.Tensor,
    cu: torch.Tensor,
    lens: torch.Tensor,
    *,
    page_size: int,
    levels: tuple[str | int, str | int] = ("123", "123"),
) -> None:
    """Quantize the new tokens' ``k``/``v [T, Hkv, D]`` (bf16 or fp32, D 64 or 128, any token
    and head strides) to HiF4 and write them into their ``pages`` (uint8 ``[num_pages,
    ...]``, ``hif4_page_bytes`` each, ``faq_hif4_kv_write``).

    ``cu [B + 1]`` bounds each sequence's new tokens, ``lens [B]`` are the lengths that
    include them, ``table [B, columns]`` the sequences' pages (all int32, on the device):
    new token i of n goes to position ``lens - n + i``. ``levels`` are K's and V's."""
    device = _require_cuda(k, v, pages, table, cu, lens)
    if k.dim() != 3 or k.shape != v.shape or k.dtype != v.dtype:
        raise ValueError("k and v must be [tokens, kv_heads, head_dim] of one shape and dtype")
    total, h, d = k.shape
    pool, ragged = _ragged(pages, table, cu, lens, h, d, page_size)
    ks, vs = k.stride(), v.stride()
    if ks[2] != 1:
        k = k.contiguous()
        ks = k.stride()
    if vs[2] != 1:
        v = v.contiguous()
        vs = v.stride()
    _lib.call("faq_hif4_kv_write", k.data_ptr(), v.data_ptr(), _dtype_code(k), total, h, d, ks[0], ks[1], vs[0], vs[1],
              *pool, *ragged, levels_code(levels[0]), levels_code(levels[1]), _stream(device))


def hif4_kv_read(
    pages: torch.Tensor,
    table: torch.Tensor,
    cu: torch.Tensor,
    lens: torch.Tensor,
    *,
    page_size: int,
    head_dim: int,
    total: int,
    dtype: torch.dtype = torch.bfloat16,
    out: tuple[torch.Tensor, torch.Tensor] | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """The last ``cu[b + 1] - cu[b]`` cached tokens of every sequence, dequantized:
    ``(k, v)``, each ``[total, Hkv, D]`` bf16 or fp32 (``total = cu[-1]``, known on the host),
    packed in sequence order; ``out`` takes tensors of that shape with unit channel stride."""
    device = _require_cuda(pages, table, cu, lens, *(out or ()))
    h = _kv_heads(pages, head_dim, page_size)
    pool, ragged = _ragged(pages, table, cu, lens, h, head_dim, page_size)
    if total < 0:
        raise ValueError("total must not be negative")
    if out is None:
        k = pages.new_empty((total, h, head_dim), dtype=dtype)
        v = torch.empty_like(k)
        ks = vs = (h * head_dim, head_dim)
    else:
        k, v = out
        if (k.shape != (total, h, head_dim) or v.shape != k.shape or k.dtype != v.dtype or k.stride(2) != 1
                or v.stride(2) != 1):
            raise ValueError("out must be two [total, kv_heads, head_dim] tensors of one dtype with unit channel stride")
        ks, vs = k.stride(), v.stride()
    _lib.call("faq_hif4_kv_read", *pool, h, head_dim, *ragged, k.data_ptr(), v.data_ptr(), _dtype_code(k), total, ks[0],
              ks[1], vs[0], vs[1], _stream(device))
    return k, v


def hif4_paged_attention(
    q: torch.Tensor,
    pages: torch.Tensor,
    table: torch.Tensor,
    cu: torch.Tensor,
    lens: torch.Tensor,
    *,
    page_size: int,
    max_new: int,
    max_len: int | None = None,
    total_len: int | None = None,
    scale: float | None = None,
    out: torch.Tensor | None = None,
    workspace: torch.Tensor | None = None,
) -> torch.Tensor:
    """Attention of each sequence's new tokens over its HiF4 pages: ``q [T, H, D]`` bf16,
    returns ``[T, H, D]`` bf16 (``faq_hif4_paged_attention``). ``table``, ``cu`` and ``lens``
    as in :func:`hif4_kv_write`, which must have written the tokens before: new token i of
    n sees the keys ``0 .. lens - n + i``, query head h those of kv head ``h // (H / Hkv)``.

    ``max_new``, ``max_len`` (the table's capacity by default) and ``total_len`` (batch x
    ``max_len`` by default) bound the sequences' new tokens, their lengths and the sum of
    the lengths from above (sequences without a new token do not count); they are host numbers, so nothing is copied from the device, and
    with prompt chunks in the batch they size the workspace. ``workspace``: a 256-byte
    aligned device buffer to use instead of a new one."""
    device = _require_cuda(q, pages, table, cu, lens, out, workspace)
    if q.dtype is not torch.bfloat16 or q.dim() != 3:
        raise TypeError("q must be bfloat16 [tokens, heads, head_dim]")
    total, heads, d = q.shape
    h = _kv_heads(pages, d, page_size)
    pool, ragged = _ragged(pages, table, cu, lens, h, d, page_size)
    if heads % h:
        raise ValueError("query heads must be divisible by key/value heads")
    qs = q.stride()
    if qs[2] != 1 or qs[0] % 8 or qs[1] % 8 or qs[0] < 8 or qs[1] < 8 or q.data_ptr() % 16:
        q = q.contiguous()
        qs = (heads * d, d)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        os_ = (heads * d, d)
    else:
        if out.shape != q.shape or out.dtype is not torch.bfloat16 or out.stride(2) != 1:
            raise ValueError("out must be a bfloat16 tensor of q's shape with unit channel stride")
        os_ = out.stride()
    batch = ragged[5]
    if max_len is None:
        max_len = ragged[2] * page_size
    if total_len is None:
        total_len = batch * max_len
    need = _attention_workspace(device.index, total, heads, h, batch, max_new, max_len, total_len, d)
    if need and (workspace is None or workspace.numel() * workspace.element_size() < need):
        workspace = pages.new_empty(need)
    _lib.call("faq_hif4_paged_attention", q.data_ptr(), total, heads, qs[0], qs[1], *pool, h, d, *ragged, max_new, max_len,
              total_len, d**-0.5 if scale is None else float(scale), out.data_ptr(), os_[0], os_[1],
              workspace.data_ptr() if need else None, need, _stream(device))
    return out


_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _call_on(device: torch.device, name: str, *args) -> None:
    """A C call for ``device``'s tensors on its current stream, whichever device is the current one."""
    if device.index == _current_device():
        _lib.call(name, *args, _stream(device))
    else:
        with torch.cuda.device(device):
            _lib.call(name, *args, _stream(device))


def hif4_kv_append(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    pages: torch.Tensor,
    table: torch.Tensor,
    cu: torch.Tensor,
    lens: torch.Tensor,
    *,
    page_size: int,
    cos: torch.Tensor | None = None,
    sin: torch.Tensor | None = None,
    q_norm: torch.Tensor | None = None,
    k_norm: torch.Tensor | None = None,
    eps: float = 1e-6,
    rotate: bool = False,
    smooth_scale: torch.Tensor | None = None,
    key_offset: torch.Tensor | None = None,
    levels: tuple[str | int, str | int] = ("123", "123"),
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """From the projections' ``q [T, H, D]`` and ``k``/``v [T, Hkv, D]`` (bf16 or fp32, D 64 or 128, any token
    and head strides) to the cache and the attention's queries in one pass
    (``faq_hif4_kv_append``): per-head RMSNorm (``q_norm``/``k_norm [D]``), the rotation of each token's
    position, Smooth-QK (``q * smooth_scale``, ``(k - key_offset) / smooth_scale``, normal numbers; ``[D]`` or ``[Hkv, D]``, ``key_offset
    [Hkv, D]``), the Hadamard transform over D (``rotate``), each where given. K and V are quantized and written to
    their ``pages`` as :func:`hif4_kv_write` does (``table``, ``cu``, ``lens``, ``levels`` as there); the queries
    are returned in bf16 ``[T, H, D]`` (in ``out`` where given; it may be ``q`` itself).

    ``cos``/``sin [positions, D / 2]`` (or ``[positions, D]``, of which the first half is read; bf16 or fp32) hold
    a row per position: the first channel half a and the second b become ``a cos - b sin`` and ``b cos + a sin``.
    Nothing is rounded between the steps: q is computed in fp32, k in fp64 and rounded to fp32 for the fit, so
    a key's bits do not depend on the step in which it was written. A token without a place (a position below
    zero, or beyond the tables, which sets ``FAQ_STATUS_BAD_BOUND``) is not written, its row of q is zero;
    rows beyond ``cu[B]`` stay as they are."""
    device = _require_cuda(q, k, v, pages, table, cu, lens, cos, sin, q_norm, k_norm, smooth_scale, key_offset, out)
    qs, ks, dtype = q.shape, k.shape, q.dtype
    if len(qs) != 3 or len(ks) != 3 or v.shape != ks or qs[0] != ks[0] or qs[2] != ks[2]:
        raise ValueError("q must be [tokens, heads, head_dim], k and v [tokens, kv_heads, head_dim]")
    if k.dtype is not dtype or v.dtype is not dtype:
        raise TypeError("q, k and v must have one dtype")
    total, heads, d = qs
    h = ks[1]
    pool, ragged = _ragged(pages, table, cu, lens, h, d, page_size)
    if h == 0 or heads % h or heads == 0:
        raise ValueError("query heads must be divisible by key/value heads")
    q_st, k_st, v_st = q.stride(), k.stride(), v.stride()
    if q_st[2] != 1:
        q = q.contiguous()
        q_st = q.stride()
    if k_st[2] != 1:
        k = k.contiguous()
        k_st = k.stride()
    if v_st[2] != 1:
        v = v.contiguous()
        v_st = v.stride()
    q_norm_ptr = k_norm_ptr = cos_ptr = sin_ptr = smooth_ptr = offset_ptr = None
    norm_dtype = rope_dtype = _lib.FAQ_F32
    rope_ld = rope_rows = smooth_stride = 0
    if q_norm is not None or k_norm is not None:
        norm_type = (k_norm if q_norm is None else q_norm).dtype
        for n in (q_norm, k_norm):
            if n is not None and (n.shape != (d,) or n.dtype is not norm_type):
                raise ValueError("q_norm and k_norm must be [head_dim] tensors of one dtype")
        norm_dtype = _dtype_code(k_norm if q_norm is None else q_norm)
        if q_norm is not None:
            q_norm = q_norm.contiguous()
            q_norm_ptr = q_norm.data_ptr()
        if k_norm is not None:
            k_norm = k_norm.contiguous()
            k_norm_ptr = k_norm.data_ptr()
    if cos is not None and sin is not None:
        shape = cos.shape
        if len(shape) != 2 or sin.shape != shape or shape[1] not in (d // 2, d) or sin.dtype is not cos.dtype:
            raise ValueError("cos and sin must be [positions, head_dim / 2] or [positions, head_dim], of one dtype")
        if not (cos.is_contiguous() and sin.is_contiguous()):
            cos, sin = cos.contiguous(), sin.contiguous()
        rope_rows, rope_ld = shape
        rope_dtype, cos_ptr, sin_ptr = _dtype_code(cos), cos.data_ptr(), sin.data_ptr()
    elif cos is not None or sin is not None:
        raise ValueError("cos and sin go together")
    if smooth_scale is not None:
        if smooth_scale.shape not in ((d,), (h, d)):
            raise ValueError("smooth_scale must be [head_dim] or [kv_heads, head_dim]")
        smooth_stride = d if smooth_scale.dim() == 2 else 0
        smooth_scale = smooth_scale.to(torch.float32).contiguous()
        smooth_ptr = smooth_scale.data_ptr()
    if key_offset is not None:
        if key_offset.shape != (h, d):
            raise ValueError("key_offset must be [kv_heads, head_dim]")
        key_offset = key_offset.to(torch.float32).contiguous()
        offset_ptr = key_offset.data_ptr()
    if out is None:
        # of a contiguous tensor the like is made sooner
        out = torch.empty_like(q) if dtype is torch.bfloat16 and q.is_contiguous() else q.new_empty(qs, dtype=torch.bfloat16)
        out_st = (heads * d, d)
    else:
        if out.shape != qs or out.dtype is not torch.bfloat16 or out.stride(2) != 1:
            raise ValueError("out must be a bfloat16 tensor of q's shape with unit channel stride")
        out_st = out.stride()
    k_levels, v_levels = levels
    _call_on(device, "faq_hif4_kv_append", q.data_ptr(), k.data_ptr(), v.data_ptr(), _dtype_code(q), total, heads, h, d,
             q_st[0], q_st[1], k_st[0], k_st[1], v_st[0], v_st[1], q_norm_ptr, k_norm_ptr, norm_dtype, eps, cos_ptr, sin_ptr,
             rope_dtype, rope_ld, rope_rows, offset_ptr, smooth_ptr, smooth_stride, rotate, out.data_ptr(), out_st[0],
             out_st[1], *pool, *ragged, levels_code(k_levels), levels_code(v_levels))
    return out


def hif4_bounds_bytes(head_dim: int) -> int:
    """Bytes of the bounds of one page's keys of one kv head (:func:`hif4_key_bounds`)."""
    if head_dim not in (64, 128):
        raise ValueError("head_dim must be 64 or 128")
    return 2 * head_dim + 16


def hif4_key_bounds(
    pages: torch.Tensor,
    bounds: torch.Tensor,
    table: torch.Tensor,
    cu: torch.Tensor,
    lens: torch.Tensor,
    *,
    page_size: int,
    total: int,
) -> None:
    """The bounds of the keys of every page that the batch's new tokens lie in, anew from the page's tokens
    below ``lens`` (``faq_hif4_key_bounds``): ``bounds`` uint8 ``[num_pages, Hkv, hif4_bounds_bytes(D)]``, per
    page and kv head the least and the greatest value of each channel, in 8 bits with one exponent,
    rounded outward. Call it after the tokens are written (:func:`hif4_kv_append`, :func:`hif4_kv_write`) and before
    :func:`hif4_select_pages`. ``total`` is a host number, at least ``cu[B]``."""
    device = _require_cuda(pages, bounds, table, cu, lens)
    h, d = _bounds_shape(bounds)
    pool, ragged = _ragged(pages, table, cu, lens, h, d, page_size)
    if bounds.shape[0] != pool[1]:
        raise ValueError("pages and bounds must have one number of pages")
    _call_on(device, "faq_hif4_key_bounds", *pool, h, d, *ragged, total, bounds.data_ptr())


def _bounds_shape(bounds: torch.Tensor) -> tuple[int, int]:
    """``(kv_heads, head_dim)`` of a bounds tensor."""
    shape = bounds.shape
    if bounds.dtype is not torch.uint8 or len(shape) != 3 or not bounds.is_contiguous():
        raise TypeError("bounds must be a contiguous uint8 tensor [num_pages, kv_heads, hif4_bounds_bytes(head_dim)]")
    d = (shape[2] - 16) // 2
    if d not in (64, 128) or shape[2] != 2 * d + 16:
        raise ValueError("bounds must be [num_pages, kv_heads, hif4_bounds_bytes(head_dim)]")
    return shape[1], d


def hif4_select_pages(
    q: torch.Tensor,
    bounds: torch.Tensor,
    table: torch.Tensor,
    cu: torch.Tensor,
    lens: torch.Tensor,
    *,
    page_size: int,
    count: int,
    first: int = 1,
    last: int = 2,
    want_scores: bool = False,
    out: torch.Tensor | None = None,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """The pages that each new token attends to: int32 ``[T, Hkv, count]``, columns of the sequence's row of
    ``table`` in ascending order, -1 behind them (``faq_hif4_select_pages``). ``q [T, H, D]`` bf16 are the queries
    of the attention, ``bounds`` those of :func:`hif4_key_bounds`.

    A page's score is the greatest ``q . K`` that its bounds allow, ``sum_d max(q_d lo_d, q_d hi_d)``, the greatest over
    the query heads of the kv head, with q in 8 bits (one exponent for the kv head's queries): whole numbers, so the
    choice is exact. Taken are the sequence's ``first`` pages, the ``last`` ones up to the token's own (at
    least one), then those of the greatest scores, ties to the lowest column. Pages that the table does not hold
    are not taken and set ``FAQ_STATUS_BAD_PAGE``; entries of q that are not finite count as zero. With
    ``want_scores`` returns ``(selected, scores)``, scores fp32 of the same shape, -inf behind the pages. Rows
    beyond ``cu[B]`` stay as they are. At most 32768 columns and 128 query heads per kv head; the columns choose the
    kernel, so give no more of them than the longest sequence has (a slice of a wider table)."""
    device = _require_cuda(q, bounds, table, cu, lens, out)
    qs = q.shape
    if q.dtype is not torch.bfloat16 or len(qs) != 3:
        raise TypeError("q must be bfloat16 [tokens, heads, head_dim]")
    total, heads, d = qs
    h, bounds_d = _bounds_shape(bounds)
    if bounds_d != d or h == 0 or heads % h or heads == 0:
        raise ValueError("q's heads must be divisible by the kv heads of the bounds, of one head_dim")
    hif4_page_bytes(h, d, page_size)
    ragged = _batch(table, cu, lens)
    st = q.stride()
    if st[2] != 1:
        q = q.contiguous()
        st = q.stride()
    shape = (total, h, count)
    if out is None:
        if count < 1:
            raise ValueError("count must be positive")
        out = q.new_empty(shape, dtype=torch.int32)
    elif out.shape != shape or out.dtype is not torch.int32 or not out.is_contiguous():
        raise ValueError("out must be a contiguous int32 tensor [tokens, kv_heads, count]")
    scores = q.new_empty(shape, dtype=torch.float32) if want_scores else None
    _call_on(device, "faq_hif4_select_pages", q.data_ptr(), total, heads, st[0], st[1], bounds.data_ptr(), bounds.shape[0],
             page_size, h, d, *ragged, count, first, last, out.data_ptr(), _ptr(scores))
    return (out, scores) if want_scores else out


def hif4_sparse_attention(
    q: torch.Tensor,
    pages: torch.Tensor,
    table: torch.Tensor,
    cu: torch.Tensor,
    lens: torch.Tensor,
    selected: torch.Tensor,
    *,
    page_size: int,
    scale: float | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Attention of each new token over the tokens of the pages listed for it: ``q [T, H, D]`` bf16, returns
    ``[T, H, D]`` bf16 (``faq_hif4_sparse_attention``). ``selected`` int32 ``[T, Hkv, count]``
    (:func:`hif4_select_pages`) holds columns of the sequence's row of ``table``, in any order; entries below zero and
    pages behind the token are passed over, a column listed twice counts once, and no token sees keys behind
    itself (at most 32768 entries; lists that ascend are read fastest). With every visible page listed this is :func:`hif4_paged_attention`, up to the rounding of its sums.
    A row without a key is zero; rows beyond ``cu[B]`` stay as they are; pages that the table does not hold are
    left out and set ``FAQ_STATUS_BAD_PAGE``."""
    device = _require_cuda(q, pages, table, cu, lens, selected, out)
    shape = q.shape
    if q.dtype is not torch.bfloat16 or len(shape) != 3:
        raise TypeError("q must be bfloat16 [tokens, heads, head_dim]")
    total, heads, d = shape
    h = _kv_heads(pages, d, page_size)
    pool, ragged = _ragged(pages, table, cu, lens, h, d, page_size)
    if heads % h or heads == 0:
        raise ValueError("query heads must be divisible by key/value heads")
    lists = selected.shape
    if selected.dtype is not torch.int32 or len(lists) != 3 or lists[0] != total or lists[1] != h:
        raise ValueError("selected must be int32 [tokens, kv_heads, count]")
    if not selected.is_contiguous():
        selected = selected.contiguous()
    st = q.stride()
    if st[2] != 1 or st[0] % 8 or st[1] % 8 or st[0] < 8 or st[1] < 8 or q.data_ptr() % 16:
        q = q.contiguous() if not q.is_contiguous() else q.clone()
        st = (heads * d, d)
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else q.new_empty(shape)
        out_st = (heads * d, d)
    else:
        if out.shape != shape or out.dtype is not torch.bfloat16 or out.stride(2) != 1:
            raise ValueError("out must be a bfloat16 tensor of q's shape with unit channel stride")
        out_st = out.stride()
    _call_on(device, "faq_hif4_sparse_attention", q.data_ptr(), total, heads, st[0], st[1], *pool, h, d, *ragged,
             selected.data_ptr(), lists[2], d**-0.5 if scale is None else scale, out.data_ptr(), out_st[0], out_st[1])
    return out


def verify_drafts(
    draft_tokens: torch.Tensor,
    target_probs: torch.Tensor,
    draft_probs: torch.Tensor | None,
    accept_u: torch.Tensor,
    sample_u: torch.Tensor,
    *,
    num_drafts: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Speculative sampling's check of drafted tokens (``faq_verify_drafts``).

    ``draft_tokens [B, K]`` int64, ``target_probs [B, K + 1, V]`` and ``draft_probs [B, K, V]``
    (bf16 or fp32; None for drafts without a distribution, such as tokens looked up in the
    context), uniform random numbers ``accept_u [B, K]`` and ``sample_u [B]`` (fp32),
    ``num_drafts [B]`` int32 for a ragged batch. Returns ``(tokens [B, K + 1] int64, accepted
    [B] int32)``: the accepted drafts, one token sampled from the residual or the target,
    then -1. The result does not depend on the order of summation."""
    device = _require_cuda(draft_tokens, target_probs, draft_probs, accept_u, sample_u, num_drafts)
    if target_probs.dim() != 3 or draft_tokens.dim() != 2:
        raise ValueError("draft_tokens must be [B, K] and target_probs [B, K + 1, V]")
    b, k1, vocab = target_probs.shape
    k = k1 - 1
    if draft_tokens.shape != (b, k) or accept_u.shape != (b, k) or sample_u.shape != (b,):
        raise ValueError("draft_tokens and accept_u must be [B, K], sample_u [B], target_probs [B, K + 1, V]")
    if draft_tokens.dtype is not torch.int64 or accept_u.dtype is not torch.float32 or sample_u.dtype is not torch.float32:
        raise TypeError("draft_tokens must be int64, accept_u and sample_u float32")
    ts = target_probs.stride()
    if ts[2] != 1:
        target_probs = target_probs.contiguous()
        ts = target_probs.stride()
    ds = (0, 0)
    if draft_probs is not None:
        if draft_probs.shape != (b, k, vocab) or draft_probs.dtype != target_probs.dtype:
            raise ValueError("draft_probs must be [B, K, V] of target_probs' dtype")
        ds = draft_probs.stride()
        if ds[2] != 1:
            draft_probs = draft_probs.contiguous()
            ds = draft_probs.stride()
    if num_drafts is not None:
        if num_drafts.shape != (b,) or num_drafts.dtype is not torch.int32:
            raise ValueError("num_drafts must be int32 [B]")
        num_drafts = num_drafts.contiguous()
    draft_tokens, accept_u, sample_u = draft_tokens.contiguous(), accept_u.contiguous(), sample_u.contiguous()
    tokens = draft_tokens.new_empty((b, k1))
    accepted = draft_tokens.new_empty((b,), dtype=torch.int32)
    _lib.call("faq_verify_drafts", draft_tokens.data_ptr(), target_probs.data_ptr(), _ptr(draft_probs),
              _dtype_code(target_probs), b, k, vocab, ts[0], ts[1], ds[0], ds[1], accept_u.data_ptr(),
              sample_u.data_ptr(), _ptr(num_drafts), tokens.data_ptr(), accepted.data_ptr(), _stream(device))
    return tokens, accepted
