"""comfy_kitchen for MI355X: quantize / block-scaled GEMM / RoPE on gfx950.

Drop-in for the reference's public op API (comfy_kitchen/__init__.py:60-366): the
same function names, signatures, defaults and return types.  Every op goes through
the `comfy_kitchen::*` custom ops and the backend registry to the "hip" backend,
whose kernels are hand-written for gfx950 and reached through a C-ABI library.
"""
import torch

from . import ops as _ops  # noqa: F401  (registers torch.ops.comfy_kitchen.*)
from .backends import hip as _hip_backend  # noqa: F401  (registers the "hip" backend)
from .exceptions import (
    BackendError,
    BackendNotFoundError,
    BackendNotImplementedError,
    NoCapableBackendError,
)
from .float_utils import from_blocked, swap_nibbles, to_blocked
from .ops import DTYPE_TO_CODE, _dispatch, _quantize_fp8_dynamic, changed, direct, untouched
from .paged import OutOfPages, PagedKVCache
from .registry import registry

__version__ = "0.1.0"

__all__ = [
    "quantize_per_tensor_fp8",
    "dequantize_per_tensor_fp8",
    "quantize_fp8_dynamic",
    "quantize_nvfp4",
    "quantize_nvfp4_dynamic",
    "dequantize_nvfp4",
    "quantize_mxfp8",
    "dequantize_mxfp8",
    "scaled_mm_nvfp4",
    "scaled_mm_mxfp8",
    "quantize_int4",
    "dequantize_int4",
    "linear_int4",
    "paged_attention",
    "paged_write",
    "paged_copy",
    "window_attention",
    "PagedKVCache",
    "OutOfPages",
    "apply_rope",
    "apply_rope1",
    "swap_nibbles",
    "to_blocked",
    "from_blocked",
    "list_backends",
    "set_backend_priority",
    "enable_backend",
    "disable_backend",
    "stochastic_rounding_fp8",
    "use_backend",
    "BackendError",
    "BackendNotFoundError",
    "BackendNotImplementedError",
    "NoCapableBackendError",
]


def amax_scale(x: torch.Tensor, divisor: float) -> torch.Tensor:
    """amax(|x|) / divisor computed in x's dtype, returned as a 0-dim fp32 device tensor.

    Not part of the reference's public API: it is the default scale of the layouts'
    quantize (reference tensor/fp8.py:56-61, tensor/nvfp4.py:64-69) as one device-side
    reduction, so dynamic quantization needs no host round trip.
    """
    divisor = float(divisor)
    if direct(x) and untouched("amax_scale"):
        return _dispatch("amax_scale", x=x, divisor=divisor)
    return torch.ops.comfy_kitchen.amax_scale(x, divisor)


def quantize_per_tensor_fp8(x: torch.Tensor, scale: torch.Tensor,
                            output_type: torch.dtype = torch.float8_e4m3fn) -> torch.Tensor:
    """FP8 quantize with one fp32 scale: fp8(clamp(x * (1/scale), +-max))."""
    code = DTYPE_TO_CODE[output_type]
    if direct(x, scale) and untouched("quantize_fp8"):
        return _dispatch("quantize_per_tensor_fp8", x=x, scale=scale, output_type=output_type)
    return torch.ops.comfy_kitchen.quantize_fp8(x, scale, code)


def quantize_fp8_dynamic(x: torch.Tensor, divisor: float = 448.0,
                         output_type: torch.dtype = torch.float8_e4m3fn) -> tuple[torch.Tensor, torch.Tensor]:
    """quantize_per_tensor_fp8 with the scale amax(|x|) / divisor (in x's dtype) formed on the
    device in the same call: returns (codes, 0-dim fp32 scale).

    Not part of the reference's public API: it is the scale=None branch of the FP8 layout's
    quantize (reference tensor/fp8.py:56-61) with the reduction fused into the quantize
    launch.  The results equal amax_scale followed by quantize_per_tensor_fp8 bit for bit."""
    divisor, code = float(divisor), DTYPE_TO_CODE[output_type]
    if direct(x) and untouched("quantize_fp8_dynamic"):
        return _quantize_fp8_dynamic(x, divisor, output_type)
    return torch.ops.comfy_kitchen.quantize_fp8_dynamic(x, divisor, code)


def dequantize_per_tensor_fp8(x: torch.Tensor, scale: torch.Tensor,
                              output_type: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """FP8 dequantize: x.to(output_type) * scale.to(output_type)."""
    code = DTYPE_TO_CODE[output_type]
    if direct(x, scale) and untouched("dequantize_fp8"):
        return _dispatch("dequantize_per_tensor_fp8", x=x, scale=scale, output_type=output_type)
    return torch.ops.comfy_kitchen.dequantize_fp8(x, scale, code)


def stochastic_rounding_fp8(x: torch.Tensor, rng: torch.Tensor,
                            output_type: torch.dtype = torch.float8_e4m3fn) -> torch.Tensor:
    """Stochastic FP8 rounding.  Not provided by the hip backend (raises NoCapableBackendError)."""
    kwargs = {"x": x, "rng": rng, "output_type": output_type}
    return registry.get_implementation("stochastic_rounding_fp8", kwargs=kwargs)(**kwargs)


def quantize_nvfp4(x: torch.Tensor, per_tensor_scale: torch.Tensor, epsilon: float = 0.0,
                   pad_16x: bool = False, hi_first: bool = True) -> tuple[torch.Tensor, torch.Tensor]:
    """NVFP4: packed E2M1 codes [M, K/2] uint8 and swizzled E4M3 block-16 scales."""
    if (type(epsilon) is float and type(pad_16x) is bool and type(hi_first) is bool
            and direct(x, per_tensor_scale) and untouched("quantize_nvfp4")):
        return _dispatch("quantize_nvfp4", x=x, per_tensor_scale=per_tensor_scale, epsilon=epsilon,
                         pad_16x=pad_16x, hi_first=hi_first)
    return torch.ops.comfy_kitchen.quantize_nvfp4(x, per_tensor_scale, epsilon, pad_16x, hi_first)


def quantize_nvfp4_dynamic(x: torch.Tensor, divisor: float = 448.0 * 6.0, pad_16x: bool = False,
                           hi_first: bool = True) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """quantize_nvfp4 with the per-tensor scale amax(|x|) / divisor (in x's dtype) formed on
    the device in the same call: returns (codes, block scales, 0-dim fp32 scale).

    Not part of the reference's public API: it is the scale=None branch of the NVFP4
    layout's quantize (reference tensor/nvfp4.py:64-69, the dynamic activation scale of
    samples/nvfp4_linear.py:55-59) with the reduction fused into the quantize launch.
    The results equal amax_scale followed by quantize_nvfp4 bit for bit."""
    divisor = float(divisor)
    if type(pad_16x) is bool and type(hi_first) is bool and direct(x) and untouched("quantize_nvfp4_dynamic"):
        return _dispatch("quantize_nvfp4_dynamic", x=x, divisor=divisor, pad_16x=pad_16x, hi_first=hi_first)
    return torch.ops.comfy_kitchen.quantize_nvfp4_dynamic(x, divisor, pad_16x, hi_first)


def dequantize_nvfp4(qx: torch.Tensor, per_tensor_scale: torch.Tensor, block_scales: torch.Tensor,
                     output_type: torch.dtype = torch.bfloat16, hi_first: bool = True) -> torch.Tensor:
    code = DTYPE_TO_CODE[output_type]
    if type(hi_first) is bool and direct(qx, per_tensor_scale, block_scales) and untouched("dequantize_nvfp4"):
        return _dispatch("dequantize_nvfp4", qx=qx, per_tensor_scale=per_tensor_scale, block_scales=block_scales,
                         output_type=output_type, hi_first=hi_first)
    return torch.ops.comfy_kitchen.dequantize_nvfp4(qx, per_tensor_scale, block_scales, code, hi_first)


def scaled_mm_nvfp4(a: torch.Tensor, b: torch.Tensor, tensor_scale_a: torch.Tensor,
                    tensor_scale_b: torch.Tensor, block_scale_a: torch.Tensor,
                    block_scale_b: torch.Tensor, bias: torch.Tensor | None = None,
                    out_dtype: torch.dtype | None = None,
                    alpha: torch.Tensor | None = None) -> torch.Tensor:
    """y = (a @ b.T) * (tensor_scale_a * tensor_scale_b) + bias on NVFP4 operands."""
    out_dtype = out_dtype if out_dtype is not None else torch.bfloat16
    code = DTYPE_TO_CODE[out_dtype]
    if (direct(a, b, tensor_scale_a, tensor_scale_b, block_scale_a, block_scale_b, bias, alpha)
            and untouched("scaled_mm_nvfp4")):
        return _dispatch("scaled_mm_nvfp4", a=a, b=b, tensor_scale_a=tensor_scale_a, tensor_scale_b=tensor_scale_b,
                         block_scale_a=block_scale_a, block_scale_b=block_scale_b, bias=bias, out_dtype=out_dtype,
                         alpha=alpha)
    return torch.ops.comfy_kitchen.scaled_mm_nvfp4(
        a, b, tensor_scale_a, tensor_scale_b, block_scale_a, block_scale_b, bias, code, alpha)


def quantize_mxfp8(x: torch.Tensor, pad_32x: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """MXFP8: E4M3 codes [M, K] and swizzled E8M0 block-32 scales."""
    if type(pad_32x) is bool and direct(x) and untouched("quantize_mxfp8"):
        return _dispatch("quantize_mxfp8", x=x, pad_32x=pad_32x)
    return torch.ops.comfy_kitchen.quantize_mxfp8(x, pad_32x)


def dequantize_mxfp8(qx: torch.Tensor, block_scales: torch.Tensor,
                     output_type: torch.dtype = torch.bfloat16) -> torch.Tensor:
    code = DTYPE_TO_CODE[output_type]
    if direct(qx, block_scales) and untouched("dequantize_mxfp8"):
        return _dispatch("dequantize_mxfp8", qx=qx, block_scales=block_scales, output_type=output_type)
    return torch.ops.comfy_kitchen.dequantize_mxfp8(qx, block_scales, code)


def scaled_mm_mxfp8(a: torch.Tensor, b: torch.Tensor, block_scale_a: torch.Tensor,
                    block_scale_b: torch.Tensor, bias: torch.Tensor | None = None,
                    out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """y = a @ b.T + bias on MXFP8 operands (both K-major, E8M0 block-32 scales)."""
    out_dtype = out_dtype if out_dtype is not None else torch.bfloat16
    code = DTYPE_TO_CODE[out_dtype]
    if direct(a, b, block_scale_a, block_scale_b, bias) and untouched("scaled_mm_mxfp8"):
        return _dispatch("scaled_mm_mxfp8", a=a, b=b, block_scale_a=block_scale_a, block_scale_b=block_scale_b,
                         bias=bias, out_dtype=out_dtype)
    return torch.ops.comfy_kitchen.scaled_mm_mxfp8(a, b, block_scale_a, block_scale_b, bias, code)


def scaled_mm_fp8(a: torch.Tensor, b: torch.Tensor, scale_a: torch.Tensor, scale_b: torch.Tensor,
                  bias: torch.Tensor | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """y = scale_a * scale_b * (a @ b.T) + bias on per-tensor E4M3 operands (both K-major).

    Not part of the reference's public API: it is the matmul behind TensorCoreFP8Layout's
    linear / mm / addmm, where the reference calls torch F.scaled_mm (scaled_mm_v2.py:27-53).
    """
    out_dtype = out_dtype if out_dtype is not None else torch.bfloat16
    code = DTYPE_TO_CODE[out_dtype]
    if direct(a, b, scale_a, scale_b, bias) and untouched("scaled_mm_fp8"):
        return _dispatch("scaled_mm_fp8", a=a, b=b, scale_a=scale_a, scale_b=scale_b, bias=bias, out_dtype=out_dtype)
    return torch.ops.comfy_kitchen.scaled_mm_fp8(a, b, scale_a, scale_b, bias, code)


def quantize_int4(w: torch.Tensor, group_size: int = 128) -> tuple[torch.Tensor, torch.Tensor]:
    """4-bit codes [N, K/2] (uint8, the even k in the low nibble) and scales [N, ceil(K/group_size)]
    in w's dtype of a weight [N, K]: w ~= (code - 8) * scale, scale = amax(|group|) / 7.

    K and group_size are multiples of 32; the last group of a row may be shorter."""
    if type(group_size) is int and direct(w) and untouched("quantize_int4"):
        return _dispatch("quantize_int4", w=w, group_size=group_size)
    return torch.ops.comfy_kitchen.quantize_int4(w, group_size)


def dequantize_int4(codes: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None,
                    group_size: int = 128, output_type: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """(code - zero) * scale as [N, K] of output_type; zeros: uint8 of scales' shape (None: 8)."""
    code = DTYPE_TO_CODE[output_type]
    if type(group_size) is int and direct(codes, scales, zeros) and untouched("dequantize_int4"):
        return _dispatch("dequantize_int4", codes=codes, scales=scales, zeros=zeros, group_size=group_size,
                         output_type=output_type)
    return torch.ops.comfy_kitchen.dequantize_int4(codes, scales, zeros, group_size, code)


def linear_int4(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None,
                bias: torch.Tensor | None = None, group_size: int = 128) -> torch.Tensor:
    """y = x @ W.T + bias for a weight W [N, K] of 4-bit codes with a scale (and zero point) for
    each row and group of group_size inputs; x [..., K] in f16 / bf16, y [..., N] in x's dtype.

    Made for the one to some dozens of rows of text generation, where reading the codes bounds
    the call; up to 1048560 rows are served, but from some 512 on dequantize_int4 and a matrix product
    take less time (4096 rows, N=5120, K=13824: 1.63 ms against 0.48) for the memory of the 16-bit
    weight.  A row of x that holds an infinity or NaN gives NaNs."""
    if type(group_size) is int and direct(x, codes, scales, zeros, bias) and untouched("linear_int4"):
        return _dispatch("linear_int4", x=x, codes=codes, scales=scales, zeros=zeros, bias=bias, group_size=group_size)
    return torch.ops.comfy_kitchen.linear_int4(x, codes, scales, zeros, bias, group_size)


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                    lengths: torch.Tensor, scale: float | None = None, window: int = 0, sinks: int = 0,
                    k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one new token per sequence, q [B, heads, head_dim] in f16 / bf16, over a cache
    held in pages; the result has q's shape and dtype.

    k_cache, v_cache: [pages, page_size, kv_heads, head_dim], in q's dtype or as E4M3 codes of
    value / k_scale, value / v_scale (one-element fp32 tensors, which multiply what either kind of cache
    holds; None: 1); any strides that are multiples of 16 bytes with head_dim contiguous, so [pages, kv_heads, page_size, head_dim] is a
    permuted view away.  heads is a multiple of kv_heads; head_dim 64, 96, 128 or 256.
    page_table: int32 [B, n]; token t of sequence b is row t % page_size of page
    page_table[b, t // page_size].  lengths: int32 [B], the tokens of each sequence, the new one
    (written before the call) among them; a sequence of none gives zeros.
    window > 0: only the last `window` tokens and the first `sinks` are visible; pages without a
    visible token are not read and may have been given away.
    scale: of the scores, head_dim ** -0.5 by default."""
    if direct(q, k_cache, v_cache, page_table, lengths, k_scale, v_scale) and untouched("paged_attention"):
        return _dispatch("paged_attention", q=q, k_cache=k_cache, v_cache=v_cache, page_table=page_table,
                         lengths=lengths, scale=scale, window=window, sinks=sinks, k_scale=k_scale, v_scale=v_scale)
    return torch.ops.comfy_kitchen.paged_attention(q, k_cache, v_cache, page_table, lengths, scale, window, sinks,
                                                   k_scale, v_scale)


def paged_write(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                slots: torch.Tensor, k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None) -> None:
    """Store the keys and values of new tokens [T, kv_heads, head_dim] (f16 / bf16) in their slots of
    a cache held in pages, in place: slot page * page_size + row for each token (int32 or int64,
    on the device; a slot outside the cache, such as -1, skips its token; slots are distinct).

    The caches are [pages, page_size, kv_heads, head_dim] of key's dtype, which take the rows as they
    are (no scales), or E4M3, which take the codes of clamp(x / scale, +-448).  head_dim is a
    multiple of 16."""
    if direct(key, value, k_cache, v_cache, slots, k_scale, v_scale) and untouched("paged_write"):
        _dispatch("paged_write", key=key, value=value, k_cache=k_cache, v_cache=v_cache, slots=slots,
                  k_scale=k_scale, v_scale=v_scale)
        return changed(k_cache, v_cache)
    torch.ops.comfy_kitchen.paged_write(key, value, k_cache, v_cache, slots, k_scale, v_scale)


def paged_copy(k_cache: torch.Tensor, v_cache: torch.Tensor, src: torch.Tensor, dst: torch.Tensor) -> None:
    """Copy token rows of a cache held in pages from slots src to slots dst (int32 or int64, on the
    device), in place, in K and V: [pages, page_size, kv_heads, head_dim], or of all layers at
    once with a leading dimension.  No slot of dst may be in src; pairs with a slot outside the
    cache are skipped."""
    if direct(k_cache, v_cache, src, dst) and untouched("paged_copy"):
        _dispatch("paged_copy", k_cache=k_cache, v_cache=v_cache, src=src, dst=dst)
        return changed(k_cache, v_cache)
    torch.ops.comfy_kitchen.paged_copy(k_cache, v_cache, src, dst)


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int = 0, sinks: int = 0,
                     lengths: torch.Tensor | None = None, scale: float | None = None) -> torch.Tensor:
    """Causal attention of prompts: q [B, queries, heads, head_dim], k and v [B, keys, kv_heads,
    head_dim] in one of f16 / bf16; the result has q's shape and dtype.

    Query i stands at position i + keys - queries (the last query at the last key, so k and v may
    begin with tokens of earlier calls) and sees the keys up to its position: with window > 0 the
    last `window` of them, and in any case the first `sinks` keys of the sequence.  lengths:
    int32 [B], keys of each sequence where the batch is padded behind (keys past them are not
    seen).  A query that sees nothing gives zeros.
    heads is a multiple of kv_heads; head_dim 64, 96, 128 or 256.  Any strides with head_dim
    contiguous are taken ([B, heads, tokens, head_dim] is a transposed view away); tensors whose
    rows are not on 16-byte boundaries are copied.  scale: of the scores, head_dim ** -0.5 by default."""
    if direct(q, k, v, lengths) and untouched("window_attention"):
        return _dispatch("window_attention", q=q, k=k, v=v, window=window, sinks=sinks, lengths=lengths, scale=scale)
    return torch.ops.comfy_kitchen.window_attention(q, k, v, window, sinks, lengths, scale)


def apply_rope(xq: torch.Tensor, xk: torch.Tensor,
               freqs_cis: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rotate query and key by the 2x2 matrices in freqs_cis [..., head_dim/2, 2, 2]."""
    if direct(xq, xk, freqs_cis) and untouched("apply_rope"):
        return _dispatch("apply_rope", xq=xq, xk=xk, freqs_cis=freqs_cis)
    return torch.ops.comfy_kitchen.apply_rope(xq, xk, freqs_cis)


def apply_rope1(x: torch.Tensor, freqs_cis: torch.Tensor) -> torch.Tensor:
    if direct(x, freqs_cis) and untouched("apply_rope1"):
        return _dispatch("apply_rope1", x=x, freqs_cis=freqs_cis)
    return torch.ops.comfy_kitchen.apply_rope1(x, freqs_cis)


def set_backend_priority(priority: list[str]) -> None:
    registry.set_priority(priority)


def disable_backend(name: str) -> None:
    registry.disable(name)


def enable_backend(name: str) -> None:
    registry.enable(name)


def list_backends() -> dict:
    return registry.list_backends()


def use_backend(name: str):
    return registry.use_backend(name)
