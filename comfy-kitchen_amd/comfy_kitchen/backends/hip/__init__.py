"""The "hip" backend: gfx950 kernels from libckh.so, called through its C ABI.

Role and contract follow the reference's CUDA backend (backends/cuda/__init__.py):
module-level functions with the eager backend's keyword arguments, outputs allocated
here with torch (the C side never allocates), launches on torch's current stream
(reference __init__.py:152), and per-function constraints registered with the
registry (reference __init__.py:516-691).  The binding is ctypes over a plain C ABI
(include/ckh.h) instead of nanobind/DLPack: raw device pointers, int64 sizes, dtype
codes and the stream handle.

There is no fallback: if libckh.so is missing or the device is not gfx950 the
backend is marked unavailable with the reason, and every `ck.*` call raises
NoCapableBackendError naming it.
"""
from __future__ import annotations

import ctypes
import functools
import os
from pathlib import Path

import torch

from ...float_utils import roundup
from ...ops import DTYPE_TO_CODE

__all__ = [
    "amax_scale",
    "apply_rope",
    "apply_rope1",
    "dequantize_int4",
    "dequantize_mxfp8",
    "dequantize_nvfp4",
    "dequantize_per_tensor_fp8",
    "linear_int4",
    "paged_attention",
    "paged_copy",
    "paged_write",
    "paged_write_rope",
    "quantize_fp8_dynamic",
    "quantize_int4",
    "quantize_mxfp8",
    "quantize_nvfp4",
    "quantize_nvfp4_dynamic",
    "quantize_per_tensor_fp8",
    "rms_norm",
    "rms_norm_fp8",
    "rms_norm_mxfp8",
    "sample_tokens",
    "scaled_mm_fp8",
    "scaled_mm_mxfp8",
    "scaled_mm_nvfp4",
    "shared_attention",
    "window_attention",
]

LIB_PATH = Path(os.environ.get("CKH_LIBRARY", Path(__file__).with_name("libckh.so")))
REQUIRED_ARCH = ("gfx950",)

_p, _i64, _i32, _f32, _u64 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_float, ctypes.c_uint64
_f64 = ctypes.c_double

# C signatures, exactly as declared in include/ckh.h
SIGNATURES: dict[str, tuple] = {
    "ckh_abi_version": (_i32, []),
    "ckh_last_error": (ctypes.c_char_p, []),
    "ckh_quantize_fp8": (_i32, [_p, _p, _p, _i64, _i32, _i32, _u64]),
    "ckh_dequantize_fp8": (_i32, [_p, _p, _p, _i64, _i32, _i32, _i32, _u64]),
    "ckh_quantize_mxfp8": (_i32, [_p, _p, _p, _i64, _i64, _i64, _i64, _i32, _u64]),
    "ckh_dequantize_mxfp8": (_i32, [_p, _p, _p, _i64, _i64, _i32, _u64]),
    "ckh_quantize_nvfp4": (_i32, [_p, _p, _p, _p, _i64, _i64, _i64, _i64, _f32, _i32, _i32, _u64]),
    "ckh_dequantize_nvfp4": (_i32, [_p, _p, _p, _p, _i64, _i64, _i32, _i32, _u64]),
    "ckh_apply_rope": (_i32, [_p, _p, _p, _p, _p] + [_i64] * 13 + [_i32, _i32, _u64]),
    "ckh_scaled_mm_workspace_bytes": (_i64, [_i64] * 3),
    "ckh_scaled_mm_mxfp8": (_i32, [_p] * 6 + [_i64] * 3 + [_i32, _i32, _p, _i64, _u64]),
    "ckh_scaled_mm_fp8": (_i32, [_p] * 6 + [_i64] * 3 + [_i32, _i32, _p, _i64, _u64]),
    "ckh_scaled_mm_nvfp4": (_i32, [_p] * 7 + [_i64] * 3 + [_i32, _i32, _p, _i64, _u64]),
    "ckh_scaled_mm_nvfp4_scales": (_i32, [_p] * 8 + [_i64] * 3 + [_i32, _i32, _p, _i64, _u64]),
    "ckh_scaled_mm_nvfp4_workspace_bytes": (_i64, [_i64] * 3),
    "ckh_amax_scale": (_i32, [_p, _i64, _i32, _f32, _p, _p, _u64]),
    "ckh_amax_scale_noalloc": (_i32, [_p, _i64, _i32, _f32, _p, _u64]),
    "ckh_quantize_fp8_dynamic": (_i32, [_p, _f32, _p, _p, _i64, _i32, _i32, _p, _u64]),
    "ckh_quantize_nvfp4_dynamic": (_i32, [_p, _f32, _p, _p, _p, _i64, _i64, _i64, _i64, _f32, _i32, _i32, _p, _u64]),
    "ckh_quantize_int4": (_i32, [_p] * 3 + [_i64] * 3 + [_i32, _u64]),
    "ckh_dequantize_int4": (_i32, [_p] * 4 + [_i64] * 3 + [_i32, _i32, _u64]),
    "ckh_linear_int4_workspace_bytes": (_i64, [_i64] * 4),
    "ckh_linear_int4": (_i32, [_p] * 6 + [_i64] * 5 + [_i32] * 3 + [_p, _i64, _u64]),
    "ckh_paged_attention_workspace_bytes": (_i64, [_i64] * 6),
    "ckh_paged_attention": (_i32, [_p] * 8 + [_i64] * 8 + [_p] + [_i64] * 2 + [_f32, _i32, _i32, _p, _i64, _u64]),
    "ckh_paged_write": (_i32, [_p] * 7 + [_i64] * 5 + [_p] + [_i32] * 3 + [_u64]),
    "ckh_paged_copy": (_i32, [_p] * 4 + [_i64] * 6 + [_p] + [_i32] * 2 + [_u64]),
    "ckh_window_attention_workspace_bytes": (_i64, [_i64] * 8),
    "ckh_window_attention": (_i32, [_p] * 5 + [_i64] * 6 + [_p] + [_i64] * 2 + [_f32, _i32, _p, _i64, _u64]),
    "ckh_rms_norm": (_i32, [_p] * 7 + [_i64] * 6 + [_f32] + [_i32] * 4 + [_u64]),
    "ckh_paged_write_rope": (_i32, [_p] * 12 + [_i64] * 7 + [_p, _i32, _f32] + [_i32] * 4 + [_u64]),
    "ckh_sample_workspace_bytes": (_i64, [_i64] * 2),
    "ckh_sample": (_i32, [_p] * 6 + [_f64, _i64, _f64, _f64, _p] + [_i64] * 3 + [_i32, _p, _i64, _u64]),
    "ckh_shared_attention_workspace_bytes": (_i64, [_i64] * 7),
    "ckh_shared_attention": (_i32, [_p] * 10 + [_i64] * 9 + [_p, _f32, _i32, _i32, _p, _i64, _u64]),
}
ABI_VERSION = 8
# CKH_AMAX_WORKSPACE_BYTES of include/ckh.h: the workspace ckh_amax_scale takes
AMAX_WORKSPACE_BYTES = 8192

_lib: ctypes.CDLL | None = None


def load_library(path: Path | str | None = None) -> ctypes.CDLL:
    """Load libckh.so and bind every entry point's signature (no GPU needed).

    torch is imported first (module import above), so the library binds to torch's
    HIP runtime: both carry the SONAME libamdhip64.so.7 and the loader reuses it.
    """
    global _lib
    if _lib is not None and path is None:
        return _lib
    p = Path(path) if path is not None else LIB_PATH
    if not p.exists():
        raise OSError(f"{p} not found: build it with `python comfy-kitchen_amd/build.py`")
    lib = ctypes.CDLL(str(p))
    for name, (res, args) in SIGNATURES.items():
        try:
            fn = getattr(lib, name)
        except AttributeError:  # an older build: entry points were added without a new ABI version
            raise OSError(f"{p}: no entry point {name}: rebuild it with `python comfy-kitchen_amd/build.py`") from None
        fn.restype, fn.argtypes = res, args
    if lib.ckh_abi_version() != ABI_VERSION:
        raise OSError(f"{p}: ABI version {lib.ckh_abi_version()} != expected {ABI_VERSION}")
    if path is None:
        _lib = lib
    return lib


def _call(name: str, *args) -> None:
    status = getattr(_lib, name)(*args)
    if status != 0:
        raise RuntimeError(f"{name}: {_lib.ckh_last_error().decode(errors='replace')}")


# (the public forms where a torch lacks the bindings below them)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda device: torch.cuda.current_stream(device).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _launch(name: str, t: torch.Tensor, *args) -> None:
    """Call entry point `name` with args and the current stream of t's device, which is made
    current for the call (a no-op when it already is)."""
    device = t.get_device()
    if device == _current_device():
        return _call(name, *args, _raw_stream(device))
    with torch.cuda.device(device):
        _call(name, *args, _raw_stream(device))


def _scalar_on(t: torch.Tensor | float, device: torch.device, name: str) -> torch.Tensor:
    """A one-element fp32 tensor on `device` (moving a host scalar if needed)."""
    if not isinstance(t, torch.Tensor):
        t = torch.tensor(float(t), dtype=torch.float32)
    if t.numel() != 1:
        raise ValueError(f"{name} must have exactly one element, got shape {tuple(t.shape)}")
    if t.dtype != torch.float32:
        t = t.to(torch.float32)
    return t if t.device == device else t.to(device)


def _scalar_keep(t: torch.Tensor, device: torch.device, name: str) -> torch.Tensor:
    """A one-element tensor of t's own float dtype on `device`: the kernel reads and widens
    it, as eager's scale.to(out dtype) does."""
    if not isinstance(t, torch.Tensor) or t.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        return _scalar_on(t, device, name)
    if t.numel() != 1:
        raise ValueError(f"{name} must have exactly one element, got shape {tuple(t.shape)}")
    return t if t.device == device else t.to(device)


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _like(t: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor of t's shape and dtype (empty_like takes two thirds of new_empty's time)."""
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


# ------------------------------------------------------------------ per-tensor FP8
def quantize_per_tensor_fp8(x: torch.Tensor, scale: torch.Tensor,
                            output_type: torch.dtype = torch.float8_e4m3fn) -> torch.Tensor:
    x = x.contiguous()
    s = _scalar_on(scale, x.device, "scale")
    out = torch.empty(x.shape, dtype=output_type, device=x.device)
    _launch("ckh_quantize_fp8", x, x.data_ptr(), out.data_ptr(), s.data_ptr(), x.numel(),
            DTYPE_TO_CODE[x.dtype], DTYPE_TO_CODE[output_type])
    return out


def dequantize_per_tensor_fp8(x: torch.Tensor, scale: torch.Tensor,
                              output_type: torch.dtype = torch.bfloat16) -> torch.Tensor:
    x = x.contiguous()
    s = _scalar_keep(scale, x.device, "scale")
    out = torch.empty(x.shape, dtype=output_type, device=x.device)
    _launch("ckh_dequantize_fp8", x, x.data_ptr(), out.data_ptr(), s.data_ptr(), x.numel(),
            DTYPE_TO_CODE[x.dtype], DTYPE_TO_CODE[output_type], DTYPE_TO_CODE[s.dtype])
    return out


def amax_scale(x: torch.Tensor, divisor: float) -> torch.Tensor:
    """amax(|x|) / divisor computed in x's dtype, as a 0-dim fp32 tensor on x's device
    (the layouts' default scale, reference tensor/fp8.py:56-61, tensor/nvfp4.py:64-69)."""
    x = x.contiguous()
    if x.numel() == 0:
        raise RuntimeError("amax_scale: empty tensor")
    out = torch.empty((), dtype=torch.float32, device=x.device)
    # per-workgroup partial maxima (CKH_AMAX_WORKSPACE_BYTES), from torch's allocator
    work = torch.empty(AMAX_WORKSPACE_BYTES // 4, dtype=torch.int32, device=x.device)
    _launch("ckh_amax_scale", x, x.data_ptr(), x.numel(), DTYPE_TO_CODE[x.dtype], float(divisor),
            out.data_ptr(), work.data_ptr())
    return out


def quantize_fp8_dynamic(x: torch.Tensor, divisor: float,
                         output_type: torch.dtype = torch.float8_e4m3fn) -> tuple[torch.Tensor, torch.Tensor]:
    """quantize_per_tensor_fp8 with the scale amax(|x|) / divisor formed on the device in the
    same call: (codes, 0-dim fp32 scale), equal to amax_scale + quantize_per_tensor_fp8."""
    x = x.contiguous()
    if x.numel() == 0:
        raise RuntimeError("quantize_fp8_dynamic: empty tensor")
    out = torch.empty(x.shape, dtype=output_type, device=x.device)
    scale = torch.empty((), dtype=torch.float32, device=x.device)
    work = torch.empty(AMAX_WORKSPACE_BYTES // 4, dtype=torch.int32, device=x.device)
    _launch("ckh_quantize_fp8_dynamic", x, x.data_ptr(), float(divisor), scale.data_ptr(), out.data_ptr(),
            x.numel(), DTYPE_TO_CODE[x.dtype], DTYPE_TO_CODE[output_type], work.data_ptr())
    return out, scale


# --------------------------------------------------------------------------- MXFP8
def quantize_mxfp8(x: torch.Tensor, pad_32x: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    if x.dim() != 2:
        raise ValueError(f"quantize_mxfp8 expects a 2-D tensor, got {x.dim()}-D")
    x = x.contiguous()
    orows, ocols = x.shape
    rows, cols = (roundup(orows, 32), roundup(ocols, 32)) if pad_32x else (orows, ocols)
    if cols % 32:
        raise ValueError(f"K dimension must be divisible by 32 (got {cols}); pass pad_32x=True")
    qx = torch.empty((rows, cols), dtype=torch.float8_e4m3fn, device=x.device)
    sx = torch.empty((roundup(rows, 128), roundup(cols // 32, 4)), dtype=torch.float8_e8m0fnu, device=x.device)
    _launch("ckh_quantize_mxfp8", x, x.data_ptr(), qx.data_ptr(), sx.data_ptr(), rows, cols, orows, ocols,
            DTYPE_TO_CODE[x.dtype])
    return qx, sx


def dequantize_mxfp8(qx: torch.Tensor, block_scales: torch.Tensor,
                     output_type: torch.dtype = torch.bfloat16) -> torch.Tensor:
    qx = qx.contiguous()
    rows, cols = qx.shape
    sc = block_scales.contiguous()
    need = roundup(rows, 128) * roundup(cols // 32, 4)
    if cols % 32 or sc.nbytes < need:
        raise ValueError(f"dequantize_mxfp8: qx {tuple(qx.shape)} needs K % 32 == 0 and {need} scale bytes, "
                         f"got {sc.nbytes}")
    out = torch.empty((rows, cols), dtype=output_type, device=qx.device)
    _launch("ckh_dequantize_mxfp8", qx, qx.data_ptr(), sc.data_ptr(), out.data_ptr(), rows, cols,
            DTYPE_TO_CODE[output_type])
    return out


# --------------------------------------------------------------------------- NVFP4
def quantize_nvfp4(x: torch.Tensor, per_tensor_scale: torch.Tensor, epsilon: float = 0.0,
                   pad_16x: bool = False, hi_first: bool = True) -> tuple[torch.Tensor, torch.Tensor]:
    if x.dim() != 2:
        raise ValueError(f"quantize_nvfp4 expects a 2-D tensor, got {x.dim()}-D")
    x = x.contiguous()
    g = _scalar_on(per_tensor_scale, x.device, "per_tensor_scale")
    orows, ocols = x.shape
    rows, cols = (roundup(orows, 16), roundup(ocols, 16)) if pad_16x else (orows, ocols)
    if cols % 16:
        raise ValueError(f"K dimension must be divisible by 16 (got {cols}); pass pad_16x=True")
    qx = torch.empty((rows, cols // 2), dtype=torch.uint8, device=x.device)
    sx = torch.empty((roundup(rows, 128), roundup(cols // 16, 4)), dtype=torch.float8_e4m3fn, device=x.device)
    _launch("ckh_quantize_nvfp4", x, x.data_ptr(), g.data_ptr(), qx.data_ptr(), sx.data_ptr(), rows, cols,
            orows, ocols, float(epsilon), DTYPE_TO_CODE[x.dtype], int(bool(hi_first)))
    return qx, sx


def quantize_nvfp4_dynamic(x: torch.Tensor, divisor: float, pad_16x: bool = False,
                           hi_first: bool = True) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """quantize_nvfp4 with the scale amax(|x|) / divisor formed on the device in the same
    pass: (codes, block scales, 0-dim fp32 scale), equal to amax_scale + quantize_nvfp4."""
    if x.dim() != 2:
        raise ValueError(f"quantize_nvfp4 expects a 2-D tensor, got {x.dim()}-D")
    x = x.contiguous()
    if x.numel() == 0:
        raise RuntimeError("quantize_nvfp4_dynamic: empty tensor")
    orows, ocols = x.shape
    rows, cols = (roundup(orows, 16), roundup(ocols, 16)) if pad_16x else (orows, ocols)
    if cols % 16:
        raise ValueError(f"K dimension must be divisible by 16 (got {cols}); pass pad_16x=True")
    qx = torch.empty((rows, cols // 2), dtype=torch.uint8, device=x.device)
    sx = torch.empty((roundup(rows, 128), roundup(cols // 16, 4)), dtype=torch.float8_e4m3fn, device=x.device)
    scale = torch.empty((), dtype=torch.float32, device=x.device)
    work = torch.empty(AMAX_WORKSPACE_BYTES // 4, dtype=torch.int32, device=x.device)
    _launch("ckh_quantize_nvfp4_dynamic", x, x.data_ptr(), float(divisor), scale.data_ptr(), qx.data_ptr(),
            sx.data_ptr(), rows, cols, orows, ocols, 0.0, DTYPE_TO_CODE[x.dtype], int(bool(hi_first)),
            work.data_ptr())
    return qx, sx, scale


def dequantize_nvfp4(qx: torch.Tensor, per_tensor_scale: torch.Tensor, block_scales: torch.Tensor,
                     output_type: torch.dtype = torch.bfloat16, hi_first: bool = True) -> torch.Tensor:
    qx = qx.contiguous()
    rows, half = qx.shape
    cols = 2 * half
    g = _scalar_on(per_tensor_scale, qx.device, "per_tensor_scale")
    sc = block_scales.contiguous()
    need = roundup(rows, 128) * roundup(cols // 16, 4)
    if cols % 16 or sc.nbytes < need:
        raise ValueError(f"dequantize_nvfp4: qx {tuple(qx.shape)} needs K % 16 == 0 and {need} scale bytes, "
                         f"got {sc.nbytes}")
    out = torch.empty((rows, cols), dtype=output_type, device=qx.device)
    _launch("ckh_dequantize_nvfp4", qx, qx.data_ptr(), g.data_ptr(), sc.data_ptr(), out.data_ptr(), rows, cols,
            DTYPE_TO_CODE[output_type], int(bool(hi_first)))
    return out


# ---------------------------------------------------------------------------- GEMMs
def _bias_args(bias: torch.Tensor | None, n: int, device) -> tuple[torch.Tensor | None, int]:
    if bias is None or bias.numel() == 0:
        return None, 0
    if bias.numel() != n:
        raise ValueError(f"bias must have {n} elements, got {bias.numel()}")
    b = bias.detach().reshape(-1).contiguous()
    if b.device != device:
        b = b.to(device)
    if b.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        b = b.to(torch.float32)
    return b, DTYPE_TO_CODE[b.dtype]


@functools.lru_cache(maxsize=256)
def _split_workspace_bytes(fn: str, m: int, n: int, k: int) -> int:
    return int(getattr(_lib, fn)(m, n, k))


def _gemm_workspace(m: int, n: int, k: int, device: torch.device,
                    fn: str = "ckh_scaled_mm_workspace_bytes") -> tuple[torch.Tensor | None, int]:
    """The workspace a GEMM splits K in at this shape (small tile grids), from torch's
    allocator (graph-capture safe), or (None, 0)."""
    nbytes = _split_workspace_bytes(fn, m, n, k)
    if nbytes <= 0:
        return None, 0
    return torch.empty(nbytes, dtype=torch.uint8, device=device), nbytes


def scaled_mm_mxfp8(a: torch.Tensor, b: torch.Tensor, block_scale_a: torch.Tensor,
                    block_scale_b: torch.Tensor, bias: torch.Tensor | None = None,
                    out_dtype: torch.dtype | None = None) -> torch.Tensor:
    out_dtype = out_dtype or torch.bfloat16
    a, b = a.contiguous(), b.contiguous()
    m, k = a.shape
    n, kb = b.shape
    if k != kb:
        raise ValueError(f"scaled_mm_mxfp8: K mismatch {k} vs {kb}")
    sa, sb = block_scale_a.contiguous(), block_scale_b.contiguous()
    for name, s, rows in (("block_scale_a", sa, m), ("block_scale_b", sb, n)):
        need = roundup(rows, 128) * roundup(k // 32, 4)
        if s.nbytes < need:
            raise ValueError(f"scaled_mm_mxfp8: {name} has {s.nbytes} bytes, needs {need}")
    bias_t, bias_code = _bias_args(bias, n, a.device)
    out = torch.empty((m, n), dtype=out_dtype, device=a.device)
    ws, ws_bytes = _gemm_workspace(m, n, k, a.device)
    _launch("ckh_scaled_mm_mxfp8", a, a.data_ptr(), b.data_ptr(), sa.data_ptr(), sb.data_ptr(), _ptr(bias_t),
            out.data_ptr(), m, n, k, DTYPE_TO_CODE[out_dtype], bias_code, _ptr(ws), ws_bytes)
    return out


def scaled_mm_fp8(a: torch.Tensor, b: torch.Tensor, scale_a: torch.Tensor, scale_b: torch.Tensor,
                  bias: torch.Tensor | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    out_dtype = out_dtype or torch.bfloat16
    a, b = a.contiguous(), b.contiguous()
    m, k = a.shape
    n, kb = b.shape
    if k != kb:
        raise ValueError(f"scaled_mm_fp8: K mismatch {k} vs {kb}")
    sa = _scalar_on(scale_a, a.device, "scale_a")
    sb = _scalar_on(scale_b, a.device, "scale_b")
    bias_t, bias_code = _bias_args(bias, n, a.device)
    out = torch.empty((m, n), dtype=out_dtype, device=a.device)
    ws, ws_bytes = _gemm_workspace(m, n, k, a.device)
    _launch("ckh_scaled_mm_fp8", a, a.data_ptr(), b.data_ptr(), sa.data_ptr(), sb.data_ptr(), _ptr(bias_t),
            out.data_ptr(), m, n, k, DTYPE_TO_CODE[out_dtype], bias_code, _ptr(ws), ws_bytes)
    return out


def scaled_mm_nvfp4(a: torch.Tensor, b: torch.Tensor, tensor_scale_a: torch.Tensor,
                    tensor_scale_b: torch.Tensor, block_scale_a: torch.Tensor,
                    block_scale_b: torch.Tensor, bias: torch.Tensor | None = None,
                    out_dtype: torch.dtype | None = None,
                    alpha: torch.Tensor | None = None) -> torch.Tensor:
    out_dtype = out_dtype or torch.bfloat16
    a, b = a.contiguous(), b.contiguous()
    m, ka = a.shape
    n, kb = b.shape
    if ka != kb:
        raise ValueError(f"scaled_mm_nvfp4: K mismatch {2 * ka} vs {2 * kb}")
    k = 2 * ka
    if alpha is None:  # the kernel multiplies the two tensor scales
        fn = "ckh_scaled_mm_nvfp4_scales"
        scales = (_scalar_on(tensor_scale_a, a.device, "tensor_scale_a"),
                  _scalar_on(tensor_scale_b, a.device, "tensor_scale_b"))
    else:
        fn, scales = "ckh_scaled_mm_nvfp4", (_scalar_on(alpha, a.device, "alpha"),)
    sa, sb = block_scale_a.contiguous(), block_scale_b.contiguous()
    for name, s, rows in (("block_scale_a", sa, m), ("block_scale_b", sb, n)):
        need = roundup(rows, 128) * roundup(k // 16, 4)
        if s.nbytes < need:
            raise ValueError(f"scaled_mm_nvfp4: {name} has {s.nbytes} bytes, needs {need}")
    bias_t, bias_code = _bias_args(bias, n, a.device)
    out = torch.empty((m, n), dtype=out_dtype, device=a.device)
    ws, ws_bytes = _gemm_workspace(m, n, k, a.device, "ckh_scaled_mm_nvfp4_workspace_bytes")
    _launch(fn, a, a.data_ptr(), b.data_ptr(), sa.data_ptr(), sb.data_ptr(), *(s.data_ptr() for s in scales),
            _ptr(bias_t), out.data_ptr(), m, n, k, DTYPE_TO_CODE[out_dtype], bias_code, _ptr(ws), ws_bytes)
    return out


# -------------------------------------------------------------- weight-only 4-bit linears
def quantize_int4(w: torch.Tensor, group_size: int) -> tuple[torch.Tensor, torch.Tensor]:
    n, k = w.shape
    if k % 32 or k == 0 or group_size < 32 or group_size % 32:
        raise ValueError(f"quantize_int4: K ({k}) and group_size ({group_size}) must be positive multiples of 32")
    w = w.contiguous()
    codes = torch.empty((n, k // 2), dtype=torch.uint8, device=w.device)
    scales = torch.empty((n, -(-k // group_size)), dtype=w.dtype, device=w.device)
    _launch("ckh_quantize_int4", w, w.data_ptr(), codes.data_ptr(), scales.data_ptr(), n, k, group_size,
            DTYPE_TO_CODE[w.dtype])
    return codes, scales


def _check_groups(name: str, codes_shape, scales_shape, zeros_shape, group_size: int) -> None:
    """Scales and zero points of the shape that the codes ask for."""
    if group_size < 32 or group_size % 32:
        raise ValueError(f"{name}: group_size must be a positive multiple of 32, got {group_size}")
    shape = (codes_shape[0], -(-2 * codes_shape[1] // group_size))
    if scales_shape != shape:
        raise ValueError(f"{name}: scales must be {list(shape)} for codes {list(codes_shape)} and group_size "
                         f"{group_size}, got {list(scales_shape)}")
    if zeros_shape is not None and zeros_shape != shape:
        raise ValueError(f"{name}: zeros must be {list(shape)}, got {list(zeros_shape)}")


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """t, contiguous and on a 16-byte boundary (copied where it is not)."""
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def _same_device(name: str, first: torch.Tensor, *others: torch.Tensor | None) -> None:
    device = first.get_device()
    for t in others:
        if t is not None and t.get_device() != device:
            raise ValueError(f"{name}: tensors on different devices ({first.device} and {t.device})")


def dequantize_int4(codes: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None, group_size: int,
                    output_type: torch.dtype = torch.bfloat16) -> torch.Tensor:
    _same_device("dequantize_int4", codes, scales, zeros)
    _check_groups("dequantize_int4", codes.shape, scales.shape, None if zeros is None else zeros.shape, group_size)
    codes, scales = _aligned(codes), scales.contiguous()
    zeros = None if zeros is None else zeros.contiguous()
    n, k = codes.shape[0], 2 * codes.shape[1]
    out = torch.empty((n, k), dtype=output_type, device=codes.device)
    _launch("ckh_dequantize_int4", codes, codes.data_ptr(), scales.data_ptr(), _ptr(zeros), out.data_ptr(), n, k,
            group_size, DTYPE_TO_CODE[scales.dtype], DTYPE_TO_CODE[output_type])
    return out


def _used_strides(shape: tuple, stride: tuple) -> tuple:
    """stride, where it places elements: 0 (the last: 1) for dimensions of one element and row-major
    for a tensor of none, whose own may be anything, and stay so in what contiguous() returns."""
    if 0 in shape:
        stride, step = [], 1
        for size in reversed(shape):
            stride.insert(0, step)
            step *= max(size, 1)
    *outer, last = (s if size != 1 else None for size, s in zip(shape, stride))
    return (*(s or 0 for s in outer), 1 if last is None else last)


@functools.lru_cache(maxsize=512)
def _linear_plan(x_shape, x_stride, x_dtype, codes_shape, scales_shape, scales_dtype, zeros_shape, group_size):
    """The call's checks, and its sizes as the C side takes them: (out's shape, sizes, codes behind
    them, workspace bytes), or None where x has to be copied."""
    n, half = codes_shape
    k = 2 * half
    x_stride = _used_strides(x_shape, x_stride)
    _check_groups("linear_int4", codes_shape, scales_shape, zeros_shape, group_size)
    if x_shape[-1] != k:
        raise ValueError(f"linear_int4: x has {x_shape[-1]} inputs, the weight {k}")
    m = 1
    for size in x_shape[:-1]:
        m *= size
    stride = k
    if len(x_shape) == 2 and m > 1:
        stride = x_stride[0]
    elif len(x_shape) > 2 and m > 0:  # rows of one step, or a copy
        step = 1
        for size, s in zip(x_shape[-2::-1], x_stride[-2::-1]):
            if size == 1:
                continue
            if step == 1:
                stride, step = s, size
            elif s != stride * step:
                return None
            else:
                step *= size
    if x_stride[-1] != 1 or stride % 8 or stride < k:
        return None
    nbytes = int(_lib.ckh_linear_int4_workspace_bytes(m, n, k, group_size))
    return ((*x_shape[:-1], n), (m, n, k, stride, group_size, DTYPE_TO_CODE[x_dtype], DTYPE_TO_CODE[scales_dtype]), nbytes)


def linear_int4(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None,
                bias: torch.Tensor | None = None, group_size: int = 128) -> torch.Tensor:
    _same_device("linear_int4", x, codes, scales, zeros, bias)
    rest = (codes.shape, scales.shape, scales.dtype, None if zeros is None else zeros.shape, group_size)
    plan = _linear_plan(x.shape, x.stride(), x.dtype, *rest)
    if plan is None or x.data_ptr() % 16:
        x = _aligned(x)
        plan = _linear_plan(x.shape, x.stride(), x.dtype, *rest)
    shape, sizes, nbytes = plan
    codes, scales = _aligned(codes), scales.contiguous()
    if zeros is not None:
        zeros = zeros.contiguous()
    bias_code = 0
    if bias is not None:
        bias, bias_code = _bias_args(bias, codes.shape[0], x.device)
    out = torch.empty(shape, dtype=x.dtype, device=x.device)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device) if nbytes else None
    _launch("ckh_linear_int4", x, x.data_ptr(), codes.data_ptr(), scales.data_ptr(), _ptr(zeros), _ptr(bias),
            out.data_ptr(), *sizes, bias_code, _ptr(ws), nbytes)
    return out


# -------------------------------------------------------- key-value cache held in pages
# A call's checks depend on its tensors' shapes, strides and dtypes alone, and cost more than the
# call itself (14 us of paged_write's 22 on one token of each of 48 sequences), so each is a
# function of those whose answers are kept: the call's sizes and strides as the C side takes them,
# or None where a tensor that may be copied does not lie on 16-byte rows.
def _strides(*values: int):
    return (_i64 * len(values))(*values)


def _on_rows16(stride: tuple, size: int) -> bool:
    """Whether the last dimension is contiguous and the others step by multiples of 16 bytes."""
    return stride[-1] == 1 and not any(s * size % 16 for s in stride[:-1])


def _cache_pair(name: str, k_shape, k_stride, k_dtype, v_shape, v_stride, v_dtype) -> tuple[tuple, tuple]:
    """What every call asks of the two caches: one shape and dtype, rows that 16-byte pieces fit.
    They are used in place, so nothing is copied to fit.  Returns their strides."""
    if k_shape != v_shape or k_dtype != v_dtype:
        raise ValueError(f"{name}: k_cache {list(k_shape)} {k_dtype} and v_cache {list(v_shape)} {v_dtype} differ")
    strides = _used_strides(k_shape, k_stride), _used_strides(v_shape, v_stride)
    for stride in strides:
        if not _on_rows16(stride, k_dtype.itemsize):
            raise ValueError(f"{name}: a cache of strides {stride} is not 16-byte aligned with head_dim contiguous")
    return strides


def _cache_pointers(name: str, k_cache: torch.Tensor, v_cache: torch.Tensor) -> tuple[int, int]:
    k, v = k_cache.data_ptr(), v_cache.data_ptr()
    if (k | v) & 15:
        raise ValueError(f"{name}: a cache is not 16-byte aligned with head_dim contiguous")
    return k, v


def _rows16(t: torch.Tensor) -> torch.Tensor:
    """t, its last dimension contiguous and its rows on 16-byte boundaries (copied where they are not)."""
    if not t.data_ptr() % 16 and _on_rows16(_used_strides(t.shape, t.stride()), t.element_size()):
        return t
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


@functools.lru_cache(maxsize=512)
def _attention_plan(q_shape, q_stride, q_dtype, k_shape, k_stride, k_dtype, v_shape, v_stride, v_dtype, table_shape,
                    table_stride, sequences, window, sinks, scale):
    k_stride, v_stride = _cache_pair("paged_attention", k_shape, k_stride, k_dtype, v_shape, v_stride, v_dtype)
    batch, heads, dim = q_shape
    pages, page_size, kv_heads, cache_dim = k_shape
    if dim != cache_dim or kv_heads == 0 or heads % kv_heads:
        raise ValueError(f"paged_attention: q {list(q_shape)} does not fit a cache of {kv_heads} heads of {cache_dim}")
    if dim not in (64, 96, 128, 256):
        raise ValueError(f"paged_attention: head_dim {dim} is not 64, 96, 128 or 256")
    if k_dtype not in (q_dtype, torch.float8_e4m3fn):
        raise ValueError(f"paged_attention: a cache of {k_dtype} with queries of {q_dtype}")
    if table_shape[0] != batch or sequences != batch:
        raise ValueError(f"paged_attention: page_table {list(table_shape)} and {sequences} lengths for {batch} sequences")
    if window < 0 or sinks < 0:
        raise ValueError(f"paged_attention: window ({window}) and sinks ({sinks}) must not be negative")
    q_stride = _used_strides(q_shape, q_stride)
    if not _on_rows16(q_stride, 2):
        return None
    max_pages = table_shape[1]
    nbytes = int(_lib.ckh_paged_attention_workspace_bytes(batch, heads, kv_heads, dim, page_size, max_pages))
    return ((batch, heads, kv_heads, dim, pages, page_size, max_pages, table_stride[0],
             _strides(*q_stride[:2], *k_stride[:3], *v_stride[:3]), window, sinks, dim ** -0.5 if scale is None else scale,
             DTYPE_TO_CODE[q_dtype], DTYPE_TO_CODE[k_dtype]), nbytes)


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                    lengths: torch.Tensor, scale: float | None = None, window: int = 0, sinks: int = 0,
                    k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None) -> torch.Tensor:
    _same_device("paged_attention", q, k_cache, v_cache, page_table, lengths)
    lengths = lengths.contiguous()
    if page_table.stride(1) != 1 and page_table.shape[1] > 1:
        page_table = page_table.contiguous()
    rest = (k_cache.shape, k_cache.stride(), k_cache.dtype, v_cache.shape, v_cache.stride(), v_cache.dtype, page_table.shape,
            page_table.stride(), lengths.shape[0], window, sinks, scale)
    plan = _attention_plan(q.shape, q.stride(), q.dtype, *rest)
    if plan is None or q.data_ptr() % 16:
        q = _rows16(q)
        plan = _attention_plan(q.shape, q.stride(), q.dtype, *rest)
    sizes, nbytes = plan
    k, v = _cache_pointers("paged_attention", k_cache, v_cache)
    if k_scale is not None:
        k_scale = _scalar_on(k_scale, q.device, "k_scale")
    if v_scale is not None:
        v_scale = _scalar_on(v_scale, q.device, "v_scale")
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
    _launch("ckh_paged_attention", q, q.data_ptr(), k, v, page_table.data_ptr(), lengths.data_ptr(), _ptr(k_scale),
            _ptr(v_scale), out.data_ptr(), *sizes, _ptr(ws), nbytes)
    return out


@functools.lru_cache(maxsize=512)
def _write_plan(key_shape, key_stride, key_dtype, value_shape, value_stride, value_dtype, k_shape, k_stride, k_dtype, v_shape,
                v_stride, v_dtype, slots, slots_dtype):
    k_stride, v_stride = _cache_pair("paged_write", k_shape, k_stride, k_dtype, v_shape, v_stride, v_dtype)
    tokens, kv_heads, dim = key_shape
    pages, page_size = k_shape[:2]
    if value_shape != key_shape or value_dtype != key_dtype or k_shape[2:] != key_shape[1:]:
        raise ValueError(f"paged_write: key {list(key_shape)} {key_dtype}, value {list(value_shape)} {value_dtype} and "
                         f"a cache {list(k_shape)} do not fit")
    if k_dtype not in (key_dtype, torch.float8_e4m3fn):
        raise ValueError(f"paged_write: {key_dtype} into a cache of {k_dtype}")
    if dim % 16:
        raise ValueError(f"paged_write: head_dim {dim} is not a multiple of 16")
    if slots != tokens:
        raise ValueError(f"paged_write: {slots} slots for {tokens} tokens")
    key_stride, value_stride = _used_strides(key_shape, key_stride), _used_strides(value_shape, value_stride)
    if not (_on_rows16(key_stride, 2) and _on_rows16(value_stride, 2)):
        return None
    return (tokens, kv_heads, dim, pages, page_size, _strides(*key_stride[:2], *value_stride[:2], *k_stride[:3], *v_stride[:3]),
            DTYPE_TO_CODE[key_dtype], DTYPE_TO_CODE[k_dtype], int(slots_dtype == torch.int64))


def paged_write(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                slots: torch.Tensor, k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None) -> None:
    _same_device("paged_write", key, value, k_cache, v_cache, slots)
    rest = (k_cache.shape, k_cache.stride(), k_cache.dtype, v_cache.shape, v_cache.stride(), v_cache.dtype, slots.shape[0],
            slots.dtype)
    plan = _write_plan(key.shape, key.stride(), key.dtype, value.shape, value.stride(), value.dtype, *rest)
    if plan is None or (key.data_ptr() | value.data_ptr()) & 15:
        key, value = _rows16(key), _rows16(value)
        plan = _write_plan(key.shape, key.stride(), key.dtype, value.shape, value.stride(), value.dtype, *rest)
    k, v = _cache_pointers("paged_write", k_cache, v_cache)
    if k_scale is not None:
        k_scale = _scalar_on(k_scale, key.device, "k_scale")
    if v_scale is not None:
        v_scale = _scalar_on(v_scale, key.device, "v_scale")
    if (k_scale is not None or v_scale is not None) and k_cache.dtype != torch.float8_e4m3fn:
        raise ValueError(f"paged_write: k_scale and v_scale are for a cache of float8_e4m3fn, not {k_cache.dtype}")
    slots = slots.contiguous()
    _launch("ckh_paged_write", key, key.data_ptr(), value.data_ptr(), k, v, slots.data_ptr(), _ptr(k_scale), _ptr(v_scale), *plan)


@functools.lru_cache(maxsize=512)
def _copy_plan(k_shape, k_stride, k_dtype, v_shape, v_stride, v_dtype, src_shape, src_dtype, dst_shape, dst_dtype):
    k_stride, v_stride = _cache_pair("paged_copy", k_shape, k_stride, k_dtype, v_shape, v_stride, v_dtype)
    if len(k_shape) not in (4, 5):
        raise ValueError(f"paged_copy: a cache has 4 dimensions, or 5 with the layers first, got {len(k_shape)}")
    if src_shape != dst_shape or src_dtype != dst_dtype:
        raise ValueError(f"paged_copy: src {list(src_shape)} {src_dtype} and dst {list(dst_shape)} {dst_dtype} differ")
    layers = k_shape[0] if len(k_shape) == 5 else 1
    pages, page_size, kv_heads, dim = k_shape[-4:]
    if dim * k_dtype.itemsize % 16:
        raise ValueError(f"paged_copy: a head of {dim} elements is not a multiple of 16 bytes")
    if layers == 1:
        k_stride, v_stride = (0, *k_stride[-4:]), (0, *v_stride[-4:])
    return (layers, src_shape[0], kv_heads, dim, pages, page_size, _strides(*k_stride[:4], *v_stride[:4]), k_dtype.itemsize,
            int(src_dtype == torch.int64))


def paged_copy(k_cache: torch.Tensor, v_cache: torch.Tensor, src: torch.Tensor, dst: torch.Tensor) -> None:
    _same_device("paged_copy", k_cache, v_cache, src, dst)
    k, v = _cache_pointers("paged_copy", k_cache, v_cache)
    plan = _copy_plan(k_cache.shape, k_cache.stride(), k_cache.dtype, v_cache.shape, v_cache.stride(), v_cache.dtype,
                      src.shape, src.dtype, dst.shape, dst.dtype)
    src, dst = src.contiguous(), dst.contiguous()
    _launch("ckh_paged_copy", k_cache, k, v, src.data_ptr(), dst.data_ptr(), *plan)


@functools.lru_cache(maxsize=512)
def _window_plan(q_shape, q_stride, q_dtype, k_shape, k_stride, k_dtype, v_shape, v_stride, v_dtype, sequences, window, sinks,
                 scale):
    batch, queries, heads, dim = q_shape
    keys, kv_heads = k_shape[1:3]
    if k_shape != v_shape or k_shape[0] != batch or k_shape[3] != dim or kv_heads == 0 or heads % kv_heads:
        raise ValueError(f"window_attention: q {list(q_shape)}, k {list(k_shape)} and v {list(v_shape)} do not fit")
    if k_dtype != q_dtype or v_dtype != q_dtype:
        raise ValueError(f"window_attention: q, k and v of different dtypes ({q_dtype}, {k_dtype}, {v_dtype})")
    if dim not in (64, 96, 128, 256):
        raise ValueError(f"window_attention: head_dim {dim} is not 64, 96, 128 or 256")
    if window < 0 or sinks < 0:
        raise ValueError(f"window_attention: window ({window}) and sinks ({sinks}) must not be negative")
    if sequences is not None and sequences != batch:
        raise ValueError(f"window_attention: {sequences} lengths for a batch of {batch}")
    q_stride, k_stride, v_stride = (_used_strides(k_shape if i else q_shape, s) for i, s in enumerate((q_stride, k_stride, v_stride)))
    overlap = keys > 1 and min(k_stride[1], v_stride[1]) < dim  # broadcast keys have no rows of their own
    if overlap or not (_on_rows16(q_stride, 2) and _on_rows16(k_stride, 2) and _on_rows16(v_stride, 2)):
        return None
    nbytes = int(_lib.ckh_window_attention_workspace_bytes(batch, queries, keys, heads, kv_heads, dim, window, sinks))
    return ((batch, queries, keys, heads, kv_heads, dim, _strides(*q_stride[:3], *k_stride[:3], *v_stride[:3]), window, sinks,
             dim ** -0.5 if scale is None else scale, DTYPE_TO_CODE[q_dtype]), nbytes)


def _own_rows16(t: torch.Tensor) -> torch.Tensor:
    """_rows16 of keys or values, copied too where tokens share memory."""
    return _rows16(t.contiguous() if t.shape[1] > 1 and t.stride(1) < t.shape[3] else t)


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int = 0, sinks: int = 0,
                     lengths: torch.Tensor | None = None, scale: float | None = None) -> torch.Tensor:
    _same_device("window_attention", q, k, v, lengths)
    rest = (None if lengths is None else lengths.shape[0], window, sinks, scale)
    plan = _window_plan(q.shape, q.stride(), q.dtype, k.shape, k.stride(), k.dtype, v.shape, v.stride(), v.dtype, *rest)
    if plan is None or (q.data_ptr() | k.data_ptr() | v.data_ptr()) & 15:
        q, k, v = _rows16(q), _own_rows16(k), _own_rows16(v)
        plan = _window_plan(q.shape, q.stride(), q.dtype, k.shape, k.stride(), k.dtype, v.shape, v.stride(), v.dtype, *rest)
    if lengths is not None:
        lengths = lengths.contiguous()
    sizes, nbytes = plan
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
    _launch("ckh_window_attention", q, q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(lengths), out.data_ptr(), *sizes,
            _ptr(ws), nbytes)
    return out


@functools.lru_cache(maxsize=512)
def _rope_write_plan(q_shape, q_stride, q_dtype, key_shape, key_stride, key_dtype, value_shape, value_stride, value_dtype, k_shape,
                     k_stride, k_dtype, v_shape, v_stride, v_dtype, positions, positions_dtype, slots, slots_dtype, rates, interleaved,
                     magnitude):
    k_stride, v_stride = _cache_pair("paged_write_rope", k_shape, k_stride, k_dtype, v_shape, v_stride, v_dtype)
    tokens, heads, dim = q_shape
    kv_heads = key_shape[1]
    pages, page_size = k_shape[:2]
    if (value_shape != key_shape or key_shape[0] != tokens or key_shape[2] != dim or k_shape[2:] != key_shape[1:]
            or not q_dtype == key_dtype == value_dtype):
        raise ValueError(f"paged_write_rope: q {list(q_shape)} {q_dtype}, key {list(key_shape)} {key_dtype}, value {list(value_shape)} "
                         f"{value_dtype} and a cache {list(k_shape)} do not fit")
    if k_dtype not in (key_dtype, torch.float8_e4m3fn):
        raise ValueError(f"paged_write_rope: {key_dtype} into a cache of {k_dtype}")
    if dim % 16:
        raise ValueError(f"paged_write_rope: head_dim {dim} is not a multiple of 16")
    if 2 * rates > dim:
        raise ValueError(f"paged_write_rope: {rates} rates turn more than head_dim {dim}")
    if positions != tokens or slots != tokens:
        raise ValueError(f"paged_write_rope: {positions} positions and {slots} slots for {tokens} tokens")
    strides = [_used_strides(*t) for t in ((q_shape, q_stride), (key_shape, key_stride), (value_shape, value_stride))]
    if not all(_on_rows16(s, 2) for s in strides):
        return None
    return (tokens, heads, kv_heads, dim, 2 * rates, pages, page_size,
            _strides(*(s for t in strides for s in t[:2]), *k_stride[:3], *v_stride[:3]), int(interleaved), magnitude,
            DTYPE_TO_CODE[key_dtype], DTYPE_TO_CODE[k_dtype], int(positions_dtype == torch.int64), int(slots_dtype == torch.int64))


def paged_write_rope(q: torch.Tensor, key: torch.Tensor, value: torch.Tensor, positions: torch.Tensor, rates: torch.Tensor,
                     k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor, interleaved: bool = True,
                     magnitude: float = 1.0, k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                     keep_key: bool = False) -> tuple[torch.Tensor, torch.Tensor | None]:
    """(q', key'); key' is None where it is not kept."""
    _same_device("paged_write_rope", q, key, value, positions, rates, k_cache, v_cache, slots)
    rest = (k_cache.shape, k_cache.stride(), k_cache.dtype, v_cache.shape, v_cache.stride(), v_cache.dtype, positions.shape[0],
            positions.dtype, slots.shape[0], slots.dtype, rates.shape[0], interleaved, magnitude)
    plan = _rope_write_plan(q.shape, q.stride(), q.dtype, key.shape, key.stride(), key.dtype, value.shape, value.stride(), value.dtype,
                            *rest)
    if plan is None or (q.data_ptr() | key.data_ptr() | value.data_ptr()) & 15:
        q, key, value = _rows16(q), _rows16(key), _rows16(value)
        plan = _rope_write_plan(q.shape, q.stride(), q.dtype, key.shape, key.stride(), key.dtype, value.shape, value.stride(),
                                value.dtype, *rest)
    k, v = _cache_pointers("paged_write_rope", k_cache, v_cache)
    if k_scale is not None:
        k_scale = _scalar_on(k_scale, key.device, "k_scale")
    if v_scale is not None:
        v_scale = _scalar_on(v_scale, key.device, "v_scale")
    if (k_scale is not None or v_scale is not None) and k_cache.dtype != torch.float8_e4m3fn:
        raise ValueError(f"paged_write_rope: k_scale and v_scale are for a cache of float8_e4m3fn, not {k_cache.dtype}")
    positions, rates, slots = positions.contiguous(), rates.contiguous(), slots.contiguous()
    out = _like(q)
    key_out = _like(key) if keep_key else None
    _launch("ckh_paged_write_rope", q, q.data_ptr(), key.data_ptr(), value.data_ptr(), positions.data_ptr(), rates.data_ptr(),
            out.data_ptr(), _ptr(key_out), k, v, slots.data_ptr(), _ptr(k_scale), _ptr(v_scale), *plan)
    return out, key_out


@functools.lru_cache(maxsize=512)
def _shared_plan(q_shape, q_stride, q_dtype, k_shape, k_stride, k_dtype, v_shape, v_stride, v_dtype, table_shape, table_stride,
                 sequences, starts, shared, scale):
    k_stride, v_stride = _cache_pair("shared_attention", k_shape, k_stride, k_dtype, v_shape, v_stride, v_dtype)
    batch, heads, dim = q_shape
    pages, page_size, kv_heads, cache_dim = k_shape
    if dim != cache_dim or kv_heads == 0 or heads % kv_heads:
        raise ValueError(f"shared_attention: q {list(q_shape)} does not fit a cache of {kv_heads} heads of {cache_dim}")
    if dim not in (64, 96, 128, 256):
        raise ValueError(f"shared_attention: head_dim {dim} is not 64, 96, 128 or 256")
    if k_dtype not in (q_dtype, torch.float8_e4m3fn):
        raise ValueError(f"shared_attention: a cache of {k_dtype} with queries of {q_dtype}")
    if table_shape[0] != batch or sequences != batch:
        raise ValueError(f"shared_attention: page_table {list(table_shape)} and {sequences} lengths for {batch} sequences")
    if starts != shared + 1:
        raise ValueError(f"shared_attention: {starts} group bounds for {shared} groups, which need one more than that")
    q_stride = _used_strides(q_shape, q_stride)
    if not _on_rows16(q_stride, 2):
        return None
    nbytes = int(_lib.ckh_shared_attention_workspace_bytes(batch, heads, kv_heads, dim, shared, page_size, table_shape[1]))
    return ((batch, heads, kv_heads, dim, shared, pages, page_size, table_shape[1], table_stride[0],
             _strides(*q_stride[:2], *k_stride[:3], *v_stride[:3]), dim ** -0.5 if scale is None else scale,
             DTYPE_TO_CODE[q_dtype], DTYPE_TO_CODE[k_dtype]), nbytes)


def shared_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor,
                     groups: torch.Tensor, shared: torch.Tensor, scale: float | None = None, k_scale: torch.Tensor | None = None,
                     v_scale: torch.Tensor | None = None) -> torch.Tensor:
    _same_device("shared_attention", q, k_cache, v_cache, page_table, lengths, groups, shared)
    lengths, groups, shared = lengths.contiguous(), groups.contiguous(), shared.contiguous()
    if page_table.stride(1) != 1 and page_table.shape[1] > 1:
        page_table = page_table.contiguous()
    rest = (k_cache.shape, k_cache.stride(), k_cache.dtype, v_cache.shape, v_cache.stride(), v_cache.dtype, page_table.shape,
            page_table.stride(), lengths.shape[0], groups.shape[0], shared.shape[0], scale)
    plan = _shared_plan(q.shape, q.stride(), q.dtype, *rest)
    if plan is None or q.data_ptr() % 16:
        q = _rows16(q)
        plan = _shared_plan(q.shape, q.stride(), q.dtype, *rest)
    sizes, nbytes = plan
    k, v = _cache_pointers("shared_attention", k_cache, v_cache)
    if k_scale is not None:
        k_scale = _scalar_on(k_scale, q.device, "k_scale")
    if v_scale is not None:
        v_scale = _scalar_on(v_scale, q.device, "v_scale")
    out = _like(q)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
    _launch("ckh_shared_attention", q, q.data_ptr(), k, v, page_table.data_ptr(), lengths.data_ptr(), groups.data_ptr(),
            shared.data_ptr(), _ptr(k_scale), _ptr(v_scale), out.data_ptr(), *sizes, _ptr(ws), nbytes)
    return out


# ------------------------------------------------------------------------------- norms
def _row_step(shape: tuple, stride: tuple) -> int | None:
    """The elements between the rows of [..., cols], or None where they are not one step apart (or cols not contiguous)."""
    if 0 in shape:
        return shape[-1]
    *outer, last = _used_strides(shape, stride)
    if last != 1:
        return None
    step, run = shape[-1], None
    for size, s in zip(shape[-2::-1], outer[::-1]):
        if size == 1:
            continue
        if run is None:
            step, run = s, size
        elif s != step * run:
            return None
        else:
            run *= size
    return step


@functools.lru_cache(maxsize=512)
def _norm_plan(name, x_shape, x_stride, x_dtype, weight_shape, weight_dtype, residual_shape, residual_stride, residual_dtype, output_type,
               pad_32x):
    """The call's checks, and its sizes as the C side takes them (result's shape, scales' shape, sizes, the codes of the
    dtypes), or None where x or the residual has to be copied."""
    cols = x_shape[-1]
    if weight_shape is not None and weight_shape[0] != cols:
        raise ValueError(f"{name}: {weight_shape[0]} weights for rows of {cols}")
    if residual_shape is not None and (residual_shape != x_shape or residual_dtype != x_dtype):
        raise ValueError(f"{name}: x {list(x_shape)} {x_dtype} and residual {list(residual_shape)} {residual_dtype} differ")
    if cols > 65536:
        raise ValueError(f"{name}: rows of {cols} elements, 65536 at most")
    rows = 1
    for size in x_shape[:-1]:
        rows *= size
    mx = pad_32x is not None
    out_rows, out_cols = (roundup(rows, 32), roundup(cols, 32)) if pad_32x else (rows, cols)
    if mx and out_cols % 32:
        raise ValueError(f"K dimension must be divisible by 32 (got {cols}); pass pad_32x=True")
    x_step = _row_step(x_shape, x_stride)
    r_step = 0 if residual_shape is None else _row_step(residual_shape, residual_stride)
    if x_step is None or r_step is None:
        return None
    return ((out_rows, out_cols) if mx else x_shape, (roundup(rows, 128), roundup(out_cols // 32, 4)),
            (rows, cols, out_rows, out_cols, x_step, r_step),
            (DTYPE_TO_CODE[x_dtype], 0 if weight_dtype is None else DTYPE_TO_CODE[weight_dtype], DTYPE_TO_CODE[output_type], int(mx)))


def _rms_norm(name: str, x: torch.Tensor, weight: torch.Tensor | None, residual: torch.Tensor | None, eps: float,
              scale: torch.Tensor | None, output_type: torch.dtype, pad_32x: bool | None):
    """(result, scales or None, h or None)."""
    _same_device(name, x, weight, residual)
    w = (None, None) if weight is None else (weight.shape, weight.dtype)
    r = (None, None, None) if residual is None else (residual.shape, residual.stride(), residual.dtype)
    plan = _norm_plan(name, x.shape, x.stride(), x.dtype, *w, *r, output_type, pad_32x)
    if plan is None:
        x = x.contiguous()
        if residual is not None:
            residual = residual.contiguous()
            r = (residual.shape, residual.stride(), residual.dtype)
        plan = _norm_plan(name, x.shape, x.stride(), x.dtype, *w, *r, output_type, pad_32x)
    shape, scales_shape, sizes, codes = plan
    plain = x.is_contiguous()  # empty_like takes half of empty's time
    same = plain and shape == x.shape
    y = torch.empty_like(x, dtype=output_type) if same else torch.empty(shape, dtype=output_type, device=x.device)
    scales = torch.empty(scales_shape, dtype=torch.float8_e8m0fnu, device=x.device) if codes[3] else None
    h = None
    if residual is not None:
        h = torch.empty_like(x) if plain else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if sizes[0] and sizes[1]:
        if weight is not None:
            weight = weight.contiguous()
        _launch("ckh_rms_norm", x, x.data_ptr(), _ptr(residual), _ptr(weight), _ptr(scale), y.data_ptr(), _ptr(scales), _ptr(h), *sizes, eps,
                *codes)
    return y, scales, h


def rms_norm(x: torch.Tensor, weight: torch.Tensor | None = None, residual: torch.Tensor | None = None,
             eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor | None]:
    """(y, h); h is None where there is no residual."""
    y, _, h = _rms_norm("rms_norm", x, weight, residual, eps, None, x.dtype, None)
    return y, h


def rms_norm_fp8(x: torch.Tensor, scale: torch.Tensor, weight: torch.Tensor | None = None, residual: torch.Tensor | None = None,
                 eps: float = 1e-6, output_type: torch.dtype = torch.float8_e4m3fn) -> tuple[torch.Tensor, torch.Tensor | None]:
    codes, _, h = _rms_norm("rms_norm_fp8", x, weight, residual, eps, _scalar_on(scale, x.device, "scale"), output_type, None)
    return codes, h


def rms_norm_mxfp8(x: torch.Tensor, weight: torch.Tensor | None = None, residual: torch.Tensor | None = None, eps: float = 1e-6,
                   pad_32x: bool = False) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
    return _rms_norm("rms_norm_mxfp8", x, weight, residual, eps, None, torch.float8_e4m3fn, bool(pad_32x))


# ---------------------------------------------------------------------------- sampling
@functools.lru_cache(maxsize=256)
def _sample_workspace_bytes(rows: int, vocab: int) -> int:
    return int(_lib.ckh_sample_workspace_bytes(rows, vocab))


def sample_tokens(logits: torch.Tensor, u: torch.Tensor, temperature: torch.Tensor | float = 1.0, top_k: torch.Tensor | int = 0,
                  top_p: torch.Tensor | float = 1.0, min_p: torch.Tensor | float = 0.0) -> torch.Tensor:
    """Each of the four is a number for all rows, or a tensor of one a row."""
    rows, vocab = logits.shape
    if u.shape[0] != rows:
        raise ValueError(f"sample_tokens: {u.shape[0]} random numbers for {rows} rows")
    if vocab == 0:
        raise ValueError("sample_tokens: no logits")
    per_row, common = [], []
    for name, value, dtype in (("temperature", temperature, torch.float32), ("top_k", top_k, torch.int32), ("top_p", top_p, torch.float32),
                               ("min_p", min_p, torch.float32)):
        if isinstance(value, torch.Tensor):
            if value.shape != (rows,) or value.dtype != dtype:
                raise ValueError(f"sample_tokens: {name} {list(value.shape)} {value.dtype} is not one {dtype} for each of {rows} rows")
            per_row.append(value.contiguous())
            common.append(0)
        else:
            per_row.append(None)
            common.append(value)
    _same_device("sample_tokens", logits, u, *per_row)
    if vocab > 1 and logits.stride(1) != 1:
        logits = logits.contiguous()
    u = u.contiguous()
    out = torch.empty(rows, dtype=torch.int64, device=logits.device)
    nbytes = _sample_workspace_bytes(rows, vocab)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=logits.device)
    _launch("ckh_sample", logits, logits.data_ptr(), u.data_ptr(), *(_ptr(t) for t in per_row), common[0], common[1], common[2], common[3],
            out.data_ptr(), rows, vocab, logits.stride(0) if rows > 1 else vocab, DTYPE_TO_CODE[logits.dtype], ws.data_ptr(), nbytes)
    return out


# ----------------------------------------------------------------------------- RoPE
def _rope_call(xq: torch.Tensor, xk: torch.Tensor | None, freqs_cis: torch.Tensor):
    if xq.dim() != 4 or freqs_cis.dim() != 6:
        raise ValueError(f"apply_rope expects 4-D x and 6-D freqs, got {xq.dim()}-D and {freqs_cis.dim()}-D")
    xq = xq.contiguous()
    xk = xk.contiguous() if xk is not None else None
    b, d1, d2, hd = xq.shape
    fb, fd1, fd2 = freqs_cis.shape[:3]
    if tuple(freqs_cis.shape[3:]) != (hd // 2, 2, 2) or hd % 2:
        raise ValueError(f"freqs_cis inner dims {tuple(freqs_cis.shape[3:])} != ({hd // 2}, 2, 2)")
    if d2 == 1 and fd2 != 1:
        raise ValueError(f"x dim 2 is 1 but freqs dim 2 is {fd2}: shapes do not broadcast back to x")
    f = freqs_cis
    if f.device != xq.device:
        f = f.to(xq.device)
    if f.stride(5) != 1 or f.stride(4) != 2 or f.stride(3) != 4:
        f = f.contiguous()
    oq = torch.empty_like(xq)
    ok = torch.empty_like(xk) if xk is not None else None
    _launch("ckh_apply_rope", xq, xq.data_ptr(), _ptr(xk), f.data_ptr(), oq.data_ptr(), _ptr(ok), b, d1, d2, hd,
            fb, fd1, fd2, xq.stride(0), xq.stride(1), xq.stride(2), f.stride(0), f.stride(1), f.stride(2),
            DTYPE_TO_CODE[xq.dtype], DTYPE_TO_CODE[f.dtype])
    return oq, ok


def apply_rope1(x: torch.Tensor, freqs_cis: torch.Tensor) -> torch.Tensor:
    return _rope_call(x, None, freqs_cis)[0]


def apply_rope(xq: torch.Tensor, xk: torch.Tensor, freqs_cis: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    if xq.shape != xk.shape or xq.dtype != xk.dtype:
        return apply_rope1(xq, freqs_cis), apply_rope1(xk, freqs_cis)
    return _rope_call(xq, xk, freqs_cis)


# ---------------------------------------------------------------------- registration
def _build_constraints() -> dict:
    from ...constraints import DivisibleBy, ExactDims, FunctionConstraints, MinDims, ParamConstraint

    dev = frozenset({"cuda"})
    floats = frozenset({torch.float32, torch.float16, torch.bfloat16})
    half = frozenset({torch.float16, torch.bfloat16})
    fp8 = frozenset({torch.float8_e4m3fn, torch.float8_e5m2})
    f32 = frozenset({torch.float32})
    u8 = frozenset({torch.uint8})
    i32, ints = frozenset({torch.int32}), frozenset({torch.int32, torch.int64})
    e4m3 = frozenset({torch.float8_e4m3fn})

    def fc(**params):
        return FunctionConstraints(params=params, default_devices=dev, required_arch=REQUIRED_ARCH)

    two_d = (ExactDims(2),)
    return {
        "amax_scale": fc(x=ParamConstraint(dtypes=floats)),
        "quantize_per_tensor_fp8": fc(x=ParamConstraint(dtypes=floats), scale=ParamConstraint(dtypes=f32, devices=frozenset({"cuda", "cpu"})),
                                      output_type=ParamConstraint(dtypes=fp8)),
        "dequantize_per_tensor_fp8": fc(x=ParamConstraint(dtypes=fp8), scale=ParamConstraint(dtypes=floats, devices=frozenset({"cuda", "cpu"})),
                                        output_type=ParamConstraint(dtypes=floats)),
        "quantize_fp8_dynamic": fc(x=ParamConstraint(dtypes=floats), output_type=ParamConstraint(dtypes=fp8)),
        "quantize_mxfp8": fc(x=ParamConstraint(dtypes=floats, shape_rules=two_d)),
        "dequantize_mxfp8": fc(qx=ParamConstraint(dtypes=frozenset({torch.float8_e4m3fn}),
                                                  shape_rules=two_d + (DivisibleBy(1, 32),)),
                               block_scales=ParamConstraint(dtypes=frozenset({torch.float8_e8m0fnu})),
                               output_type=ParamConstraint(dtypes=floats)),
        "quantize_nvfp4": fc(x=ParamConstraint(dtypes=floats, shape_rules=two_d),
                             per_tensor_scale=ParamConstraint(dtypes=f32, devices=frozenset({"cuda", "cpu"}))),
        "quantize_nvfp4_dynamic": fc(x=ParamConstraint(dtypes=floats, shape_rules=two_d)),
        "dequantize_nvfp4": fc(qx=ParamConstraint(dtypes=frozenset({torch.uint8}),
                                                  shape_rules=two_d + (DivisibleBy(1, 8),)),
                               per_tensor_scale=ParamConstraint(dtypes=f32, devices=frozenset({"cuda", "cpu"})),
                               block_scales=ParamConstraint(dtypes=frozenset({torch.float8_e4m3fn})),
                               output_type=ParamConstraint(dtypes=floats)),
        "scaled_mm_mxfp8": fc(a=ParamConstraint(dtypes=frozenset({torch.float8_e4m3fn}),
                                                shape_rules=two_d + (DivisibleBy(1, 32),)),
                              b=ParamConstraint(dtypes=frozenset({torch.float8_e4m3fn}),
                                                shape_rules=two_d + (DivisibleBy(1, 32),)),
                              block_scale_a=ParamConstraint(dtypes=frozenset({torch.float8_e8m0fnu})),
                              block_scale_b=ParamConstraint(dtypes=frozenset({torch.float8_e8m0fnu})),
                              bias=ParamConstraint(dtypes=floats),
                              out_dtype=ParamConstraint(dtypes=floats)),
        "scaled_mm_fp8": fc(a=ParamConstraint(dtypes=frozenset({torch.float8_e4m3fn}),
                                              shape_rules=two_d + (DivisibleBy(1, 16),)),
                            b=ParamConstraint(dtypes=frozenset({torch.float8_e4m3fn}),
                                              shape_rules=two_d + (DivisibleBy(1, 16),)),
                            scale_a=ParamConstraint(dtypes=f32, devices=frozenset({"cuda", "cpu"})),
                            scale_b=ParamConstraint(dtypes=f32, devices=frozenset({"cuda", "cpu"})),
                            bias=ParamConstraint(dtypes=floats),
                            out_dtype=ParamConstraint(dtypes=floats)),
        "scaled_mm_nvfp4": fc(a=ParamConstraint(dtypes=frozenset({torch.uint8}),
                                                shape_rules=two_d + (DivisibleBy(1, 16),)),
                              b=ParamConstraint(dtypes=frozenset({torch.uint8}),
                                                shape_rules=two_d + (DivisibleBy(1, 16),)),
                              tensor_scale_a=ParamConstraint(dtypes=f32, devices=frozenset({"cuda", "cpu"})),
                              tensor_scale_b=ParamConstraint(dtypes=f32, devices=frozenset({"cuda", "cpu"})),
                              block_scale_a=ParamConstraint(dtypes=frozenset({torch.float8_e4m3fn})),
                              block_scale_b=ParamConstraint(dtypes=frozenset({torch.float8_e4m3fn})),
                              bias=ParamConstraint(dtypes=floats),
                              out_dtype=ParamConstraint(dtypes=floats)),
        "quantize_int4": fc(w=ParamConstraint(dtypes=floats, shape_rules=two_d)),
        "dequantize_int4": fc(codes=ParamConstraint(dtypes=u8, shape_rules=two_d + (DivisibleBy(1, 16),)),
                              scales=ParamConstraint(dtypes=floats, shape_rules=two_d),
                              zeros=ParamConstraint(dtypes=u8, shape_rules=two_d),
                              output_type=ParamConstraint(dtypes=floats)),
        "linear_int4": fc(x=ParamConstraint(dtypes=half, shape_rules=(MinDims(1),)),
                          codes=ParamConstraint(dtypes=u8, shape_rules=two_d + (DivisibleBy(1, 16),)),
                          scales=ParamConstraint(dtypes=floats, shape_rules=two_d),
                          zeros=ParamConstraint(dtypes=u8, shape_rules=two_d),
                          bias=ParamConstraint(dtypes=floats)),
        "paged_attention": fc(q=ParamConstraint(dtypes=half, shape_rules=(ExactDims(3),)),
                              k_cache=ParamConstraint(dtypes=half | e4m3, shape_rules=(ExactDims(4),)),
                              v_cache=ParamConstraint(dtypes=half | e4m3, shape_rules=(ExactDims(4),)),
                              page_table=ParamConstraint(dtypes=i32, shape_rules=two_d),
                              lengths=ParamConstraint(dtypes=i32, shape_rules=(ExactDims(1),)),
                              k_scale=ParamConstraint(dtypes=f32, devices=frozenset({"cuda", "cpu"})),
                              v_scale=ParamConstraint(dtypes=f32, devices=frozenset({"cuda", "cpu"}))),
        "paged_write": fc(key=ParamConstraint(dtypes=half, shape_rules=(ExactDims(3),)),
                          value=ParamConstraint(dtypes=half, shape_rules=(ExactDims(3),)),
                          k_cache=ParamConstraint(dtypes=half | e4m3, shape_rules=(ExactDims(4),)),
                          v_cache=ParamConstraint(dtypes=half | e4m3, shape_rules=(ExactDims(4),)),
                          slots=ParamConstraint(dtypes=ints, shape_rules=(ExactDims(1),)),
                          k_scale=ParamConstraint(dtypes=f32, devices=frozenset({"cuda", "cpu"})),
                          v_scale=ParamConstraint(dtypes=f32, devices=frozenset({"cuda", "cpu"}))),
        "paged_copy": fc(k_cache=ParamConstraint(dtypes=half | e4m3, shape_rules=(MinDims(4),)),
                         v_cache=ParamConstraint(dtypes=half | e4m3, shape_rules=(MinDims(4),)),
                         src=ParamConstraint(dtypes=ints, shape_rules=(ExactDims(1),)),
                         dst=ParamConstraint(dtypes=ints, shape_rules=(ExactDims(1),))),
        "window_attention": fc(q=ParamConstraint(dtypes=half, shape_rules=(ExactDims(4),)),
                               k=ParamConstraint(dtypes=half, shape_rules=(ExactDims(4),)),
                               v=ParamConstraint(dtypes=half, shape_rules=(ExactDims(4),)),
                               lengths=ParamConstraint(dtypes=i32, shape_rules=(ExactDims(1),))),
        "shared_attention": fc(q=ParamConstraint(dtypes=half, shape_rules=(ExactDims(3),)),
                               k_cache=ParamConstraint(dtypes=half | e4m3, shape_rules=(ExactDims(4),)),
                               v_cache=ParamConstraint(dtypes=half | e4m3, shape_rules=(ExactDims(4),)),
                               page_table=ParamConstraint(dtypes=i32, shape_rules=two_d),
                               lengths=ParamConstraint(dtypes=i32, shape_rules=(ExactDims(1),)),
                               groups=ParamConstraint(dtypes=i32, shape_rules=(ExactDims(1),)),
                               shared=ParamConstraint(dtypes=i32, shape_rules=(ExactDims(1),)),
                               k_scale=ParamConstraint(dtypes=f32, devices=frozenset({"cuda", "cpu"})),
                               v_scale=ParamConstraint(dtypes=f32, devices=frozenset({"cuda", "cpu"}))),
        "paged_write_rope": fc(q=ParamConstraint(dtypes=half, shape_rules=(ExactDims(3),)),
                               key=ParamConstraint(dtypes=half, shape_rules=(ExactDims(3),)),
                               value=ParamConstraint(dtypes=half, shape_rules=(ExactDims(3),)),
                               positions=ParamConstraint(dtypes=ints, shape_rules=(ExactDims(1),)),
                               rates=ParamConstraint(dtypes=f32, shape_rules=(ExactDims(1),)),
                               k_cache=ParamConstraint(dtypes=half | e4m3, shape_rules=(ExactDims(4),)),
                               v_cache=ParamConstraint(dtypes=half | e4m3, shape_rules=(ExactDims(4),)),
                               slots=ParamConstraint(dtypes=ints, shape_rules=(ExactDims(1),)),
                               k_scale=ParamConstraint(dtypes=f32, devices=frozenset({"cuda", "cpu"})),
                               v_scale=ParamConstraint(dtypes=f32, devices=frozenset({"cuda", "cpu"}))),
        "rms_norm": fc(x=ParamConstraint(dtypes=floats, shape_rules=(MinDims(1),)),
                       weight=ParamConstraint(dtypes=floats, shape_rules=(ExactDims(1),)),
                       residual=ParamConstraint(dtypes=floats)),
        "rms_norm_fp8": fc(x=ParamConstraint(dtypes=floats, shape_rules=(MinDims(1),)),
                           scale=ParamConstraint(dtypes=f32, devices=frozenset({"cuda", "cpu"})),
                           weight=ParamConstraint(dtypes=floats, shape_rules=(ExactDims(1),)),
                           residual=ParamConstraint(dtypes=floats), output_type=ParamConstraint(dtypes=fp8)),
        "rms_norm_mxfp8": fc(x=ParamConstraint(dtypes=floats, shape_rules=two_d),
                             weight=ParamConstraint(dtypes=floats, shape_rules=(ExactDims(1),)),
                             residual=ParamConstraint(dtypes=floats)),
        "sample_tokens": fc(logits=ParamConstraint(dtypes=floats, shape_rules=two_d),
                            u=ParamConstraint(dtypes=f32, shape_rules=(ExactDims(1),))),
        "apply_rope1": fc(x=ParamConstraint(dtypes=floats, shape_rules=(ExactDims(4),)),
                          freqs_cis=ParamConstraint(dtypes=floats, shape_rules=(ExactDims(6),))),
        "apply_rope": fc(xq=ParamConstraint(dtypes=floats, shape_rules=(ExactDims(4),)),
                         xk=ParamConstraint(dtypes=floats, shape_rules=(ExactDims(4),)),
                         freqs_cis=ParamConstraint(dtypes=floats, shape_rules=(ExactDims(6),))),
    }


def _register() -> None:
    from ...registry import registry

    try:
        load_library()
    except OSError as e:
        registry.mark_unavailable("hip", f"failed to load {LIB_PATH.name}: {e}")
        return
    if not torch.cuda.is_available() or torch.version.hip is None:
        registry.mark_unavailable("hip", "no ROCm GPU visible (torch.cuda.is_available() is False)")
        return
    arch = getattr(torch.cuda.get_device_properties(torch.cuda.current_device()), "gcnArchName", "")
    if not any(arch.startswith(a) for a in REQUIRED_ARCH):
        registry.mark_unavailable("hip", f"device arch {arch!r} is not one of {REQUIRED_ARCH}")
        return
    registry.register("hip", __import__(__name__, fromlist=__all__), _build_constraints())


_register()
