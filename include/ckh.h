/*
 * ckh.h -- C ABI of the MI355X (gfx950) kernels behind comfy_kitchen's "hip" backend.
 *
 * Conventions (all entry points):
 *   - Plain device pointers, int64 sizes, int dtype codes, and the HIP stream as an
 *     integer handle (hipStream_t cast to uintptr_t; 0 = the null stream).
 *   - Nothing allocates, nothing synchronises, no device scalar is read on the host:
 *     scales (`scale`, `global_scale`, `alpha`) stay in device memory and are read by
 *     the kernels.  Launches are asynchronous on `stream` and safe to capture in a
 *     hipGraph.
 *   - Return value: CKH_OK, or an error code with a message retrievable through
 *     ckh_last_error() (thread-local; valid until the next failing call on the thread).
 *   - Outputs are written in full, including the zero padding of swizzled scale
 *     tensors, so callers may allocate them uninitialised.
 *
 * Dtype codes are the reference's (backends/cuda/dlpack_bindings.cpp:27-41,
 * backends/eager/quantization.py:31-39): 0=f32 1=f16 2=bf16 3=u8 4=i8 5=e4m3fn 6=e5m2.
 *
 * Byte layouts: E4M3 / E5M2 codes are OCP FP8 bytes; NVFP4 codes are E2M1 nibbles,
 * two per byte, the even element in the high nibble when hi_first != 0; block scales
 * (E8M0 for MXFP8, E4M3 for NVFP4) use the 32_4_4 swizzle: logical scale (r, c) of a
 * [R, C] matrix padded to [ceil(R/128)*128, ceil(C/4)*4] lives at byte offset
 *   ((r/128 * ceil(C/4) + c/4) * 32 + r%32) * 16 + ((r%128)/32) * 4 + c%4.
 */
#ifndef CKH_H
#define CKH_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define CKH_ABI_VERSION 8

enum ckh_dtype {
    CKH_F32 = 0,
    CKH_F16 = 1,
    CKH_BF16 = 2,
    CKH_U8 = 3,
    CKH_I8 = 4,
    CKH_E4M3 = 5,
    CKH_E5M2 = 6,
};

enum ckh_status {
    CKH_OK = 0,
    CKH_ERR_INVALID = 1, /* bad argument: shape, dtype, alignment, null pointer */
    CKH_ERR_LAUNCH = 2,  /* the HIP runtime rejected the launch */
};

/* Version of this ABI (CKH_ABI_VERSION of the built library). */
int ckh_abi_version(void);

/* Message of the last failing call on this thread ("" if none). */
const char* ckh_last_error(void);

/*
 * Per-tensor FP8 quantize: out = fp8(clamp(x * r, +-max)), r = (1/scale) rounded to
 * x's dtype, the product rounded to x's dtype, then round-to-nearest-even to FP8.
 * x: numel elements of in_code (f32/f16/bf16); scale: one f32 on device;
 * out: numel bytes of out_code (e4m3 / e5m2).  A NaN product gives the byte eager's
 * vectorised CPU loop writes: 0xFF for bf16 x; 0x7F | sign for f16 / f32 x (the sign of
 * r's NaN, else of x's NaN, else negative for 0 * inf).
 * Replaces launch_quantize_fp8_kernel (reference backends/cuda/dlpack_bindings.cpp:45-48,
 * ops/per_tensor_quantize.cu:170-209), with the same argument order; arithmetic follows
 * backends/eager/quantization.py:41-55.
 */
int ckh_quantize_fp8(const void* x, void* out, const void* scale, int64_t numel,
                     int in_code, int out_code, uintptr_t stream);

/*
 * Per-tensor FP8 dequantize: out = x.to(out) * scale.to(out), rounded to out_code.
 * scale: one element of scale_code (f32 / f16 / bf16) on device, as eager accepts it.
 * Replaces launch_dequantize_fp8_kernel (dlpack_bindings.cpp:50-53,
 * ops/per_tensor_quantize.cu:211-249): the same arguments in the same order, plus
 * scale_code before the stream (that launcher reads an f32 scale only); arithmetic
 * follows eager quantization.py:57-61.
 */
int ckh_dequantize_fp8(const void* x, void* out, const void* scale, int64_t numel,
                       int in_code, int out_code, int scale_code, uintptr_t stream);

/*
 * MXFP8 quantize of x [orig_rows, orig_cols] (row-major, in_code f32/f16/bf16) into
 * codes [rows, cols] e4m3 (rows/cols >= orig, zero padded) and E8M0 block-32 scales in
 * the swizzled layout [roundup(rows,128), roundup(cols/32,4)].  cols % 32 == 0.
 * Replaces launch_quantize_mxfp8_kernel (dlpack_bindings.cpp:130-139,
 * ops/quantize_mxfp8.cu:148-208); arithmetic follows eager quantization.py:257-324.
 */
int ckh_quantize_mxfp8(const void* x, void* qx, void* scales, int64_t rows, int64_t cols,
                       int64_t orig_rows, int64_t orig_cols, int in_code, uintptr_t stream);

/*
 * MXFP8 dequantize: out[r,k] = (float(q[r,k]) * 2^(s[r,k/32]-127), s==0 -> 0).to(out).
 * qx [rows, cols] e4m3, scales swizzled, out [rows, cols] of out_code.
 * No native counterpart in the reference; arithmetic follows eager quantization.py:327-364.
 */
int ckh_dequantize_mxfp8(const void* qx, const void* scales, void* out, int64_t rows,
                         int64_t cols, int out_code, uintptr_t stream);

/*
 * NVFP4 quantize of x [orig_rows, orig_cols] with device f32 global scale g into packed
 * E2M1 codes [rows, cols/2] u8 and E4M3 block-16 scales, swizzled
 * [roundup(rows,128), roundup(cols/16,4)].  cols % 16 == 0 (rows need not be a
 * multiple of anything; the layouts pad them to 16 as the reference's pad_16x does).
 * epsilon is accepted and ignored, as in the reference.
 * Replaces launch_quantize_nvfp4_kernel (dlpack_bindings.cpp:104-116,
 * ops/quantize_nvfp4.cu:323-384); arithmetic follows eager quantization.py:115-160.
 */
int ckh_quantize_nvfp4(const void* x, const void* global_scale, void* qx, void* scales,
                       int64_t rows, int64_t cols, int64_t orig_rows, int64_t orig_cols,
                       float epsilon, int in_code, int hi_first, uintptr_t stream);

/*
 * NVFP4 dequantize: out = E2M1(q) * (g.to(out) * s8.to(out)) in out_code arithmetic.
 * qx [rows, cols/2] u8, scales swizzled, out [rows, cols].
 * Replaces launch_dequantize_nvfp4_kernel (dlpack_bindings.cpp:118-127,
 * ops/quantize_nvfp4.cu:386-434); arithmetic follows eager quantization.py:171-219.
 */
int ckh_dequantize_nvfp4(const void* qx, const void* global_scale, const void* scales,
                         void* out, int64_t rows, int64_t cols, int out_code, int hi_first,
                         uintptr_t stream);

/*
 * RoPE on x [batch, dim1, dim2, head_dim] (element strides sx_*; innermost stride 1)
 * with freqs [fb, fd1, fd2, head_dim/2, 2, 2] (element strides sf_* for the first
 * three dims; the inner [head_dim/2, 2, 2] must be contiguous).  A freqs dim of size 1
 * broadcasts; otherwise it must equal x's (dim 2 may be longer and is then truncated).
 * out_i = f[i,0]*x0 + f[i,1]*x1 per pair, computed in the freqs dtype, rounded to x's.
 * x: in_code f32 / f16 / bf16; freqs: freqs_code f32 / f16 / bf16.
 * xk / xk_out may be NULL (apply_rope1).  Outputs are contiguous [batch,dim1,dim2,hd].
 * Replaces launch_apply_rope_kernel (dlpack_bindings.cpp:76-102,
 * ops/apply_rope.cu:317-362); arithmetic follows eager rope.py:7-18.
 */
int ckh_apply_rope(const void* xq, const void* xk, const void* freqs, void* xq_out,
                   void* xk_out, int64_t batch, int64_t dim1, int64_t dim2,
                   int64_t head_dim, int64_t freqs_batch, int64_t freqs_dim1,
                   int64_t freqs_dim2, int64_t sx_batch, int64_t sx_dim1, int64_t sx_dim2,
                   int64_t sf_batch, int64_t sf_dim1, int64_t sf_dim2, int in_code,
                   int freqs_code, uintptr_t stream);

/*
 * Bytes of device workspace ckh_scaled_mm_mxfp8 / ckh_scaled_mm_fp8 may use at this shape to
 * split K (0: the shape does not split; a call that runs faster in one launch leaves the
 * workspace untouched).  A small grid of 256 x 256 output tiles with long
 * K (e.g. M = 256, N = 13824, K = 5120) splits K over up to 256 workgroups, which write fp32
 * partial tiles to the workspace: grids of at most 64 tiles as 256 x 128 half tiles
 * (128 KB partials) from 32 stages of 64 along K, grids of 65-128 tiles as whole tiles
 * (256 KB) from 64 stages when three ranges or more fit.  A second launch adds the
 * partials in a fixed order and applies scale, bias and output rounding.  No counterpart
 * in the reference (torch's scaled_mm takes no workspace).
 */
int64_t ckh_scaled_mm_workspace_bytes(int64_t M, int64_t N, int64_t K);

/*
 * MXFP8 GEMM: out[M,N] = sum_k A[m,k]*2^(sa-127) * B[n,k]*2^(sb-127) (+ bias[n]).
 * a [M,K] e4m3, b [N,K] e4m3 (both K-major), sa/sb E8M0 swizzled with logical shapes
 * [M, K/32] / [N, K/32]; bias NULL or [N] of bias_code (f32/f16/bf16);
 * out [M,N] row-major of out_code (f32/f16/bf16).  K % 32 == 0.
 * workspace: NULL, or ckh_scaled_mm_workspace_bytes(M, N, K) bytes of device memory
 * (16-byte aligned) that the call may overwrite; with less than that the call does not
 * split K (same result within fp32 summation order, slower where it would have split).  Calls
 * running at the same time need workspaces of their own.
 * No native counterpart in the reference (eager quantization.py:367-402 routes to
 * torch F.scaled_mm via scaled_mm_v2.py:27-53); replaces that call.
 */
int ckh_scaled_mm_mxfp8(const void* a, const void* b, const void* sa, const void* sb,
                        const void* bias, void* out, int64_t M, int64_t N, int64_t K,
                        int out_code, int bias_code, void* workspace, int64_t workspace_bytes,
                        uintptr_t stream);

/*
 * Per-tensor FP8 GEMM: out[M,N] = scale_a * scale_b * sum_k A[m,k] * B[n,k] (+ bias[n]).
 * a [M,K] e4m3, b [N,K] e4m3 (both K-major), scale_a / scale_b one f32 each on device;
 * bias NULL or [N] of bias_code; out [M,N] row-major of out_code.  K % 16 == 0.
 * workspace: as for ckh_scaled_mm_mxfp8.
 * Replaces the TensorWise torch F.scaled_mm call behind TensorCoreFP8Layout's
 * linear / mm / addmm (tensor/fp8.py:86-101 -> scaled_mm_v2.py:27-53).
 */
int ckh_scaled_mm_fp8(const void* a, const void* b, const float* scale_a, const float* scale_b,
                      const void* bias, void* out, int64_t M, int64_t N, int64_t K,
                      int out_code, int bias_code, void* workspace, int64_t workspace_bytes,
                      uintptr_t stream);

/*
 * NVFP4 GEMM: out[M,N] = alpha * sum_k E2M1(a)*sa[m,k/16] * E2M1(b)*sb[n,k/16] (+bias[n]).
 * a [M,K/2] u8, b [N,K/2] u8 (hi_first packing), sa/sb E4M3 swizzled with logical
 * shapes [M, K/16] / [N, K/16]; alpha one f32 on device; bias NULL or [N].
 * K % 32 == 0.
 * Replaces launch_cublas_gemm_blockwise_fp4_kernel (dlpack_bindings.cpp:59-74,
 * ops/cublas_gemm_nvfp4.cu:297-342); semantics follow eager quantization.py:222-246.
 * workspace: NULL, or ckh_scaled_mm_nvfp4_workspace_bytes(M, N, K) bytes of device memory
 * (16-byte aligned) in which small tile grids split K (as ckh_scaled_mm_mxfp8); with less
 * the call does not split.  Calls running at the same time need workspaces of their own.
 * Argument differences from that launcher: the activation comes first (the launcher takes
 * B before A because cuBLASLt is column-major; the product is the same A B^T); the
 * workspace is sized by ckh_scaled_mm_nvfp4_workspace_bytes rather than by the caller's
 * choice, and there is no `accumulate` flag (its only caller,
 * backends/cuda/__init__.py:353, always passes false, i.e. out is overwritten); bias_code
 * names the bias dtype, which that launcher takes from the DLPack tensor.
 */
int ckh_scaled_mm_nvfp4(const void* a, const void* b, const void* sa, const void* sb,
                        const void* alpha, const void* bias, void* out, int64_t M,
                        int64_t N, int64_t K, int out_code, int bias_code, void* workspace,
                        int64_t workspace_bytes, uintptr_t stream);

/*
 * ckh_scaled_mm_nvfp4 with the operands' tensor scales (one f32 each on device) in place of
 * their product alpha: the kernel multiplies them, so a caller needs no launch to do so.
 */
int ckh_scaled_mm_nvfp4_scales(const void* a, const void* b, const void* sa, const void* sb,
                               const void* scale_a, const void* scale_b, const void* bias,
                               void* out, int64_t M, int64_t N, int64_t K, int out_code,
                               int bias_code, void* workspace, int64_t workspace_bytes,
                               uintptr_t stream);

/*
 * Bytes of device workspace ckh_scaled_mm_nvfp4 may use at this shape to split K (0: no
 * split; as for ckh_scaled_mm_workspace_bytes): grids of at most 64 output tiles of 256 x 256 with K of at least 2048 (split as
 * 256 x 128 half tiles), and grids of 65-128 tiles with K of at least 4096 when three K
 * ranges or more fit.  No
 * counterpart in the reference (its launcher takes a cuBLASLt workspace of the caller's
 * size).
 */
int64_t ckh_scaled_mm_nvfp4_workspace_bytes(int64_t M, int64_t N, int64_t K);

/*
 * Dynamic per-tensor scale: *scale_out = float(round_x(amax(|x|) * RN32(1/divisor))),
 * the amax and the product rounded to x's dtype (in_code), as the layouts' default scale
 * torch.amax(tensor.abs()) / max computes it on a GPU tensor (torch multiplies by the
 * fp32 reciprocal of a scalar divisor there).  x: numel contiguous elements; scale_out:
 * one f32 on device; workspace: CKH_AMAX_WORKSPACE_BYTES of device memory (4-byte
 * aligned, contents ignored and overwritten) that holds the per-workgroup partial maxima,
 * so the call allocates nothing.  Calls running at the same time need workspaces of their
 * own.  A NaN in x gives a NaN scale.  Replaces that torch expression in
 * TensorCoreFP8Layout.quantize (tensor/fp8.py:56-61, divisor 448) and
 * TensorCoreNVFP4Layout.quantize (tensor/nvfp4.py:64-69, divisor 2688); the result feeds
 * ckh_quantize_fp8 / ckh_quantize_nvfp4 on the same stream without a host round trip.
 */
#define CKH_AMAX_WORKSPACE_BYTES 8192
int ckh_amax_scale(const void* x, int64_t numel, int in_code, float divisor, void* scale_out,
                   void* workspace, uintptr_t stream);

/*
 * ckh_amax_scale without the workspace argument: the same kernels and result, with the
 * per-workgroup partial maxima in an 8 KB (CKH_AMAX_WORKSPACE_BYTES) device array that
 * the library holds on each GPU until the process ends.  The call allocates nothing
 * (no hipMalloc, no torch allocator): for callers that cannot allocate, such as code
 * under hipGraph capture with no allocator of its own or serving loops that forbid
 * allocation.  Every input size fits (the grid never has more workgroups than the array
 * has words).  `stream` must belong to the current device.  The first call on a device
 * resolves the array's address there (hipGetSymbolAddress) and must run outside stream
 * capture; later calls may be captured into a hipGraph.  All calls on one GPU share
 * its array: calls that overlap on that GPU (other streams, other threads) race and must
 * be serialised by the caller.  No counterpart in the reference.
 */
int ckh_amax_scale_noalloc(const void* x, int64_t numel, int in_code, float divisor,
                           void* scale_out, uintptr_t stream);

/*
 * Per-tensor FP8 quantize with the layouts' dynamic scale: ckh_amax_scale (divisor = the
 * largest value of out_code) followed by ckh_quantize_fp8 with that scale, in two launches
 * instead of three, or one for an aligned 16-bit x of at most 64 KB.  Codes and *scale_out
 * equal those of the two separate calls bit for bit.  x non-empty; workspace as for
 * ckh_amax_scale; f32 or unaligned x runs the separate launches.  Calls running at the same
 * time need workspaces of their own.  Replaces the scale=None branch of
 * TensorCoreFP8Layout.quantize (tensor/fp8.py:56-61).
 */
int ckh_quantize_fp8_dynamic(const void* x, float divisor, void* scale_out, void* out, int64_t numel,
                             int in_code, int out_code, void* workspace, uintptr_t stream);

/*
 * NVFP4 quantize with the layouts' dynamic global scale: ckh_amax_scale (divisor 2688 for
 * TensorCoreNVFP4Layout) followed by ckh_quantize_nvfp4 with that scale, in two launches
 * instead of three (one for x of at most 64 KB on the 16-bit fast path).  Launch 1 writes the per-workgroup partial maxima of |x| to
 * `workspace` (CKH_AMAX_WORKSPACE_BYTES, 4-byte aligned; its loads are cached, so the
 * quantize that follows finds x in the 256 MB infinity cache when it fits there); launch 2
 * quantizes, every workgroup forming the scale from those words itself, and stores the
 * scale to *scale_out (one f32 on device).  Codes, block scales and *scale_out equal those
 * of the two separate calls bit for bit.  Shapes and arguments as ckh_quantize_nvfp4,
 * plus x non-empty; shapes outside the 16-bit fast path (column padding, f32 input,
 * cols % 64, alignment) run the separate scale launch and the general quantize.  Calls running at
 * the same time need workspaces of their own.  Replaces the scale=None branch of
 * TensorCoreNVFP4Layout.quantize (tensor/nvfp4.py:64-69: torch.amax(x.abs()) / 2688, then
 * ck.quantize_nvfp4), the dynamic input quantization of samples/nvfp4_linear.py:55-59.
 */
int ckh_quantize_nvfp4_dynamic(const void* x, float divisor, void* scale_out, void* qx, void* scales,
                               int64_t rows, int64_t cols, int64_t orig_rows, int64_t orig_cols,
                               float epsilon, int in_code, int hi_first, void* workspace,
                               uintptr_t stream);

/*
 * Weight-only 4-bit linears.  A weight W [n, k] is codes [n, k/2] u8 (two codes 0..15 a byte,
 * the even k in the low nibble), scales [n, ceil(k/group)] of scale_code (f32/f16/bf16) and
 * optional zero points [n, ceil(k/group)] u8 (NULL: 8 everywhere):
 *   W[n, k] = (code - zero) * scale.
 * k % 32 == 0, group % 32 == 0; the last group of a row may be shorter than `group`.
 *
 * quantize: scale = amax(|x|) / 7 over the group, rounded to in_code, code =
 * clamp(rint(x / scale), -8, 7) + 8 (8 where the scale is 0).  A NaN in a group makes its
 * scale NaN.
 * dequantize: one rounding to out_code.
 * linear: y [m, n] = x W^T + bias, x [m, k] of x_code (f16/bf16) with x_stride elements between
 * rows (x 16-byte aligned, x_stride % 8 == 0), y of x_code, bias [n] of bias_code or NULL; sums
 * in fp32, one rounding.  An activation that is not finite makes its row of y NaN.  The workspace of
 * ckh_linear_int4_workspace_bytes lets K be split (0: it is not); with NULL or a short one the call
 * runs without (same result up to the order of fp32 sums).
 */
int64_t ckh_linear_int4_workspace_bytes(int64_t m, int64_t n, int64_t k, int64_t group);
int ckh_quantize_int4(const void* x, void* codes, void* scales, int64_t n, int64_t k, int64_t group, int in_code,
                      uintptr_t stream);
int ckh_dequantize_int4(const void* codes, const void* scales, const void* zeros, void* out, int64_t n, int64_t k,
                        int64_t group, int scale_code, int out_code, uintptr_t stream);
int ckh_linear_int4(const void* x, const void* codes, const void* scales, const void* zeros, const void* bias,
                    void* y, int64_t m, int64_t n, int64_t k, int64_t x_stride, int64_t group, int x_code,
                    int scale_code, int bias_code, void* workspace, int64_t workspace_bytes, uintptr_t stream);

/*
 * A key-value cache held in pages: K and V are [pages, page_size, kv_heads, dim] of cache_code with
 * any strides (elements; 16-byte multiples, the last dimension contiguous), 16-byte aligned.  Token
 * t of a sequence is row t % page_size of page table[t / page_size]; a slot is page * page_size + row
 * (int32, or int64 where wide_slots != 0), and slots outside the cache are skipped.
 *
 * ckh_paged_attention: one query token per sequence.  out[b, h] = softmax(scale q[b, h] K^T) V over
 * sequence b's visible tokens: its lengths[b] tokens (int32, taken into 0 .. max_pages * page_size),
 * or with window > 0 its last `window` and its first `sinks`.  q [batch, heads, dim] and out
 * (contiguous) of q_code (f16/bf16); cache_code the same or e4m3, and what the cache holds is
 * multiplied by *k_scale, *v_scale (device f32, NULL: 1).  heads % kv_heads == 0; dim 64, 96, 128 or
 * 256.  Query head h reads key-value head h / (heads / kv_heads).  A sequence without visible tokens
 * gives zeros.
 * page_table: int32 [batch, max_pages], table_stride elements a row, of under 2^31 tokens each (and 64
 * rows of under 2^36); entries that no visible token needs are not read, others outside 0 .. pages-1
 * are read as the last page.
 * strides: q batch, head; k page, token, head; v page, token, head.
 * The workspace of ckh_paged_attention_workspace_bytes lets long sequences be split (0: never
 * split); with NULL or a short one every sequence is read by one workgroup per key-value head.
 *
 * ckh_paged_write: key, value [tokens, kv_heads, dim] of x_code (f16/bf16) to slots[tokens] of K and
 * V, as they are (cache_code == x_code; no scales) or as e4m3 codes of clamp(x / *scale, +-448).
 * dim % 16 == 0.
 * strides: key token, head; value token, head; k page, token, head; v page, token, head.
 *
 * ckh_paged_copy: rows src[i] to dst[i], i < rows, of K and V in each of `layers` caches; no slot of
 * dst may be in src.  strides: k layer, page, token, head; v layer, page, token, head.
 */
int64_t ckh_paged_attention_workspace_bytes(int64_t batch, int64_t heads, int64_t kv_heads, int64_t dim,
                                            int64_t page_size, int64_t max_pages);
int ckh_paged_attention(const void* q, const void* k_cache, const void* v_cache, const void* page_table,
                        const void* lengths, const void* k_scale, const void* v_scale, void* out, int64_t batch,
                        int64_t heads, int64_t kv_heads, int64_t dim, int64_t pages, int64_t page_size,
                        int64_t max_pages, int64_t table_stride, const int64_t* strides, int64_t window,
                        int64_t sinks, float scale, int q_code, int cache_code, void* workspace,
                        int64_t workspace_bytes, uintptr_t stream);
int ckh_paged_write(const void* key, const void* value, void* k_cache, void* v_cache, const void* slots,
                    const void* k_scale, const void* v_scale, int64_t tokens, int64_t kv_heads, int64_t dim,
                    int64_t pages, int64_t page_size, const int64_t* strides, int x_code, int cache_code,
                    int wide_slots, uintptr_t stream);
int ckh_paged_copy(void* k_cache, void* v_cache, const void* src, const void* dst, int64_t layers, int64_t rows,
                   int64_t kv_heads, int64_t dim, int64_t pages, int64_t page_size, const int64_t* strides,
                   int element_bytes, int wide_slots, uintptr_t stream);

/*
 * Causal attention of prompts with a sliding window and sinks.  q [batch, queries, heads, dim],
 * k, v [batch, keys, kv_heads, dim] of one code (f16/bf16) with any strides (elements; 16-byte
 * multiples, the last dimension contiguous); out contiguous, of q's shape.  Query i stands at
 * position p = i + keys - queries and sees key j if j <= p, j < lengths[batch] (int32; NULL: all
 * keys), and p - j < window or j < sinks; window 0: no window.  A query that sees nothing gives
 * zeros.  What a pair that is not visible holds has no influence, infinities and NaN included.
 * heads % kv_heads == 0; dim 64, 96, 128 or 256.  strides: q, k, v: batch, token, head each.
 * The workspace of ckh_window_attention_workspace_bytes lets few rows' keys be split over the GPU (0:
 * they are not); NULL or a short one is no error.
 */
int64_t ckh_window_attention_workspace_bytes(int64_t batch, int64_t queries, int64_t keys, int64_t heads,
                                             int64_t kv_heads, int64_t dim, int64_t window, int64_t sinks);
int ckh_window_attention(const void* q, const void* k, const void* v, const void* lengths, void* out, int64_t batch,
                         int64_t queries, int64_t keys, int64_t heads, int64_t kv_heads, int64_t dim,
                         const int64_t* strides, int64_t window, int64_t sinks, float scale, int code,
                         void* workspace, int64_t workspace_bytes, uintptr_t stream);

/*
 * Root-mean-square norm with the residual's addition.  With T the rounding to x's type:
 *   h = T(x + residual) (x without one),  y = T(h rsqrt(mean(h^2) + eps) weight)
 * for x [rows, cols] of x_code (f32/f16/bf16), x_stride elements between rows; residual the same with
 * residual_stride, or NULL; weight [cols] of weight_code (f32/f16/bf16) or NULL (ones); h contiguous, written
 * where there is a residual.  cols up to 65536; squares are summed in fp32.
 * The result: y itself (out_code == x_code), contiguous; or the codes that ckh_quantize_fp8 gives for y and
 * *scale (out_code e4m3 / e5m2); or with mx != 0 the codes [out_rows, out_cols] and swizzled scales that
 * ckh_quantize_mxfp8 gives for y (out_code e4m3; out_cols % 32 == 0, out_rows at most rows rounded up to 128;
 * padding is zeros).  out_rows and out_cols are rows and cols where mx is 0.
 */
int ckh_rms_norm(const void* x, const void* residual, const void* weight, const void* scale, void* y, void* scales,
                 void* h, int64_t rows, int64_t cols, int64_t out_rows, int64_t out_cols, int64_t x_stride,
                 int64_t residual_stride, float eps, int x_code, int weight_code, int out_code, int mx,
                 uintptr_t stream);

/*
 * ckh_paged_write of keys that are turned to their positions first, and queries with them.  Pair i of the
 * first `rotary` elements of a head turns by position * rates[i] (rates: f32 [rotary / 2]; the product in 64
 * bits), (x, y) -> magnitude (x cos - y sin, x sin + y cos): neighbours (2i, 2i + 1) where interleaved != 0,
 * else (i, i + rotary / 2).  q [tokens, heads, dim] -> q_out, key -> its slots, rounded once, and key_out
 * (NULL: not kept), value -> its slots; q_out and key_out contiguous, of x_code.  positions [tokens]: int32, or
 * int64 where wide_positions != 0.  The rest as for ckh_paged_write; rotary is even, 0 .. dim.
 * strides: q token, head; key token, head; value token, head; k page, token, head; v page, token, head.
 */
int ckh_paged_write_rope(const void* q, const void* key, const void* value, const void* positions, const void* rates,
                         void* q_out, void* key_out, void* k_cache, void* v_cache, const void* slots,
                         const void* k_scale, const void* v_scale, int64_t tokens, int64_t heads, int64_t kv_heads,
                         int64_t dim, int64_t rotary, int64_t pages, int64_t page_size, const int64_t* strides,
                         int interleaved, float magnitude, int x_code, int cache_code, int wide_positions,
                         int wide_slots, uintptr_t stream);

/*
 * The next token of each row of logits [rows, vocab] (code f32/f16/bf16, row_stride elements between rows),
 * drawn with u [rows] (f32, 0 <= u < 1).  Tokens stand in the order of their logits, the largest first, equal
 * ones by number; w = exp((logit - max) / temperature).  Kept are the first tokens of that order that are among
 * the first top_k (0: all), and needed to reach top_p of the weight of those (1 and over: all), and have
 * w >= min_p; the first always is.  out [rows] (int64) is the first token whose running weight exceeds u times
 * the weight of all kept.  Temperature 0: the first of the largest logits.  -inf and NaN are never drawn, nor
 * what lies 32 temperatures or more (some of it from 31.94 on) under the largest; a row of nothing else gives -1.
 * Weights are held to some 2^-33 of themselves, and a running weight within 2^-36 of a border has reached it.
 * temperature, top_p, min_p (f32) and top_k (int32): device arrays of one a row, or NULL, then the *_all
 * values hold.  In an array, a temperature that is not over 0 counts as 0, a top_k under 1 as all, a min_p over
 * 1 as 1.  vocab up to 2^24.  The workspace is needed.
 */
int64_t ckh_sample_workspace_bytes(int64_t rows, int64_t vocab);
int ckh_sample(const void* logits, const void* u, const void* temperature, const void* top_k, const void* top_p,
               const void* min_p, double temperature_all, int64_t top_k_all, double top_p_all, double min_p_all,
               void* out, int64_t rows, int64_t vocab, int64_t row_stride, int code, void* workspace,
               int64_t workspace_bytes, uintptr_t stream);

/*
 * ckh_paged_attention (without a window) for sequences that begin with the same tokens, which are read once.
 * Sequences group_starts[g] .. group_starts[g + 1] - 1 form group g (int32 [groups + 1], ascending; a sequence
 * outside all groups shares nothing), and the first shared[g] of their tokens (int32 [groups]; at most the shortest's length
 * counts) have the same rows, found by the table of the group's first sequence: what is read for each of
 * the others are its tokens behind them.  Everything else as for ckh_paged_attention.  The workspace is needed.
 */
int64_t ckh_shared_attention_workspace_bytes(int64_t batch, int64_t heads, int64_t kv_heads, int64_t dim, int64_t groups,
                                             int64_t page_size, int64_t max_pages);
int ckh_shared_attention(const void* q, const void* k_cache, const void* v_cache, const void* page_table,
                         const void* lengths, const void* group_starts, const void* shared, const void* k_scale,
                         const void* v_scale, void* out, int64_t batch, int64_t heads, int64_t kv_heads, int64_t dim,
                         int64_t groups, int64_t pages, int64_t page_size, int64_t max_pages, int64_t table_stride,
                         const int64_t* strides, float scale, int q_code, int cache_code, void* workspace,
                         int64_t workspace_bytes, uintptr_t stream);

#ifdef __cplusplus
}
#endif

#endif /* CKH_H */
