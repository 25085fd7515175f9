// Root-mean-square norm with the residual's addition, its result in the input's type or in 8 bits, for
// gfx950.  With T the rounding to x's type:
//   h = T(x + residual) (or x),  y = T(h rsqrt(mean(h^2) + eps) weight),
// and then y itself, the codes quantize_per_tensor_fp8 gives for it, or the codes and swizzled scales of
// quantize_mxfp8: bit for bit those of the two calls, without y's way through memory.
//
// Bound by the bytes of x, residual, h and the result (16384 rows of 5120 with a residual, bf16: 112 us, 6.0 TB/s; to MXFP8 108;
// 16384 rows of 5119, on no boundary of 16 bytes, 88 us without a residual for 65).  A workgroup holds a row in its registers (of
// short rows several), so every input is read once: a thread has 8 consecutive elements of every so many.  The squares are summed
// in fp32 in one order whatever the launch: those of 8 elements, of 64 such pieces over a wave's lanes, then of
// these in LDS; so y does not depend on how many rows there are, on alignment, or on what becomes of it.
// Results (MXFP8 codes aside) go past the caches.  With what reads them behind the call (replayed, rows of 5120 with a residual, bf16; ordinary stores second): a
// linear_int4 of one row 10.4 and 10.5 us, of 48 28.1 and 28.1; the sum of both results of 777 rows 18.9 and 18.1, of 16384
// 202 and 218.
// A block of 32 that shares a scale lies in four neighbouring lanes, the four blocks of a scale word in sixteen.
#include <algorithm>

#include "ckh_common.h"
#include "dispatch.h"
#include "quant_math.h"

namespace ckh {
namespace norm {

enum Out { kSame, kE4M3, kE5M2, kMX };

struct Args {
    const uint8_t *x, *residual, *weight;  // residual, weight: may be null
    const float* scale;
    uint8_t *y, *h;
    uint32_t* scales;
    int64_t x_row, r_row, y_row;  // bytes
    int rows, cols, out_rows, out_cols, scale_words;  // scale_words: of a row
    int weight_code;
    float eps, inv_cols;
};

// 16 bytes on the boundaries of elements.
template <int ES>
struct __attribute__((packed, aligned(ES))) Loose {
    uint32_t w[4];
};

template <int C>
__device__ __forceinline__ void unpack_loose(const uint8_t* p, float (&v)[8]) {
    if constexpr (C == CKH_F32) {
        const auto a = *reinterpret_cast<const Loose<4>*>(p), b = *reinterpret_cast<const Loose<4>*>(p + 16);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = as_f(e < 4 ? a.w[e & 3] : b.w[e & 3]);
    } else {
        const auto a = *reinterpret_cast<const Loose<2>*>(p);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t h = (a.w[e >> 1] >> (16 * (e & 1))) & 0xffffu;
            v[e] = C == CKH_BF16 ? bf16_to_f(h) : f16_to_f(h);
        }
    }
}

// 8 elements at p, of which those from `left` on are zeros.
template <int C, bool VEC>
__device__ __forceinline__ void read8(const uint8_t* p, int left, float (&v)[8]) {
    if constexpr (VEC) {
        load8<C>(p, v);
    } else if (left >= 8) {
        unpack_loose<C>(p, v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float f = load1<C>(p, min(e, left - 1));
            v[e] = e < left ? f : 0.0f;
        }
    }
}

template <bool VEC>
__device__ __forceinline__ void read_weight(const Args& a, int at, int left, float (&w)[8]) {
    if (!a.weight) {
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = 1.0f;
        return;
    }
    if (a.weight_code == CKH_F32) read8<CKH_F32, VEC>(a.weight + static_cast<int64_t>(at) * 4, left, w);
    else if (a.weight_code == CKH_BF16) read8<CKH_BF16, VEC>(a.weight + static_cast<int64_t>(at) * 2, left, w);
    else read8<CKH_F16, VEC>(a.weight + static_cast<int64_t>(at) * 2, left, w);
}

template <int C>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
    if constexpr (C == CKH_BF16) return f_to_bf16_rne(a) | f_to_bf16_rne(b) << 16;
    else return f_to_f16(a) | f_to_f16(b) << 16;
}

// 8 values, already rounded to C, to p.
template <int C, bool VEC>
__device__ __forceinline__ void write8(uint8_t* p, int left, const float (&v)[8]) {
    if constexpr (VEC && C == CKH_F32) {
        st_stream16(p, make_uint4(as_u(v[0]), as_u(v[1]), as_u(v[2]), as_u(v[3])));
        st_stream16(p + 16, make_uint4(as_u(v[4]), as_u(v[5]), as_u(v[6]), as_u(v[7])));
    } else if constexpr (VEC) {
        st_stream16(p, make_uint4(pack16<C>(v[0], v[1]), pack16<C>(v[2], v[3]), pack16<C>(v[4], v[5]), pack16<C>(v[6], v[7])));
    } else if (left >= 8) {
        if constexpr (C == CKH_F32) {
            *reinterpret_cast<Loose<4>*>(p) = {as_u(v[0]), as_u(v[1]), as_u(v[2]), as_u(v[3])};
            *reinterpret_cast<Loose<4>*>(p + 16) = {as_u(v[4]), as_u(v[5]), as_u(v[6]), as_u(v[7])};
        } else {
            *reinterpret_cast<Loose<2>*>(p) = {pack16<C>(v[0], v[1]), pack16<C>(v[2], v[3]), pack16<C>(v[4], v[5]), pack16<C>(v[6], v[7])};
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (e >= left) continue;
            if constexpr (C == CKH_F32) reinterpret_cast<float*>(p)[e] = v[e];
            else reinterpret_cast<uint16_t*>(p)[e] = static_cast<uint16_t>(pack16<C>(v[e], 0.0f));
        }
    }
}

// What becomes of 8 elements v, from `at` on, of a row whose factor is f: y, or its codes.  `live`: the row and the elements are
// there.  MXFP8: sixteen lanes have the four blocks of a scale word, `lane` is this one's place among them.
template <int C, int OUT, bool VEC>
__device__ __forceinline__ void emit(const Args& a, int64_t row, int at, bool live, float (&v)[8], float f, float sc, int lane) {
    constexpr int ES = ElemSize<C>::value;
    if (OUT != kMX && !live) return;
    if (live) {
        float w[8];
        read_weight<VEC>(a, at, a.cols - at, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = round_to_hw<C>(v[e] * f * w[e]);
        if constexpr (OUT == kMX && !VEC) {  // padding is zeros, whatever f is
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = e < a.cols - at ? v[e] : 0.0f;
        }
    }
    if constexpr (OUT == kSame) {
        write8<C, VEC>(a.y + row * a.y_row + static_cast<int64_t>(at) * ES, a.cols - at, v);
    } else if constexpr (OUT != kMX) {
        constexpr int F = OUT == kE4M3 ? CKH_E4M3 : CKH_E5M2;
        const float inv = round_to<C>(1.0f / sc);
        uint8_t* y = a.y + row * a.y_row + at;
        uint32_t code[2] = {0u, 0u};
        float t[8];
        bool odd = false;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            t[e] = round_to_hw<C>(v[e] * inv);
            odd |= is_nan(t[e]);
            constexpr float kMax = F == CKH_E4M3 ? 448.0f : 57344.0f;
            t[e] = __builtin_amdgcn_fmed3f(t[e], -kMax, kMax);
        }
#pragma unroll
        for (int q = 0; q < 2; ++q)
            code[q] = F == CKH_E4M3 ? hw_e4m3x4(t[4 * q], t[4 * q + 1], t[4 * q + 2], t[4 * q + 3])
                                    : hw_e5m2x4(t[4 * q], t[4 * q + 1], t[4 * q + 2], t[4 * q + 3]);
        if (odd) {
            code[0] = code[1] = 0u;
#pragma unroll
            for (int e = 0; e < 8; ++e) code[e >> 2] |= quantize_one<C, F>(v[e], inv, sc) << (8 * (e & 3));
        }
        if constexpr (VEC) {
            st_stream8(y, make_uint2(code[0], code[1]));
        } else if (a.cols - at >= 8) {
            struct __attribute__((packed, aligned(1))) Codes {
                uint32_t w[2];
            };
            *reinterpret_cast<Codes*>(y) = {code[0], code[1]};
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < a.cols - at) y[e] = static_cast<uint8_t>(code[e >> 2] >> (8 * (e & 3)));
        }
    } else {
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, as_u(v[e]) & 0x7fffffffu);
        top = max(top, dpp<0xb1>(top));  // the neighbouring lane's, then the other pair's
        top = max(top, dpp<0x4e>(top));
        const bool there = row < a.rows && at < a.out_cols;
        const uint32_t e8 = there ? mx_exponent(top) : 0u;
        if (row < a.out_rows && at < a.out_cols)
            *reinterpret_cast<uint2*>(a.y + row * a.out_cols + at) = there ? mx_encode8(v, top, e8) : make_uint2(0u, 0u);
        uint32_t word = e8 << (8 * (lane >> 2));
        word |= __shfl_xor(word, 4, 64);
        word |= __shfl_xor(word, 8, 64);
        if (lane == 0) a.scales[swz_offset(row, at >> 5, a.scale_words) >> 2] = word;
    }
}

// Short rows of whole pieces: P lanes a row, 256 / P rows at once, `passes` times.  (MXFP8: 128 rows a workgroup, those
// that share lines of scales.)
template <int C, int OUT, int P>
__global__ __launch_bounds__(256) void short_kernel(Args a, int passes) {
    constexpr int ES = ElemSize<C>::value;
    const int at = static_cast<int>(threadIdx.x % P) * 8;
    for (int pass = 0; pass < passes; ++pass) {
        const int64_t row = (static_cast<int64_t>(blockIdx.x) * passes + pass) * (256 / P) + threadIdx.x / P;
        const bool live = at < a.cols && row < a.rows;
        float v[8] = {};
        if (live) load8<C>(a.x + row * a.x_row + at * ES, v);
        if (a.residual && live) {
            float u[8];
            load8<C>(a.residual + row * a.r_row + at * ES, u);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = round_to_hw<C>(v[e] + u[e]);
            write8<C, true>(a.h + (row * a.cols + at) * ES, 8, v);
        }
        float squares = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) squares = __fmaf_rn(v[e], v[e], squares);
#pragma unroll
        for (int s = P / 2; s >= 1; s >>= 1) squares += __shfl_xor(squares, s, 64);  // (a longer row's tree, without its zeros)
        const float f = rsqrtf(__fmaf_rn(squares, a.inv_cols, a.eps));
        if (OUT != kMX || at < a.scale_words * 128) emit<C, OUT, true>(a, row, at, live, v, f, OUT == kE4M3 || OUT == kE5M2 ? a.scale[0] : 1.0f, threadIdx.x & 15);
    }
}

// N: pieces of 8 elements a thread.  VEC: rows are whole pieces on 16-byte boundaries.
template <int C, int OUT, int N, bool VEC>
__global__ void norm_kernel(Args a) {
    constexpr int ES = ElemSize<C>::value;
    __shared__ float part[128];  // of 64 pieces each
    const int threads = blockDim.x;
    int row = blockIdx.x;
    if constexpr (OUT == kMX) {
        // the rows of a 128-row tile, whose scales share lines, go to one XCD (workgroups go round the
        // eight in turn)
        const int n = row >> 3;
        row = ((n >> 7) * 8 + (row & 7)) * 128 + (n & 127);
        if (row >= (a.rows + 127 & ~127)) return;
        if (row >= a.rows) {  // padding: zero codes up to out_rows, zero scales up to 128 rows
            for (int i = threadIdx.x; i < a.scale_words; i += threads) a.scales[swz_offset(row, 4 * i, a.scale_words) >> 2] = 0u;
            if (row < a.out_rows)
                for (int i = threadIdx.x; i < a.out_cols / 8; i += threads)
                    *reinterpret_cast<uint2*>(a.y + static_cast<int64_t>(row) * a.out_cols + i * 8) = make_uint2(0u, 0u);
            return;
        }
    }
    const uint8_t* x = a.x + row * a.x_row;
    const uint8_t* r = a.residual ? a.residual + row * a.r_row : nullptr;
    float v[N][8];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int at = (threadIdx.x + i * threads) * 8;
        if (at < a.cols) read8<C, VEC>(x + static_cast<int64_t>(at) * ES, a.cols - at, v[i]);
        else
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] = 0.0f;
    }
    if (r) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int at = (threadIdx.x + i * threads) * 8;
            if (at < a.cols) {
                float u[8];
                read8<C, VEC>(r + static_cast<int64_t>(at) * ES, a.cols - at, u);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[i][e] = round_to_hw<C>(v[i][e] + u[e]);
            }
        }
    }
    float squares[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        squares[i] = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) squares[i] = __fmaf_rn(v[i][e], v[i][e], squares[i]);
    }
#pragma unroll
    for (int s = 32; s >= 1; s >>= 1)
#pragma unroll
        for (int i = 0; i < N; ++i) squares[i] += __shfl_xor(squares[i], s, 64);
    if ((threadIdx.x & 63) == 0)
#pragma unroll
        for (int i = 0; i < N; ++i) part[(threadIdx.x + i * threads) >> 6] = squares[i];
    if (r) {
        uint8_t* h = a.h + static_cast<int64_t>(row) * a.cols * ES;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int at = (threadIdx.x + i * threads) * 8;
            if (at < a.cols) write8<C, VEC>(h + static_cast<int64_t>(at) * ES, a.cols - at, v[i]);
        }
    }
    __syncthreads();
    float sum = part[0];
    for (int w = 1; w < (a.cols + 511) >> 9; ++w) sum += part[w];
    const float f = rsqrtf(__fmaf_rn(sum, a.inv_cols, a.eps));

    const float sc = OUT == kE4M3 || OUT == kE5M2 ? a.scale[0] : 1.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int piece = threadIdx.x + i * threads, at = piece * 8;
        const bool live = at < a.cols;
        if (OUT == kMX && piece >= a.scale_words * 16) continue;  // whole groups of sixteen lanes
        emit<C, OUT, VEC>(a, row, at, live, v[i], f, sc, threadIdx.x & 15);
    }
}

template <int C, int OUT, bool VEC>
void launch_rows(const Args& a, hipStream_t st) {
    const int pieces = OUT == kMX ? a.scale_words * 16 : static_cast<int>(cdiv(a.cols, 8));
    const auto [n, threads] = norm_launch(pieces, a.rows, OUT != kSame, device_cus());
    const unsigned grid = OUT == kMX ? static_cast<unsigned>(rup(cdiv(a.rows, 128), 8) * 128) : static_cast<unsigned>(a.rows);
    if (n == 1) norm_kernel<C, OUT, 1, VEC><<<grid, threads, 0, st>>>(a);
    else if (n == 2) norm_kernel<C, OUT, 2, VEC><<<grid, threads, 0, st>>>(a);
    else if (n == 4) norm_kernel<C, OUT, 4, VEC><<<grid, threads, 0, st>>>(a);
    else norm_kernel<C, OUT, 8, VEC><<<grid, threads, 0, st>>>(a);
}

template <int C, int OUT, int P>
void launch_short(const Args& a, hipStream_t st) {
    const int passes = OUT == kMX ? 128 * P / 256 : 1;
    const unsigned grid = static_cast<unsigned>(cdiv(a.rows, 256 / P * passes));
    short_kernel<C, OUT, P><<<grid, 256, 0, st>>>(a, passes);
}

template <int C, int OUT>
void launch(const Args& a, bool vec, hipStream_t st) {
    const int pieces = OUT == kMX ? a.scale_words * 16 : static_cast<int>(cdiv(a.cols, 8));
    if (!vec) launch_rows<C, OUT, false>(a, st);
    // Many short rows: a workgroup each is a matter of launching them (replayed, bf16: 900001 rows of 128 258 us, here 92; 450000 of
    // 256 142 and 86; 220000 of 512 86 and 83, to MXFP8 95 and 85), and few of them have a place each anyway.
    else if (pieces > 64 || a.rows < 8 * device_cus()) launch_rows<C, OUT, true>(a, st);
    else if (OUT != kMX && pieces <= 8) launch_short<C, OUT, 8>(a, st);
    else if (pieces <= 16) launch_short<C, OUT, 16>(a, st);
    else if (pieces <= 32) launch_short<C, OUT, 32>(a, st);
    else launch_short<C, OUT, 64>(a, st);
}

template <int C>
void launch(const Args& a, Out out, bool vec, hipStream_t st) {
    if (out == kSame) launch<C, kSame>(a, vec, st);
    else if (out == kE4M3) launch<C, kE4M3>(a, vec, st);
    else if (out == kE5M2) launch<C, kE5M2>(a, vec, st);
    else launch<C, kMX>(a, vec, st);
}

}  // namespace norm
}  // namespace ckh

using namespace ckh;

extern "C" int ckh_rms_norm(const void* x, const void* residual, const void* weight, const void* scale, void* y, void* scales,
                            void* h, int64_t rows, int64_t cols, int64_t out_rows, int64_t out_cols, int64_t x_stride,
                            int64_t residual_stride, float eps, int x_code, int weight_code, int out_code, int mx,
                            uintptr_t stream) {
    CKH_REQUIRE(x_code == CKH_F32 || x_code == CKH_F16 || x_code == CKH_BF16, "rms_norm: unsupported dtype %d", x_code);
    CKH_REQUIRE(!weight || weight_code == CKH_F32 || weight_code == CKH_F16 || weight_code == CKH_BF16,
                "rms_norm: unsupported weight dtype %d", weight_code);
    CKH_REQUIRE(mx ? out_code == CKH_E4M3 : out_code == x_code || out_code == CKH_E4M3 || out_code == CKH_E5M2,
                "rms_norm: result of dtype %d from dtype %d", out_code, x_code);
    CKH_REQUIRE(rows >= 0 && rows <= INT32_MAX - 2048 && cols >= 0 && cols <= 65536, "rms_norm: %lld rows of %lld elements (65536 at most)",
                static_cast<long long>(rows), static_cast<long long>(cols));
    if (mx)
        CKH_REQUIRE(out_cols >= cols && out_cols % 32 == 0 && out_cols <= 65536 && out_rows >= rows && out_rows <= rup(rows, 128),
                    "rms_norm: [%lld, %lld] codes for [%lld, %lld]: rows must be a multiple of 32", static_cast<long long>(out_rows),
                    static_cast<long long>(out_cols), static_cast<long long>(rows), static_cast<long long>(cols));
    else
        CKH_REQUIRE(out_rows == rows && out_cols == cols, "rms_norm: only MXFP8 codes are padded");
    // (a launch's threads are counted in 32 bits)
    CKH_REQUIRE(rup(rows, 1024) * rup(cdiv(out_cols, 8), 64) <= UINT32_MAX, "rms_norm: too many elements (%lld rows of %lld)",
                static_cast<long long>(rows), static_cast<long long>(cols));
    if (rows == 0 || cols == 0) return CKH_OK;
    const int es = x_code == CKH_F32 ? 4 : 2;
    const norm::Out out = mx ? norm::kMX : out_code == CKH_E4M3 ? norm::kE4M3 : out_code == CKH_E5M2 ? norm::kE5M2 : norm::kSame;
    CKH_REQUIRE(x && y && (!residual || h) && (!mx || scales) && ((out != norm::kE4M3 && out != norm::kE5M2) || scale), "rms_norm: null pointer");
    CKH_REQUIRE(x_stride >= 0 && residual_stride >= 0, "rms_norm: negative stride");
    CKH_REQUIRE(aligned(x, es) && aligned(residual, es) && aligned(h, es) && aligned(weight, weight_code == CKH_F32 ? 4 : 2) &&
                    aligned(scale, 4) && aligned(scales, 4) && aligned(y, mx ? 8 : out == norm::kSame ? es : 1),
                "rms_norm: misaligned pointer");
    norm::Args a{};
    a.x = static_cast<const uint8_t*>(x), a.residual = static_cast<const uint8_t*>(residual), a.weight = static_cast<const uint8_t*>(weight);
    a.scale = static_cast<const float*>(scale);
    a.y = static_cast<uint8_t*>(y), a.h = static_cast<uint8_t*>(h), a.scales = static_cast<uint32_t*>(scales);
    a.x_row = x_stride * es, a.r_row = residual_stride * es;
    a.y_row = out == norm::kSame ? cols * es : cols;
    a.rows = static_cast<int>(rows), a.cols = static_cast<int>(cols);
    a.out_rows = static_cast<int>(out_rows), a.out_cols = static_cast<int>(out_cols);
    a.scale_words = static_cast<int>(cdiv(out_cols / 32, 4));
    a.weight_code = weight_code;
    a.eps = eps, a.inv_cols = 1.0f / static_cast<float>(cols);
    const bool vec = cols % 8 == 0 && aligned(x, 16) && a.x_row % 16 == 0 && aligned(weight, 16) && aligned(y, 16) &&
                     (!residual || (aligned(residual, 16) && a.r_row % 16 == 0 && aligned(h, 16)));
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (x_code == CKH_F32) norm::launch<CKH_F32>(a, out, vec, st);
    else if (x_code == CKH_F16) norm::launch<CKH_F16>(a, out, vec, st);
    else norm::launch<CKH_BF16>(a, out, vec, st);
    return check_launch("rms_norm");
}
