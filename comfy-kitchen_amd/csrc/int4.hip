// Weight-only 4-bit linears for gfx950: y = x W^T + bias with W[n, k] = s[n, g] (q[n, k] - z[n, g]),
// g = k / group, codes q in 0..15 (two a byte, the even k in the low nibble), and the quantizer
// and dequantizer of that format.
//
// linear_int4.  For one to some dozens of rows the call is bound by reading the codes once.
//   - The codes become MFMA operands without arithmetic: a code under the exponent bits of 128
//     (bf16) or 1024 (f16) is the number 128 + q (1024 + q), exactly, so two codes cost one
//     shift and one and-or.  The offset and the zero point leave by the group's sum:
//       sum_k x (q - z) = sum_k x (B + q) - (B + z) sum_k x,  B = 128 or 1024,
//     where sum_k x comes from one more MFMA against ones, whose result every lane holds at
//     the place of the product it corrects.  All sums are fp32; the cancellation costs some
//     2^-24 B / 8 of sum |x| |q|, far below the rounding of a 16-bit result: f16 results of K to
//     70016, of activations of one sign too, are at 1.003 of the distance in norm that the rounded exact
//     ones are at.
//   - v_mfma_f32_16x16x32: 16 activation rows by 16 weight rows; a lane (row r = lane % 16,
//     quarter c = lane / 16) loads 16 bytes = 32 codes of weight row r, so a wave's load takes
//     64 bytes of 16 rows.  Word j of the four lanes of a row then has to hold codes of one
//     32-code block, so that a scale belongs to one MFMA: a 4x4 transpose of words over the
//     lane quarters, in four lane-swap instructions.
//   - D[token][weight row]: the scale a lane needs is the one of the weight row it loads.
//   - A workgroup owns 16 R weight rows; its waves split K and add their sums in LDS in wave
//     order, so results do not depend on timing.
#include <algorithm>
#include <type_traits>

#include "ckh_common.h"

namespace ckh {
namespace i4 {

typedef unsigned v4u __attribute__((ext_vector_type(4)));
typedef unsigned v2u __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

constexpr int kScaleGroups = 128;  // groups whose scales are in LDS at a time
constexpr int kTileRows = 32;       // tile_kernel: activation rows of a workgroup
constexpr int kTileWaves = 8;       // and its waves, of 16 weight rows each
constexpr int kTileTarget = 3;      // half-workgroups wanted a CU
constexpr int kMaxSplits = 16;
constexpr int64_t kSplitBytes = 64 << 20;  // of the sums of ranges that only their groups ask for
constexpr int kVecCodes = 8192;    // matvec_kernel: codes whose activations are in LDS at a time, half as many for 4 rows

struct LinearArgs {
    const void* x;
    const uint8_t* codes;
    const void* scales;
    const uint8_t* zeros;  // null: every zero point is 8
    const void* bias;      // null: none
    void* y;
    int64_t x_stride;  // elements between activation rows
    int m, n, k, groups, group;
    FastDiv by_group;  // by the blocks of 32 codes of a group
    int chunk;  // steps of 128 codes whose groups fit kScaleGroups
    int scale_code, bias_code;
    int splits;   // tile_kernel: ranges of K
    float* part;  // their sums, [splits][m][n]

    __device__ __forceinline__ int group_of(uint32_t block) const {
        return static_cast<int>(by_group.div(block));
    }
};

template <int XC>
__device__ __forceinline__ v4f mfma(v4u a, v4u b, v4f c) {
    if constexpr (XC == CKH_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

// The exponent bits of B for two values, held in a vector register: one and-or instruction takes a
// constant from there and the mask from a scalar one, where two scalars would cost two instructions.
template <int XC>
__device__ __forceinline__ uint32_t base_bits() {
    uint32_t v = XC == CKH_BF16 ? 0x43004300u : 0x64006400u;
    __asm__("" : "+v"(v));
    return v;
}

// The 8 codes of a word as B + q, in the order (k0 k4)(k1 k5)(k2 k6)(k3 k7).
__device__ __forceinline__ v4u widen(uint32_t w, uint32_t base) {
    return v4u{(w & 0x000f000fu) | base, ((w >> 4) & 0x000f000fu) | base, ((w >> 8) & 0x000f000fu) | base,
               ((w >> 12) & 0x000f000fu) | base};
}

// 8 consecutive 16-bit activations in widen()'s order.
__device__ __forceinline__ v4u pair_order(v4u x) {
    return v4u{__builtin_amdgcn_perm(x[2], x[0], 0x05040100u), __builtin_amdgcn_perm(x[2], x[0], 0x07060302u),
               __builtin_amdgcn_perm(x[3], x[1], 0x05040100u), __builtin_amdgcn_perm(x[3], x[1], 0x07060302u)};
}

// Word j of lane quarter c becomes word c of lane quarter j.
__device__ __forceinline__ v4u transpose_quarters(v4u w) {
    const v2u a = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
    const v2u b = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
    const v2u c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
    const v2u d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
    return v4u{c[0], c[1], d[0], d[1]};
}

// y[m][n] = v + bias[n], rounded.
template <int XC>
__device__ __forceinline__ void store_result(const LinearArgs& a, int m, int n, float v) {
    if (a.bias)
        v += a.bias_code == CKH_F32    ? load1<CKH_F32>(a.bias, n)
             : a.bias_code == CKH_BF16 ? load1<CKH_BF16>(a.bias, n)
                                       : load1<CKH_F16>(a.bias, n);
    static_cast<uint16_t*>(a.y)[static_cast<int64_t>(m) * a.n + n] =
        static_cast<uint16_t>(XC == CKH_BF16 ? f_to_bf16_rne(v) : f_to_f16(v));
}

// The scales and zero points of a chunk's at most kScaleGroups groups for a workgroup's 16 R rows,
// on their way to LDS as (s, -s (B + z)): 16 lanes take a row, a lane 4 groups next to each other
// (of any alignment), then the 4 that are 64 groups on.  All loads go out at once, before the codes',
// so that they are waited for alone.
template <int XC, int R, int W>
struct ScaleLoads {
    static constexpr int kPer = (16 * R + 4 * W - 1) / (4 * W);  // times that a wave takes 4 rows
    uint32_t s[kPer][2][4], z[kPer][2];

    static __device__ __forceinline__ int row_of(int i, int wave, int lane) { return (i * W + wave) * 4 + (lane >> 4); }

    __device__ __forceinline__ void load(const LinearArgs& a, int n0, int rows, int wave, int lane, int g0, int gn) {
        const bool wide = a.scale_code == CKH_F32;
#pragma unroll
        for (int i = 0; i < kPer; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int row = row_of(i, wave, lane), g = h * 64 + (lane & 15) * 4;
                const int back = max(0, g + 4 - gn);  // the row's last 4 where its end cuts the lane's
                const int64_t at = static_cast<int64_t>(n0 + row) * a.groups + g0 + g - back;
                const uint8_t* sp = static_cast<const uint8_t*>(a.scales) + at * (wide ? 4 : 2);
                z[i][h] = 0x08080808u;
                if (row >= rows || g >= gn) continue;
                if (gn < 4) {
#pragma unroll
                    for (int e = 0; e < 3; ++e) {
                        if (e >= gn) break;
                        const uint8_t* one = sp + (e + back) * (wide ? 4 : 2);
                        s[i][h][e] = wide ? *reinterpret_cast<const uint32_t*>(one) : *reinterpret_cast<const uint16_t*>(one);
                        if (a.zeros) z[i][h] = (z[i][h] & ~(255u << (8 * e))) | (static_cast<uint32_t>(a.zeros[at + back + e]) << (8 * e));
                    }
                    continue;
                }
                if (wide) {
                    uint32_t v[4];
                    __builtin_memcpy(v, sp, 16);
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[i][h][e] = back == 0 ? v[e] : back == 1 ? v[min(e + 1, 3)] : back == 2 ? v[min(e + 2, 3)] : v[3];
                } else {
                    uint64_t v;
                    __builtin_memcpy(&v, sp, 8);
                    v >>= 16 * back;
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[i][h][e] = static_cast<uint32_t>(v >> (16 * e)) & 0xffffu;
                }
                if (a.zeros) {
                    __builtin_memcpy(&z[i][h], a.zeros + at, 4);
                    z[i][h] >>= 8 * back;
                }
            }
    }

    __device__ __forceinline__ void store(const LinearArgs& a, v2f (*sp)[16 * R + 1], int rows, int wave, int lane, int gn) const {
        constexpr float kBase = XC == CKH_BF16 ? 128.0f : 1024.0f;
#pragma unroll
        for (int i = 0; i < kPer; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int row = row_of(i, wave, lane), g = h * 64 + (lane & 15) * 4 + e;
                    const float v = a.scale_code == CKH_F32    ? as_f(s[i][h][e])
                                    : a.scale_code == CKH_BF16 ? bf16_to_f(s[i][h][e])
                                                               : f16_to_f(s[i][h][e]);
                    if (g < gn && row < rows) sp[g][row] = v2f{v, -v * (kBase + static_cast<float>((z[i][h] >> (8 * e)) & 255u))};
                }
    }
};

// XC: activation type; T: 16-row activation tiles; R: 16-row weight tiles per workgroup;
// W: waves per workgroup; U: steps of 128 codes whose loads a wave issues together; GB: the
// scale changes after GB blocks of 32 codes (4: at most once a step).
template <int XC, int T, int R, int W, int U, int GB>
__global__ __launch_bounds__(W * 64) void linear_kernel(LinearArgs a) {
    constexpr int kRows = 16 * R;
    constexpr int kSums = W * R * T * 4 * 64 * 4;  // bytes of the waves' sums
    constexpr int kScales = kScaleGroups * (kRows + 1) * 8;
    __shared__ __attribute__((aligned(16))) uint8_t lds[kSums > kScales ? kSums : kScales];
    v2f(*sp)[kRows + 1] = reinterpret_cast<v2f(*)[kRows + 1]>(lds);  // [group][row]: s, -s (B + z)
    float(*red)[R * T * 4][64] = reinterpret_cast<float(*)[R * T * 4][64]>(lds);

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, quarter = lane >> 4;
    const int n0 = blockIdx.x * kRows;
    const int rows = min(kRows, a.n - n0), toks = a.m;  // at most 16 T
    const int pitch = a.k >> 1;  // code bytes per weight row

    const __amdgpu_buffer_rsrc_t rw = buffer_rsrc(a.codes + static_cast<int64_t>(n0) * pitch, rows * pitch);
    const __amdgpu_buffer_rsrc_t rx =
        buffer_rsrc(a.x, static_cast<uint32_t>(((toks - 1) * a.x_stride + a.k) * 2));

    // Weight rows past N and activation rows past M repeat the last one: what they give is not stored.
    uint32_t ow[R], ox[T];
#pragma unroll
    for (int r = 0; r < R; ++r) ow[r] = min(r * 16 + r16, rows - 1) * pitch + quarter * 16;
#pragma unroll
    for (int t = 0; t < T; ++t)
        ox[t] = static_cast<uint32_t>((min(t * 16 + r16, toks - 1) * a.x_stride + quarter * 8) * 2);

    const uint32_t base = base_bits<XC>();
    const v4u ones = XC == CKH_BF16 ? v4u{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u}
                                    : v4u{0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u};

    struct Step {
        v4u w[R], x[T][4];
    };
    // Step s's loads.  Where K ends inside the step, words of later codes (of the next row, or
    // zeros past the operand) arrive, which use() leaves alone.  (A step's place is part of the offset
    // that the descriptor's bounds are checked for; the instruction's scalar offset is not.)
    const auto load = [&](Step& d, int s) {
        const int kq = s * 128;
#pragma unroll
        for (int r = 0; r < R; ++r)
            d.w[r] = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(rw, ow[r] + (kq >> 1), 0, 0));
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                d.x[t][j] = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(rx, ox[t] + kq * 2 + j * 64, 0, 0));
    };
    v4f total[R][T];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int t = 0; t < T; ++t) total[r][t] = v4f{0, 0, 0, 0};
    int g0 = 0;  // the staged groups' first
    // Adds the products of step s's first `blocks` blocks of 32 codes.
    const auto use = [&](Step& d, int s, int blocks) {
        v4f acc[R][T], sum[T];
#pragma unroll
        for (int r = 0; r < R; ++r) d.w[r] = transpose_quarters(d.w[r]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (j < blocks) {
                const bool fresh = j % GB == 0;
#pragma unroll
                for (int t = 0; t < T; ++t) {
                    d.x[t][j] = pair_order(d.x[t][j]);
                    sum[t] = mfma<XC>(d.x[t][j], ones, fresh ? v4f{0, 0, 0, 0} : sum[t]);
                }
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const v4u b = widen(d.w[r][j], base);
#pragma unroll
                    for (int t = 0; t < T; ++t) acc[r][t] = mfma<XC>(d.x[t][j], b, fresh ? v4f{0, 0, 0, 0} : acc[r][t]);
                }
            }
            if (j % GB == GB - 1 && j - (GB - 1) < blocks) {
                const int g = a.group_of(s * 4 + j - (GB - 1)) - g0;
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const v2f p = sp[g][r * 16 + r16];
#pragma unroll
                    for (int t = 0; t < T; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            total[r][t][i] = __fmaf_rn(p[0], acc[r][t][i], __fmaf_rn(p[1], sum[t][i], total[r][t][i]));
                }
            }
            if constexpr (GB < 4) __builtin_amdgcn_sched_barrier(0);  // else every block's scales are read ahead, into scratch
        }
    };

    const int steps = (a.k + 127) >> 7;
    for (int c0 = 0; c0 < steps; c0 += a.chunk) {  // one round unless K has very many groups
        const int c1 = min(steps, c0 + a.chunk);
        const int per = (c1 - c0 + W - 1) / W;
        const int first = c0 + wave * per, last = min(c1, first + per);
        const int full = min(last, a.k >> 7);
        int s0 = first;
        g0 = a.group_of(c0 * 4);
        const int gn = min(a.groups, a.group_of(c1 * 4 - 1) + 1) - g0;
        ScaleLoads<XC, R, W> sl;
        sl.load(a, n0, rows, wave, lane, g0, gn);
        Step d[U];
        const bool ahead = s0 + U <= full;
        if (ahead) {
#pragma unroll
            for (int u = 0; u < U; ++u) load(d[u], s0 + u);
        }
        if (c0 > 0) __syncthreads();
        sl.store(a, sp, rows, wave, lane, gn);
        __syncthreads();
        if (ahead) {
#pragma unroll
            for (int u = 0; u < U; ++u) use(d[u], s0 + u, 4);
            s0 += U;
        }
        for (; s0 + U <= full; s0 += U) {
#pragma unroll
            for (int u = 0; u < U; ++u) load(d[u], s0 + u);
#pragma unroll
            for (int u = 0; u < U; ++u) use(d[u], s0 + u, 4);
        }
        for (; s0 < last; ++s0) {
            load(d[0], s0);
            use(d[0], s0, min(4, (a.k >> 5) - s0 * 4));
        }
    }

    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) red[wave][(r * T + t) * 4 + i][lane] = total[r][t][i];
    __syncthreads();
    for (int e = threadIdx.x; e < R * T * 4 * 64; e += W * 64) {
        const int l = e & 63, slot = e >> 6;
        float v = red[0][slot][l];
#pragma unroll
        for (int w = 1; w < W; ++w) v += red[w][slot][l];
        const int row = slot / (4 * T) * 16 + (l & 15);
        const int tok = slot / 4 % T * 16 + (l >> 4) * 4 + (slot & 3);
        if (row < rows && tok < toks) store_result<XC>(a, tok, n0 + row, v);
    }
}

// The same for at most MT = 1, 2 or 4 activation rows, staged in LDS once for the workgroup in the
// operand's order (lanes of the 16-row operand repeat the MT rows), so that the step reads nothing
// but codes from memory; a wave keeps D steps of codes in flight.
template <int XC, int MT, int R, int W, int D, int GB>
__global__ __launch_bounds__(W * 64, MT > 1 && GB == 1 ? 3 : 4) void matvec_kernel(LinearArgs a) {
    constexpr int kRows = 16 * R;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    v4u* xs = reinterpret_cast<v4u*>(lds);  // [8 codes][row]
    const int x_bytes = min(a.k, a.chunk * 128) / 8 * MT * 16;
    v2f(*sp)[kRows + 1] = reinterpret_cast<v2f(*)[kRows + 1]>(lds + x_bytes);  // [group][row]: s, -s (B + z)
    float(*red)[R * 4][64] = reinterpret_cast<float(*)[R * 4][64]>(lds);

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, quarter = lane >> 4;
    const int n0 = blockIdx.x * kRows;
    const int rows = min(kRows, a.n - n0);
    const int pitch = a.k >> 1;  // code bytes per weight row

    const uint8_t* wbase = a.codes + static_cast<int64_t>(n0) * pitch;
    const __amdgpu_buffer_rsrc_t rw = buffer_rsrc(wbase, rows * pitch);
    const __amdgpu_buffer_rsrc_t none = buffer_rsrc(wbase, 0);
    const __amdgpu_buffer_rsrc_t rx = buffer_rsrc(a.x, static_cast<uint32_t>(((a.m - 1) * a.x_stride + a.k) * 2));
    constexpr int kAhead = 3;  // activation loads a thread issues before the codes'
    uint32_t ow[R];
#pragma unroll
    for (int r = 0; r < R; ++r) ow[r] = min(r * 16 + r16, rows - 1) * pitch + quarter * 16;

    const uint32_t base = base_bits<XC>();
    const v4u ones = XC == CKH_BF16 ? v4u{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u}
                                    : v4u{0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u};

    v4f total[R];
#pragma unroll
    for (int r = 0; r < R; ++r) total[r] = v4f{0, 0, 0, 0};
    int g0 = 0, c0 = 0;  // the staged groups' first, the chunk's first step
    const auto use = [&](const v4u (&codes)[R], int s, int blocks) {
        v4f acc[R], sum;
        v4u w[R];
#pragma unroll
        for (int r = 0; r < R; ++r) w[r] = transpose_quarters(codes[r]);
        const v4u* xp = xs + ((s - c0) * 16 + quarter) * MT + (r16 & (MT - 1));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (j < blocks) {
                const bool fresh = j % GB == 0;
                const v4u x = xp[j * 4 * MT];
                sum = mfma<XC>(x, ones, fresh ? v4f{0, 0, 0, 0} : sum);
#pragma unroll
                for (int r = 0; r < R; ++r) acc[r] = mfma<XC>(x, widen(w[r][j], base), fresh ? v4f{0, 0, 0, 0} : acc[r]);
            }
            if (j % GB == GB - 1 && j - (GB - 1) < blocks) {
                const int g = a.group_of(s * 4 + j - (GB - 1)) - g0;
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const v2f p = sp[g][r * 16 + r16];
#pragma unroll
                    for (int i = 0; i < MT; ++i)
                        total[r][i] = __fmaf_rn(p[0], acc[r][i], __fmaf_rn(p[1], sum[i], total[r][i]));
                }
            }
            if constexpr (GB < 4) __builtin_amdgcn_sched_barrier(0);
        }
    };

    const int steps = (a.k + 127) >> 7;
    for (; c0 < steps; c0 += a.chunk) {  // one round unless K is very long or has very many groups
        const int c1 = min(steps, c0 + a.chunk);
        const int per = (c1 - c0 + W - 1) / W;
        const int first = c0 + wave * per, last = min(c1, first + per);
        const int full = min(last, a.k >> 7);
        v4u w[D][R];
        const auto load = [&](v4u (&d)[R], int s) {
#pragma unroll
            for (int r = 0; r < R; ++r)
                d[r] = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(s < last ? rw : none, ow[r] + s * 64, 0, 0));
        };
        // activations and scales first, codes behind them
        g0 = a.group_of(c0 * 4);
        const int gn = min(a.groups, a.group_of(c1 * 4 - 1) + 1) - g0;
        const int units = (min(a.k, c1 * 128) - c0 * 128) >> 3;  // 8 activations each
        const auto x_at = [&](int e) {
            const int unit = e / MT, tok = e % MT;
            return e < units * MT ? static_cast<uint32_t>((min(tok, a.m - 1) * a.x_stride + c0 * 128 + unit * 8) * 2) : 0x80000000u;
        };
        v4u xr[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            xr[i] = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(rx, x_at(threadIdx.x + i * W * 64), 0, 0));
        ScaleLoads<XC, R, W> sl;
        sl.load(a, n0, rows, wave, lane, g0, gn);
#pragma unroll
        for (int u = 0; u < D; ++u) load(w[u], first + u);
        if (c0 > 0) __syncthreads();
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int e = threadIdx.x + i * W * 64;
            if (e < units * MT) xs[e] = pair_order(xr[i]);
        }
        sl.store(a, sp, rows, wave, lane, gn);
        for (int e = threadIdx.x + kAhead * W * 64; e < units * MT; e += W * 64)
            xs[e] = pair_order(__builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(rx, x_at(e), 0, 0)));
        __syncthreads();
        int s0 = first;
        for (; s0 + D <= full; s0 += D) {
#pragma unroll
            for (int u = 0; u < D; ++u) {
                use(w[u], s0 + u, 4);
                load(w[u], s0 + u + D);
            }
        }
#pragma unroll
        for (int u = 0; u < D; ++u)
            if (s0 + u < last) use(w[u], s0 + u, min(4, (a.k >> 5) - (s0 + u) * 4));
    }

    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < MT; ++i) red[wave][r * 4 + i][lane] = total[r][i];
    __syncthreads();
    for (int e = threadIdx.x; e < R * MT * 16; e += W * 64) {
        const int l = e & 15, i = (e >> 4) % MT, r = (e >> 4) / MT;
        float v = red[0][r * 4 + i][l];
#pragma unroll
        for (int w = 1; w < W; ++w) v += red[w][r * 4 + i][l];
        if (r * 16 + l < rows && i < a.m) store_result<XC>(a, i, n0 + r * 16 + l, v);
    }
}

// More rows: a workgroup takes 32 activation rows, 128 weight rows (eight waves of 16) and one of
// `splits` ranges of K, and its waves share the activations, which go through LDS in the operand's
// order (two buffers, a barrier a step): read by every wave itself they would cost more than the
// codes.  Where K is split, the sums go to memory in fp32 and reduce_kernel adds them in order.
// ROUNDS: a range has more groups than LDS holds, and is taken in equal parts that stage theirs.
// 24 rows, N = 5120, K = 13824 (35 MB of codes): 22-25 us, 1.5 TB/s.  Some 5 of them are the second
// launch, 6 the way to the first step and back, the rest is bound by the loads: with the products
// taken out it takes as long, without the activations' loads 5 us less, without the codes' 3.
// 64 weight rows a workgroup 26 (64 rows, N = 13824, K = 5120: 42 against 34), six steps of codes in
// flight 24.4, two 23.7; 256-byte runs of an activation row a load (whole lines) 25.1, for their
// writes to LDS meet on banks; two or four workgroups' halves a CU 27.
template <int XC, int GB, bool ROUNDS>
__global__ __launch_bounds__(kTileWaves * 64, GB == 1 ? 3 : 4) void tile_kernel(LinearArgs a) {
    constexpr int T = kTileRows / 16, R = 1;  // 16-row tiles of activations, and of a wave's weight rows
    constexpr int W = kTileWaves, D = 4, DX = 2;  // waves; steps of codes, of activations in flight
    static_assert(D % DX == 0 && D % 2 == 0, "a step's registers and buffer are known by its place in the loop");
    constexpr int kRows = 16 * R * W;
    constexpr int kUnits = T * 256;       // 16-byte pieces of a step's activations
    constexpr int kPer = kUnits / (W * 64);  // a thread's
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    v4u* xs = reinterpret_cast<v4u*>(lds);  // [2][block][tile][quarter][row]
    v2f(*sp)[16 * R * W + 1] = reinterpret_cast<v2f(*)[16 * R * W + 1]>(lds + 2 * kUnits * 16);

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, quarter = lane >> 4;
    const int n0 = blockIdx.x * kRows, m0 = blockIdx.z * 16 * T;
    const int rows = min(kRows, a.n - n0), toks = min(16 * T, a.m - m0);
    const int pitch = a.k >> 1;  // code bytes per weight row
    const int steps = (a.k + 127) >> 7;
    const int first = static_cast<int>(static_cast<int64_t>(steps) * blockIdx.y / a.splits);
    const int last = static_cast<int>(static_cast<int64_t>(steps) * (blockIdx.y + 1) / a.splits);

    const uint8_t* wbase = a.codes + static_cast<int64_t>(n0) * pitch;
    const __amdgpu_buffer_rsrc_t rw = buffer_rsrc(wbase, rows * pitch);
    const __amdgpu_buffer_rsrc_t none = buffer_rsrc(wbase, 0);
    const __amdgpu_buffer_rsrc_t rx =
        buffer_rsrc(static_cast<const uint16_t*>(a.x) + m0 * a.x_stride,
                    static_cast<uint32_t>(((toks - 1) * a.x_stride + a.k) * 2));
    uint32_t ow[R];
#pragma unroll
    for (int r = 0; r < R; ++r) ow[r] = min((wave * R + r) * 16 + r16, rows - 1) * pitch + quarter * 16;
    // piece e of a step: its block and tile by the wave, its quarter and row as the operand's lanes
    uint32_t ox[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int e = threadIdx.x + i * W * 64, l = e & 63, t = (e >> 6) % T, j = (e >> 6) / T;
        ox[i] = static_cast<uint32_t>((min(t * 16 + (l & 15), toks - 1) * a.x_stride + j * 32 + (l >> 4) * 8) * 2);
    }
    v4u w[D][R], x[DX][kPer];
    const auto load_codes = [&](v4u (&d)[R], int s, int end) __attribute__((always_inline)) {
#pragma unroll
        for (int r = 0; r < R; ++r)
            d[r] = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(s < end ? rw : none, ow[r] + s * 64, 0, 0));
    };
    const auto load_x = [&](v4u (&d)[kPer], int s) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            d[i] = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(rx, ox[i] + s * 256, 0, 0));
    };
    const auto store_x = [&](const v4u (&d)[kPer], int buffer) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) xs[buffer * kUnits + threadIdx.x + i * W * 64] = pair_order(d[i]);
    };

    const uint32_t base = base_bits<XC>();
    const v4u ones = XC == CKH_BF16 ? v4u{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u}
                                    : v4u{0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u};
    v4f total[R][T];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int t = 0; t < T; ++t) total[r][t] = v4f{0, 0, 0, 0};
    int g0 = 0;  // the staged groups' first
    const auto use = [&](const v4u (&codes)[R], int s, int buffer, auto blocks) __attribute__((always_inline)) {
        v4f acc[R][T], sum[T];
        v4u c[R];
#pragma unroll
        for (int r = 0; r < R; ++r) c[r] = transpose_quarters(codes[r]);
        const v4u* xp = xs + buffer * kUnits + lane;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (j < blocks) {
                const bool fresh = j % GB == 0;
                v4u b[R];
#pragma unroll
                for (int r = 0; r < R; ++r) b[r] = widen(c[r][j], base);
#pragma unroll
                for (int t = 0; t < T; ++t) {
                    const v4u f = xp[(j * T + t) * 64];
                    sum[t] = mfma<XC>(f, ones, fresh ? v4f{0, 0, 0, 0} : sum[t]);
#pragma unroll
                    for (int r = 0; r < R; ++r) acc[r][t] = mfma<XC>(f, b[r], fresh ? v4f{0, 0, 0, 0} : acc[r][t]);
                }
            }
            if (j % GB == GB - 1 && j - (GB - 1) < blocks) {
                const int g = a.group_of(s * 4 + j - (GB - 1)) - g0;
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const v2f p = sp[g][(wave * R + r) * 16 + r16];
#pragma unroll
                    for (int t = 0; t < T; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            total[r][t][i] = __fmaf_rn(p[0], acc[r][t][i], __fmaf_rn(p[1], sum[t][i], total[r][t][i]));
                }
            }
        }
    };

    // Steps c0 .. c1 - 1, whose groups LDS holds.  The last barrier of a round before K's end frees what the
    // next one stages.
    const auto round = [&](int c0, int c1) __attribute__((always_inline)) {
        g0 = a.group_of(c0 * 4);
        const int gn = min(a.groups, a.group_of(c1 * 4 - 1) + 1) - g0;
        int at = lane;
        if constexpr (ROUNDS) __asm__ volatile("" : "+v"(at));  // else its places are kept in registers for the next
        ScaleLoads<XC, R * W, W> sl;
        if constexpr (ROUNDS) {  // beside the sums, registers do not hold scales and codes on their way
            sl.load(a, n0, rows, wave, at, g0, gn);
            sl.store(a, sp, rows, wave, at, gn);
        }
        load_x(x[0], c0);
        if constexpr (!ROUNDS) sl.load(a, n0, rows, wave, at, g0, gn);
#pragma unroll
        for (int u = 1; u < DX; ++u) load_x(x[u], c0 + u);
#pragma unroll
        for (int u = 0; u < D; ++u) load_codes(w[u], c0 + u, c1);
        store_x(x[0], 0);
        if constexpr (!ROUNDS) sl.store(a, sp, rows, wave, at, gn);
        __syncthreads();
        const int full = min(c1, a.k >> 7);  // whole steps; K may end inside the last
        for (int s0 = c0; s0 < full; s0 += D) {
#pragma unroll
            for (int u = 0; u < D; ++u) {
                const int s = s0 + u;
                if (s >= full) break;
                load_x(x[u % DX], s + DX);  // past the round: unused, within the operand or zeros
                use(w[u], s, u & 1, std::integral_constant<int, 4>{});
                load_codes(w[u], s + D, c1);
                store_x(x[(u + 1) % DX], (u + 1) & 1);
                __syncthreads();
            }
        }
        if (full < c1) {
            load_codes(w[0], full, c1);
            use(w[0], full, (full - c0) & 1, (a.k >> 5) - full * 4);
        }
    };
    if constexpr (ROUNDS) {
        const int rounds = (last - first + a.chunk - 1) / a.chunk, per = (last - first + rounds - 1) / rounds;
#pragma unroll 1
        for (int c0 = first; c0 < last; c0 += per) round(c0, min(last, c0 + per));
    } else {
        round(first, last);
    }

#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int row = (wave * R + r) * 16 + r16;
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int tok = t * 16 + quarter * 4 + i;
                if (row < rows && tok < toks) {
                    if (a.splits == 1) store_result<XC>(a, m0 + tok, n0 + row, total[r][t][i]);
                    else a.part[(static_cast<int64_t>(blockIdx.y) * a.m + m0 + tok) * a.n + n0 + row] = total[r][t][i];
                }
            }
    }
}

template <int XC>
__global__ __launch_bounds__(256) void reduce_kernel(LinearArgs a) {
    const int64_t size = static_cast<int64_t>(a.m) * a.n, at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (at >= size) return;
    float v = a.part[at];
#pragma unroll 8
    for (int s = 1; s < a.splits; ++s) v += a.part[s * size + at];
    const int m = static_cast<int>(at / a.n);
    store_result<XC>(a, m, static_cast<int>(at - static_cast<int64_t>(m) * a.n), v);
}

// Steps of 128 codes that touch at most kScaleGroups groups, wherever the first begins.
int chunk_steps(int64_t group) {
    return static_cast<int>((128 % group == 0 ? kScaleGroups : kScaleGroups - 1) * group / 128);
}

template <int XC, int T, int R, int W, int U>
void launch_linear(const LinearArgs& a, hipStream_t st) {
    const unsigned grid = static_cast<unsigned>(cdiv(a.n, 16 * R));
    if (a.group % 128 == 0)
        linear_kernel<XC, T, R, W, U, 4><<<grid, W * 64, 0, st>>>(a);
    else if (a.group % 64 == 0)
        linear_kernel<XC, T, R, W, U, 2><<<grid, W * 64, 0, st>>>(a);
    else
        linear_kernel<XC, T, R, W, U, 1><<<grid, W * 64, 0, st>>>(a);
}

template <int XC, int MT, int R, int W, int D, int GB>
void launch_matvec(LinearArgs a, hipStream_t st) {
    a.chunk = std::min(a.chunk, kVecCodes / 128 / (MT > 1 ? 2 : 1));
    const int codes = std::min(a.k, a.chunk * 128);
    const int groups = std::min(a.groups, std::min(kScaleGroups, codes / a.group + 2));
    const size_t lds = std::max<size_t>(codes / 8 * MT * 16 + groups * (16 * R + 1) * 8, W * R * 4 * 64 * 4);
    matvec_kernel<XC, MT, R, W, D, GB><<<static_cast<unsigned>(cdiv(a.n, 16 * R)), W * 64, lds, st>>>(a);
}

template <int XC, int MT, int R, int W, int D>
void launch_matvec(const LinearArgs& a, hipStream_t st) {
    if (a.group % 128 == 0) launch_matvec<XC, MT, R, W, D, 4>(a, st);
    else if (a.group % 64 == 0) launch_matvec<XC, MT, R, W, D, 2>(a, st);
    else launch_matvec<XC, MT, R, W, D, 1>(a, st);
}

// Ranges of K for a call (1: not split), 0 where tile_kernel does not serve it: few rows, or rows that
// linear_kernel's 64-row workgroups serve better (32 rows, N = 13824, K = 5120: 22.5 against 24).
// Three workgroups for two CUs are wanted, of four steps at least.  Where that leaves a range more
// groups than LDS holds, K is split further while the ranges' sums stay within kSplitBytes (groups of
// 32, N = 5120, K = 13824: 256 rows 138 us, in rounds 162; 512 rows 270 against 305), and else
// the range goes in rounds (1024 rows 507, in ranges 535; 4096 rows 1988 against 2120), so that
// a prompt's workspace does not grow with its rows.
int tile_splits(int64_t m, int64_t n, int64_t k, int64_t group, bool may_split) {
    const int cus = device_cus();
    if (m <= 16 || (m <= 32 && n > 48 * cus)) return 0;
    const int64_t blocks = cdiv(n, 16 * kTileWaves) * cdiv(m, kTileRows), steps = cdiv(k, 128);
    if (!may_split) return 1;
    const int64_t s = std::min<int64_t>({kMaxSplits, cdiv(kTileTarget * cus, 2 * blocks), std::max<int64_t>(1, steps / 4)});
    const int64_t whole = std::min<int64_t>(kMaxSplits, cdiv(steps, chunk_steps(group)));  // ranges of one round
    return static_cast<int>(whole > s && whole * m * n * 4 <= kSplitBytes ? whole : s);
}

template <int XC, bool ROUNDS>
void launch_tile(const LinearArgs& a, dim3 grid, size_t lds, hipStream_t st) {
    if (a.group % 128 == 0) tile_kernel<XC, 4, ROUNDS><<<grid, kTileWaves * 64, lds, st>>>(a);
    else if (a.group % 64 == 0) tile_kernel<XC, 2, ROUNDS><<<grid, kTileWaves * 64, lds, st>>>(a);
    else tile_kernel<XC, 1, ROUNDS><<<grid, kTileWaves * 64, lds, st>>>(a);
}

template <int XC>
void launch_tile(const LinearArgs& a, hipStream_t st) {
    const dim3 grid(static_cast<unsigned>(cdiv(a.n, 16 * kTileWaves)), static_cast<unsigned>(a.splits), static_cast<unsigned>(cdiv(a.m, kTileRows)));
    const int64_t range = cdiv(cdiv(a.k, 128), a.splits), codes = std::min<int64_t>(a.chunk, range) * 128;
    const int64_t groups = std::min<int64_t>({a.groups, kScaleGroups, codes / a.group + 2});
    const size_t lds = 2 * kTileRows * 256 + groups * (16 * kTileWaves + 1) * 8;  // two steps' activations, the scales
    if (range <= a.chunk) launch_tile<XC, false>(a, grid, lds, st);
    else launch_tile<XC, true>(a, grid, lds, st);
    if (a.splits > 1) reduce_kernel<XC><<<static_cast<unsigned>(cdiv(static_cast<int64_t>(a.m) * a.n, 256)), 256, 0, st>>>(a);
}

// Tiles and waves by the rows of x and by whether the tiles fill the 256 CUs (us at K = 5120 and
// N = 13824, groups of 128, unless said; the operands not in cache):
//   1 row      16 weight rows a workgroup; 4 waves from two workgroups a CU on (11.3; 8 waves 12.5),
//              else 8 (N = 5120: 6.8; 4 waves 7.3)
//   2-4 rows   32 weight rows from one workgroup a CU on (14.2; 16 rows 16.3), else, and with groups
//              under 128 (their scales would not fit the registers), 16
//   5-16 rows  32 weight rows, 8 waves (16.7; 16 rows 19.9), 16 waves where there are fewer
//              workgroups than CUs (N = K = 5120, 16 rows: 12.0 against 13.6)
//   more       tile_kernel (64 rows: 34; linear_kernel 45), but linear_kernel, 64 weight rows a
//              workgroup, for up to 32 rows of wide layers (tile_splits)
template <int XC>
void linear(const LinearArgs& a, hipStream_t st) {
    const int cus = device_cus();
    if (a.splits > 0) {
        launch_tile<XC>(a, st);
    } else if (a.m == 1) {
        if (a.n > 32 * cus) launch_matvec<XC, 1, 1, 4, 2>(a, st);
        else launch_matvec<XC, 1, 1, 8, 2>(a, st);
    } else if (a.m <= 4) {
        if (a.n > 32 * cus && a.group % 128 == 0) launch_matvec<XC, 4, 2, 8, 2, 4>(a, st);
        else launch_matvec<XC, 4, 1, 8, 2>(a, st);
    } else if (a.m <= 16) {
        if (a.n > 32 * cus) launch_linear<XC, 1, 2, 8, 1>(a, st);
        else launch_linear<XC, 1, 2, 16, 1>(a, st);
    } else {
        launch_linear<XC, 2, 4, 8, 1>(a, st);
    }
}

// ------------------------------------------------------------ quantize / dequantize
// Symmetric quantize: s = amax / 7 over the group, rounded to x's type (so that the codes fit
// the scale that is stored), q = clamp(rint(x / s), -8, 7) + 8.  16 lanes take a group.
template <int C>
__global__ __launch_bounds__(256) void quantize_kernel(const void* x, uint8_t* codes, void* scales, int64_t total,
                                                       int groups, int group, int k) {
    const int64_t id = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) >> 4;
    if (id >= total) return;  // whole groups of 16 lanes leave
    const int sub = threadIdx.x & 15;
    const int64_t row = id / groups;
    const int g = static_cast<int>(id - row * groups);
    const int begin = g * group, end = min(k, begin + group);
    float top = 0.0f;
    bool bad = false;
    for (int c = begin + sub * 8; c < end; c += 128) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[i] = load1<C>(x, row * k + c + i);
            top = fmaxf(top, fabsf(v[i]));
            bad |= is_nan(v[i]);
        }
    }
#pragma unroll
    for (int s = 8; s >= 1; s >>= 1) {
        top = fmaxf(top, __shfl_xor(top, s, 16));
        bad |= __shfl_xor(static_cast<int>(bad), s, 16) != 0;
    }
    const float scale = round_to<C>(bad ? __builtin_nanf("") : __fdiv_rn(top, 7.0f));
    for (int c = begin + sub * 8; c < end; c += 128) {
        uint32_t word = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float q = scale > 0.0f ? rintf(__fdiv_rn(load1<C>(x, row * k + c + i), scale)) : 0.0f;
            word |= static_cast<uint32_t>(static_cast<int>(fminf(fmaxf(q, -8.0f), 7.0f)) + 8) << (4 * i);
        }
        *reinterpret_cast<uint32_t*>(codes + (row * k + c) / 2) = word;
    }
    if (sub == 0) {
        if constexpr (C == CKH_F32) static_cast<float*>(scales)[id] = scale;
        else static_cast<uint16_t*>(scales)[id] = static_cast<uint16_t>(C == CKH_BF16 ? f_to_bf16(scale) : f_to_f16(scale));
    }
}

// out = (q - z) s with one rounding; a thread takes 8 codes.
template <int OC>
__global__ __launch_bounds__(256) void dequantize_kernel(const uint8_t* codes, const void* scales, const uint8_t* zeros,
                                                         void* out, int64_t words, int k, int groups, int group,
                                                         int scale_code) {
    const int64_t id = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (id >= words) return;
    const int64_t row = id / (k >> 3);
    const int c = static_cast<int>(id - row * (k >> 3)) * 8;
    const uint32_t w = reinterpret_cast<const uint32_t*>(codes)[id];
    const int64_t at = row * groups + c / group;
    const float s = scale_code == CKH_F32    ? load1<CKH_F32>(scales, at)
                    : scale_code == CKH_BF16 ? load1<CKH_BF16>(scales, at)
                                             : load1<CKH_F16>(scales, at);
    const float z = zeros ? static_cast<float>(zeros[at]) : 8.0f;
    uint32_t o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float v = (static_cast<float>((w >> (4 * i)) & 15u) - z) * s;
        o[i] = OC == CKH_F32 ? as_u(v) : OC == CKH_BF16 ? f_to_bf16(v) : f_to_f16(v);
    }
    if constexpr (OC == CKH_F32) {
        uint4* p = reinterpret_cast<uint4*>(static_cast<float*>(out) + id * 8);
        p[0] = make_uint4(o[0], o[1], o[2], o[3]);
        p[1] = make_uint4(o[4], o[5], o[6], o[7]);
    } else {
        reinterpret_cast<uint4*>(out)[id] =
            make_uint4(o[0] | (o[1] << 16), o[2] | (o[3] << 16), o[4] | (o[5] << 16), o[6] | (o[7] << 16));
    }
}

bool is_float(int code) { return code == CKH_F32 || code == CKH_F16 || code == CKH_BF16; }

}  // namespace i4
}  // namespace ckh

using namespace ckh;

// Sizes and pointers that every entry point of this file checks alike.
#define CKH_REQUIRE_INT4(fn, n, k, group)                                                                       \
    CKH_REQUIRE((n) >= 0 && (k) >= 32 && (k) % 32 == 0 && (k) <= (1 << 23), fn ": K must be a multiple of 32 in 32..2^23, got %lld", \
                static_cast<long long>(k));                                                                     \
    CKH_REQUIRE((group) >= 32 && (group) % 32 == 0 && (group) <= (1 << 23), fn ": group size must be a multiple of 32, got %lld", \
                static_cast<long long>(group));                                                                 \
    CKH_REQUIRE((n) <= INT32_MAX - 64, fn ": too many rows")

extern "C" int ckh_quantize_int4(const void* x, void* codes, void* scales, int64_t n, int64_t k, int64_t group,
                                 int in_code, uintptr_t stream) {
    CKH_REQUIRE_INT4("quantize_int4", n, k, group);
    CKH_REQUIRE(i4::is_float(in_code), "quantize_int4: unsupported input dtype %d", in_code);
    if (n == 0) return CKH_OK;
    CKH_REQUIRE(x && codes && scales, "quantize_int4: null pointer");
    CKH_REQUIRE(aligned(codes, 4) && aligned(x, in_code == CKH_F32 ? 4 : 2) && aligned(scales, in_code == CKH_F32 ? 4 : 2),
                "quantize_int4: misaligned pointer");
    const int groups = static_cast<int>(cdiv(k, group));
    const int64_t total = n * groups;
    CKH_REQUIRE(cdiv(total, 16) <= INT32_MAX, "quantize_int4: tensor too large");
    const unsigned grid = static_cast<unsigned>(cdiv(total, 16));
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    uint8_t* q = static_cast<uint8_t*>(codes);
    const int gs = static_cast<int>(group), kk = static_cast<int>(k);
    if (in_code == CKH_F32) i4::quantize_kernel<CKH_F32><<<grid, 256, 0, st>>>(x, q, scales, total, groups, gs, kk);
    else if (in_code == CKH_BF16) i4::quantize_kernel<CKH_BF16><<<grid, 256, 0, st>>>(x, q, scales, total, groups, gs, kk);
    else i4::quantize_kernel<CKH_F16><<<grid, 256, 0, st>>>(x, q, scales, total, groups, gs, kk);
    return check_launch("quantize_int4");
}

extern "C" int ckh_dequantize_int4(const void* codes, const void* scales, const void* zeros, void* out, int64_t n,
                                   int64_t k, int64_t group, int scale_code, int out_code, uintptr_t stream) {
    CKH_REQUIRE_INT4("dequantize_int4", n, k, group);
    CKH_REQUIRE(i4::is_float(out_code), "dequantize_int4: unsupported output dtype %d", out_code);
    CKH_REQUIRE(i4::is_float(scale_code), "dequantize_int4: unsupported scale dtype %d", scale_code);
    if (n == 0) return CKH_OK;
    CKH_REQUIRE(codes && scales && out, "dequantize_int4: null pointer");
    CKH_REQUIRE(aligned(codes, 4) && aligned(out, 16) && aligned(scales, scale_code == CKH_F32 ? 4 : 2),
                "dequantize_int4: misaligned pointer");
    const int64_t words = n * (k / 8);
    CKH_REQUIRE(cdiv(words, 256) <= INT32_MAX, "dequantize_int4: tensor too large");
    const unsigned grid = static_cast<unsigned>(cdiv(words, 256));
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const uint8_t* q = static_cast<const uint8_t*>(codes);
    const uint8_t* z = static_cast<const uint8_t*>(zeros);
    const int groups = static_cast<int>(cdiv(k, group)), gs = static_cast<int>(group), kk = static_cast<int>(k);
    if (out_code == CKH_F32) i4::dequantize_kernel<CKH_F32><<<grid, 256, 0, st>>>(q, scales, z, out, words, kk, groups, gs, scale_code);
    else if (out_code == CKH_BF16) i4::dequantize_kernel<CKH_BF16><<<grid, 256, 0, st>>>(q, scales, z, out, words, kk, groups, gs, scale_code);
    else i4::dequantize_kernel<CKH_F16><<<grid, 256, 0, st>>>(q, scales, z, out, words, kk, groups, gs, scale_code);
    return check_launch("dequantize_int4");
}

extern "C" int64_t ckh_linear_int4_workspace_bytes(int64_t m, int64_t n, int64_t k, int64_t group) {
    if (m <= 0 || n <= 0 || k <= 0 || group < 32) return 0;
    const int64_t s = i4::tile_splits(m, n, k, group, true);
    return s > 1 ? s * m * n * 4 : 0;
}

extern "C" int ckh_linear_int4(const void* x, const void* codes, const void* scales, const void* zeros, const void* bias,
                               void* y, int64_t m, int64_t n, int64_t k, int64_t x_stride, int64_t group, int x_code,
                               int scale_code, int bias_code, void* workspace, int64_t workspace_bytes,
                               uintptr_t stream) {
    CKH_REQUIRE_INT4("linear_int4", n, k, group);
    CKH_REQUIRE(x_code == CKH_F16 || x_code == CKH_BF16, "linear_int4: unsupported activation dtype %d", x_code);
    CKH_REQUIRE(i4::is_float(scale_code), "linear_int4: unsupported scale dtype %d", scale_code);
    CKH_REQUIRE(!bias || i4::is_float(bias_code), "linear_int4: unsupported bias dtype %d", bias_code);
    CKH_REQUIRE(m >= 0 && m <= 65535 * 16 && m * n < (int64_t(1) << 38), "linear_int4: at most %d activation rows, got %lld", 65535 * 16,
                static_cast<long long>(m));
    if (m == 0 || n == 0) return CKH_OK;
    CKH_REQUIRE(x && codes && scales && y, "linear_int4: null pointer");
    CKH_REQUIRE(x_stride >= k || m == 1, "linear_int4: activation rows overlap (stride %lld < K)", static_cast<long long>(x_stride));
    CKH_REQUIRE(aligned(x, 16) && x_stride % 8 == 0 && aligned(codes, 16) && aligned(y, 2) &&
                    aligned(scales, scale_code == CKH_F32 ? 4 : 2) && (!bias || aligned(bias, bias_code == CKH_F32 ? 4 : 2)),
                "linear_int4: misaligned pointer or row stride");
    CKH_REQUIRE(x_stride <= (int64_t(1) << 23), "linear_int4: activation row stride too large");
    const int64_t need = ckh_linear_int4_workspace_bytes(m, n, k, group);
    const bool split = need > 0 && workspace && workspace_bytes >= need && aligned(workspace, 4);
    i4::LinearArgs a{};
    a.x = x, a.codes = static_cast<const uint8_t*>(codes), a.scales = scales, a.zeros = static_cast<const uint8_t*>(zeros);
    a.bias = bias, a.y = y, a.x_stride = m == 1 ? k : x_stride;
    a.m = static_cast<int>(m), a.n = static_cast<int>(n), a.k = static_cast<int>(k);
    a.groups = static_cast<int>(cdiv(k, group)), a.group = static_cast<int>(group);
    a.by_group = fast_div(static_cast<uint32_t>(group / 32));
    a.chunk = i4::chunk_steps(group);
    a.scale_code = scale_code, a.bias_code = bias_code;
    a.splits = i4::tile_splits(m, n, k, group, split);
    a.part = static_cast<float*>(workspace);
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (x_code == CKH_BF16) i4::linear<CKH_BF16>(a, st);
    else i4::linear<CKH_F16>(a, st);
    return check_launch("linear_int4");
}
