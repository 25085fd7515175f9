// Queries and keys of new tokens turned to their positions, keys and values stored in a cache held in
// pages, for gfx950.  Pair i of the first `rotary` elements of a head turns by position * rates[i]:
//   (x, y) -> magnitude (x cos - y sin, x sin + y cos),
// the pairs being neighbours (2i, 2i + 1), or (i, i + rotary / 2); the rest of the head stays as it is.
//
// The angle's turns are taken in 64 bits and brought into -1/2 .. 1/2 before they are rounded to 32: a
// product in 32 bits would be off by 0.03 radian at position 10^6.
//
// Bound by the bytes moved.  A thread holds two 16-byte pieces of a head (in the halves' layout, partners
// of each other) and goes through several heads of its token with them, so that the angles, some 50
// instructions for each of its pairs, are made once for all of these: 14 heads a thread where there are tokens for it
// (16001 tokens of 40 + 2 x 8 heads of 128, f16, 459 MB: 93 us, 4.9 TB/s; 89 without the angles; 7 heads a thread 105 against 102 at the
// time, 4 heads 112), one where there are few (48 tokens: 5.6 us, a launch and loads that wait for each other).  q, k and v are
// read past the caches, and q' and k' written past them where they are over 128 MB (102 against 93 us there).
#include <algorithm>

#include "pages.h"

namespace ckh {
namespace pages {

enum Layout { kPairs, kHalves, kUnevenHalves };  // the last: rotary / 2 is not a multiple of 8

struct RopeArgs {
    const uint8_t* x[3];  // q, key, value
    uint8_t *q_out, *k_out;  // contiguous; k_out may be null
    uint8_t* cache[2];
    const float* scale[2];
    const void* positions;
    const float* rates;
    int64_t x_tok[3], x_head[3];  // bytes
    Strides to[2];
    Slots slots;
    bool wide_positions;
    bool past_caches;  // what attention reads next is too much for them anyway
    uint32_t threads;        // of all tokens
    int per_token, per_head; // threads of a token (spread * per_head), of a head (dim / 16)
    int spread;              // heads of a token that are worked on at once
    int heads, kv_heads, dim, rotary;
    FastDiv by_token, by_head;
    float magnitude;
};

template <int XC>
__device__ __forceinline__ float widen(uint32_t h) {
    return XC == CKH_BF16 ? bf16_to_f(h) : f16_to_f(h);
}
template <int XC>
__device__ __forceinline__ uint32_t narrow(float f) {
    return XC == CKH_BF16 ? f_to_bf16_rne(f) : f_to_f16(f);
}
template <int XC>
__device__ __forceinline__ void unpack(v4u w, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = widen<XC>((w[e >> 1] >> (16 * (e & 1))) & 0xffffu);
}
template <int XC>
__device__ __forceinline__ v4u pack(const float (&v)[8]) {
    v4u w;
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = narrow<XC>(v[2 * e]) | narrow<XC>(v[2 * e + 1]) << 16;
    return w;
}
__device__ __forceinline__ v2u codes(const float (&v)[8], float s) {
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        f[e] = __fdiv_rn(v[e], s);
        f[e] = is_nan(f[e]) ? f[e] : fminf(fmaxf(f[e], -448.0f), 448.0f);
    }
    return v2u{hw_e4m3x4(f[0], f[1], f[2], f[3]), hw_e4m3x4(f[4], f[5], f[6], f[7])};
}

__device__ __forceinline__ void turn_of(double position, float rate, float magnitude, float& c, float& s) {
    // 1 / 2 pi, and the rate's product with it, as sums of two doubles: position 2^31 still has 2^-50 turns
    constexpr double kHigh = 0.15915494309189535, kLow = -9.839338337591243e-18;
    const double r = static_cast<double>(rate);
    const double high = r * kHigh, low = __fma_rn(r, kHigh, -high) + r * kLow;
    double t = position * high;
    const double rest = __fma_rn(position, high, -t) + position * low;
    t = (t - __builtin_rint(t)) + rest;
    sincospif(2.0f * static_cast<float>(t), &s, &c);
    c *= magnitude;
    s *= magnitude;
}

constexpr int kBatch = 4;  // heads whose loads a thread has in flight

template <int XC, bool F8, int LAYOUT>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs a) {
    const uint32_t i = blockIdx.x * 256u + threadIdx.x;
    if (i >= a.threads) return;
    const uint32_t tok = a.by_token.div(i), in = i - tok * a.per_token;
    const int first = a.by_head.div(in), p = in - first * a.per_head;
    const int all = a.heads + 2 * a.kv_heads;
    const int half = a.rotary / 2;
    // the thread's pieces of a head
    int piece[2];
    if (LAYOUT == kHalves && p < a.rotary / 16) {
        piece[0] = p, piece[1] = p + a.rotary / 16;
    } else if (LAYOUT == kHalves) {
        piece[0] = a.rotary / 8 + 2 * (p - a.rotary / 16), piece[1] = piece[0] + 1;
    } else {
        piece[0] = p, piece[1] = p + a.per_head;
    }
    const auto source = [&](int h) {
        const int n = h < a.heads ? 0 : h < a.heads + a.kv_heads ? 1 : 2;
        const int at = n == 0 ? h : n == 1 ? h - a.heads : h - a.heads - a.kv_heads;
        return a.x[n] + tok * a.x_tok[n] + at * a.x_head[n];
    };
    v4u w[kBatch][2];
    const auto load = [&](int h0) {
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const int h = h0 + b * a.spread;
            if (h < all) {
                const uint8_t* x = source(h);
                w[b][0] = __builtin_nontemporal_load(reinterpret_cast<const v4u*>(x + piece[0] * 16));
                w[b][1] = __builtin_nontemporal_load(reinterpret_cast<const v4u*>(x + piece[1] * 16));
            }
        }
    };
    load(first);
    const int64_t slot = a.slots.get(tok);
    // cos and sin: of the pairs within the pieces, of the pairs across them, or of every element's pair
    constexpr int kTurns = LAYOUT == kUnevenHalves ? 16 : 8;
    float c[kTurns], s[kTurns];
    {
        const double position = static_cast<double>(a.wide_positions ? static_cast<const int64_t*>(a.positions)[tok]
                                                                     : static_cast<const int*>(a.positions)[tok]);
#pragma unroll
        for (int n = 0; n < kTurns; ++n) {
            int pair;
            if constexpr (LAYOUT == kPairs) pair = piece[n >> 2] * 4 + (n & 3);
            else if constexpr (LAYOUT == kHalves) pair = piece[0] * 8 + n;
            else {
                const int d = piece[n >> 3] * 8 + (n & 7);
                pair = d >= a.rotary ? half : d >= half ? d - half : d;
            }
            if (pair < half) turn_of(position, a.rates[pair], a.magnitude, c[n], s[n]);
        }
    }
    const int64_t at[2] = {slot < 0 ? 0 : a.slots.offset(slot, a.to[0].page, a.to[0].tok),
                           slot < 0 ? 0 : a.slots.offset(slot, a.to[1].page, a.to[1].tok)};
    for (int h0 = first; h0 < all; h0 += kBatch * a.spread) {
        if (h0 != first) load(h0);
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const int h = h0 + b * a.spread;
            if (h >= all) break;
            const bool is_q = h < a.heads, is_v = h >= a.heads + a.kv_heads;
            const int kv = is_v ? h - a.heads - a.kv_heads : h - a.heads;
            float x[2][8];
            unpack<XC>(w[b][0], x[0]);
            unpack<XC>(w[b][1], x[1]);
            if (!is_v) {
                if constexpr (LAYOUT == kPairs) {
#pragma unroll
                    for (int n = 0; n < 8; ++n) {
                        if (piece[n >> 2] * 4 + (n & 3) >= half) continue;
                        float &u = x[n >> 2][2 * (n & 3)], &v = x[n >> 2][2 * (n & 3) + 1];
                        const float t = u * c[n] - v * s[n];
                        v = u * s[n] + v * c[n];
                        u = t;
                    }
                } else if constexpr (LAYOUT == kHalves) {
                    if (p < a.rotary / 16) {
#pragma unroll
                        for (int n = 0; n < 8; ++n) {
                            const float u = x[0][n], v = x[1][n];
                            x[0][n] = u * c[n] - v * s[n];
                            x[1][n] = u * s[n] + v * c[n];
                        }
                    }
                } else {
                    const uint16_t* from = reinterpret_cast<const uint16_t*>(source(h));
#pragma unroll
                    for (int n = 0; n < 16; ++n) {
                        const int d = piece[n >> 3] * 8 + (n & 7);
                        if (d >= a.rotary) continue;
                        const float other = widen<XC>(from[d < half ? d + half : d - half]);
                        float& y = x[n >> 3][n & 7];
                        y = d < half ? y * c[n] - other * s[n] : other * s[n] + y * c[n];
                    }
                }
            }
            const v4u y0 = is_v ? w[b][0] : pack<XC>(x[0]), y1 = is_v ? w[b][1] : pack<XC>(x[1]);
            if (is_q || (!is_v && a.k_out)) {
                uint8_t* out = (is_q ? a.q_out + (static_cast<int64_t>(tok) * a.heads + h) * a.dim * 2
                                     : a.k_out + (static_cast<int64_t>(tok) * a.kv_heads + kv) * a.dim * 2);
                if (a.past_caches) {
                    __builtin_nontemporal_store(y0, reinterpret_cast<v4u*>(out + piece[0] * 16));
                    __builtin_nontemporal_store(y1, reinterpret_cast<v4u*>(out + piece[1] * 16));
                } else {
                    *reinterpret_cast<v4u*>(out + piece[0] * 16) = y0;
                    *reinterpret_cast<v4u*>(out + piece[1] * 16) = y1;
                }
            }
            if (!is_q && slot >= 0) {
                uint8_t* to = a.cache[is_v] + (is_v ? at[1] : at[0]) + kv * a.to[is_v].head;
                if constexpr (F8) {
                    const float sc = a.scale[is_v] ? *a.scale[is_v] : 1.0f;
                    *reinterpret_cast<v2u*>(to + piece[0] * 8) = codes(x[0], sc);
                    *reinterpret_cast<v2u*>(to + piece[1] * 8) = codes(x[1], sc);
                } else {
                    __builtin_nontemporal_store(y0, reinterpret_cast<v4u*>(to + piece[0] * 16));
                    __builtin_nontemporal_store(y1, reinterpret_cast<v4u*>(to + piece[1] * 16));
                }
            }
        }
    }
}

template <int XC, bool F8>
void launch_rope(const RopeArgs& a, int layout, hipStream_t st) {
    const unsigned grid = static_cast<unsigned>(cdiv(a.threads, 256));
    if (layout == kPairs) rope_kernel<XC, F8, kPairs><<<grid, 256, 0, st>>>(a);
    else if (layout == kHalves) rope_kernel<XC, F8, kHalves><<<grid, 256, 0, st>>>(a);
    else rope_kernel<XC, F8, kUnevenHalves><<<grid, 256, 0, st>>>(a);
}

}  // namespace pages
}  // namespace ckh

using namespace ckh;

extern "C" int ckh_paged_write_rope(const void* q, const void* key, const void* value, const void* positions, const void* rates,
                                    void* q_out, void* key_out, void* k_cache, void* v_cache, const void* slots,
                                    const void* k_scale, const void* v_scale, int64_t tokens, int64_t heads, int64_t kv_heads,
                                    int64_t dim, int64_t rotary, int64_t pages, int64_t page_size, const int64_t* strides,
                                    int interleaved, float magnitude, int x_code, int cache_code, int wide_positions,
                                    int wide_slots, uintptr_t stream) {
    CKH_REQUIRE(x_code == CKH_F16 || x_code == CKH_BF16, "paged_write_rope: unsupported dtype %d", x_code);
    CKH_REQUIRE(cache_code == x_code || cache_code == CKH_E4M3, "paged_write_rope: cache dtype %d with dtype %d", cache_code, x_code);
    CKH_REQUIRE(tokens >= 0 && tokens <= INT32_MAX && heads >= 0 && kv_heads >= 0 && heads <= 65535 && kv_heads <= 65535 && dim > 0 &&
                    dim <= 65536 && dim % 16 == 0,
                "paged_write_rope: %lld heads and %lld key-value heads of %lld elements (a multiple of 16)", static_cast<long long>(heads),
                static_cast<long long>(kv_heads), static_cast<long long>(dim));
    CKH_REQUIRE(rotary >= 0 && rotary <= dim && rotary % 2 == 0, "paged_write_rope: %lld of %lld elements turned",
                static_cast<long long>(rotary), static_cast<long long>(dim));
    CKH_REQUIRE(pages > 0 && page_size > 0 && pages <= INT32_MAX && page_size <= INT32_MAX && pages * page_size <= INT32_MAX,
                "paged_write_rope: %lld pages of %lld tokens", static_cast<long long>(pages), static_cast<long long>(page_size));
    CKH_REQUIRE(cache_code == CKH_E4M3 || (!k_scale && !v_scale), "paged_write_rope: scales with a cache of dtype %d", cache_code);
    const int64_t all = heads + 2 * kv_heads, per_head = dim / 16;
    CKH_REQUIRE(tokens * all * per_head < INT32_MAX, "paged_write_rope: too many elements");
    if (tokens * all == 0) return CKH_OK;
    CKH_REQUIRE(positions && (rates || rotary == 0) && slots && strides && (heads == 0 || (q && q_out)) &&
                    (kv_heads == 0 || (key && value && k_cache && v_cache)),
                "paged_write_rope: null pointer");
    const int es = cache_code == CKH_E4M3 ? 1 : 2;
    // q, key, value: token, head each; k, v: page, token, head each (elements)
    for (int i = 0; i < 12; ++i)
        CKH_REQUIRE(strides[i] >= 0 && strides[i] * (i < 6 ? 2 : es) % 16 == 0,
                    "paged_write_rope: stride %d (%lld) is not a multiple of 16 bytes", i, static_cast<long long>(strides[i]));
    CKH_REQUIRE(aligned(q, 16) && aligned(key, 16) && aligned(value, 16) && aligned(q_out, 16) && aligned(key_out, 16) &&
                    aligned(k_cache, 16) && aligned(v_cache, 16) && aligned(rates, 4) && aligned(positions, wide_positions ? 8 : 4) &&
                    aligned(slots, wide_slots ? 8 : 4) && aligned(k_scale, 4) && aligned(v_scale, 4),
                "paged_write_rope: misaligned pointer");
    pages::RopeArgs a{};
    const void* from[3] = {q, key, value};
    for (int n = 0; n < 3; ++n) {
        a.x[n] = static_cast<const uint8_t*>(from[n]);
        a.x_tok[n] = strides[2 * n] * 2, a.x_head[n] = strides[2 * n + 1] * 2;
    }
    a.q_out = static_cast<uint8_t*>(q_out), a.k_out = static_cast<uint8_t*>(key_out);
    for (int n = 0; n < 2; ++n) {
        a.cache[n] = static_cast<uint8_t*>(n ? v_cache : k_cache);
        a.scale[n] = static_cast<const float*>(n ? v_scale : k_scale);
        a.to[n] = {strides[6 + 3 * n] * es, strides[7 + 3 * n] * es, strides[8 + 3 * n] * es};
    }
    a.positions = positions, a.rates = static_cast<const float*>(rates);
    a.slots = {slots, wide_slots != 0, pages * page_size, fast_div(static_cast<uint32_t>(page_size)), static_cast<int>(page_size)};
    a.wide_positions = wide_positions != 0;
    a.past_caches = tokens * (heads + kv_heads) * dim * 2 > (int64_t(1) << 27);
    a.heads = static_cast<int>(heads), a.kv_heads = static_cast<int>(kv_heads), a.dim = static_cast<int>(dim);
    a.rotary = static_cast<int>(rotary);
    a.magnitude = magnitude;
    a.per_head = static_cast<int>(per_head);
    // as many heads a thread as leave four workgroups a CU
    const int64_t per = std::clamp<int64_t>(tokens * all * per_head / (256 * 4 * device_cus()), 1, 16);
    a.spread = static_cast<int>(cdiv(all, per));
    a.per_token = a.spread * a.per_head;
    a.threads = static_cast<uint32_t>(tokens * a.per_token);
    a.by_token = fast_div(static_cast<uint32_t>(a.per_token)), a.by_head = fast_div(static_cast<uint32_t>(a.per_head));
    const int layout = interleaved ? pages::kPairs : rotary % 16 == 0 ? pages::kHalves : pages::kUnevenHalves;
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (x_code == CKH_BF16) {
        if (es == 1) pages::launch_rope<CKH_BF16, true>(a, layout, st);
        else pages::launch_rope<CKH_BF16, false>(a, layout, st);
    } else {
        if (es == 1) pages::launch_rope<CKH_F16, true>(a, layout, st);
        else pages::launch_rope<CKH_F16, false>(a, layout, st);
    }
    return check_launch("paged_write_rope");
}
