// Tokens of a key-value cache held in pages against up to 16 query columns, by waves that need each
// other only at their end: what single tokens' attention spends its time in.
#pragma once

#include "attn.h"

namespace ckh {
namespace attn {

constexpr int kWaves = 4;
constexpr uint32_t kOut = 0x80000000u;

// How a lane holds D dims of K and V.
template <int D, bool F8>
struct Lay {
    static constexpr int ES = F8 ? 1 : 2;
    static constexpr int KW = F8 && D % 64 == 0 ? 16 : 8;  // consecutive d of a K load
    static constexpr int NK = D / (4 * KW);                // K loads of a token row
    static constexpr int KD = KW * ES / 4;                 // words of a K load
    // V: 16 lanes take runs of `w` d each, in one or two sets
    static constexpr int SETS = D == 96 || D == 256 ? 2 : 1;
    static constexpr int width(int s) { return D == 64 ? 4 : D == 96 ? (s ? 2 : 4) : 8; }
    static constexpr int base(int s) { return s == 0 ? 0 : D == 96 ? 64 : 128; }
    static constexpr int words(int s) { return (width(s) * ES + 3) / 4; }
    static constexpr int at(int s) { return s == 0 ? 0 : words(0); }
    static constexpr int VD = words(0) + (SETS > 1 ? words(1) : 0);  // words of a token's V in a lane
};

// N words (or half of one) from a buffer or a pointer.
template <int N, bool HALF>
__device__ __forceinline__ void fetch(uint32_t* d, __amdgpu_buffer_rsrc_t rs, uint32_t off) {
    if constexpr (HALF) d[0] = __builtin_amdgcn_raw_buffer_load_b16(rs, off, 0, 0);
    else if constexpr (N == 1) d[0] = __builtin_amdgcn_raw_buffer_load_b32(rs, off, 0, 0);
    else if constexpr (N == 2) {
        const v2u x = __builtin_bit_cast(v2u, __builtin_amdgcn_raw_buffer_load_b64(rs, off, 0, 0));
        d[0] = x[0], d[1] = x[1];
    } else {
        const v4u x = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(rs, off, 0, 0));
        d[0] = x[0], d[1] = x[1], d[2] = x[2], d[3] = x[3];
    }
}
template <int N, bool HALF>
__device__ __forceinline__ void fetch(uint32_t* d, const uint8_t* p) {
    if constexpr (HALF) d[0] = *reinterpret_cast<const uint16_t*>(p);
    else if constexpr (N == 1) d[0] = *reinterpret_cast<const uint32_t*>(p);
    else if constexpr (N == 2) {
        const v2u x = *reinterpret_cast<const v2u*>(p);
        d[0] = x[0], d[1] = x[1];
    } else {
        const v4u x = *reinterpret_cast<const v4u*>(p);
        d[0] = x[0], d[1] = x[1], d[2] = x[2], d[3] = x[3];
    }
}

// Where a head's rows lie.
struct PagedRows {
    const uint8_t *k, *v;  // of the key-value head
    const int* table;      // of the sequence
    int64_t k_page, k_tok, v_page, v_tok;  // strides in elements
    int pages, page_size;
    FastDiv by_page;
};

// Tiles of 32 tokens, t0 .. t1 - 1 of them this workgroup's: those of the tokens 0 .. sink_end - 1, then those of start .. len - 1.
struct PagedTiles {
    int sink_tiles, sink_end, start, len, t0, t1;
};

// Every wave's unnormalised output, maxima and sums to lo, lm and ll.  A wave's query columns are q (column
// lane & 15; d as Lay has K's).  STEP: kWaves where the waves of the workgroup share the tiles, 1 where each has its
// own (and arguments of its own).  QC: type of q.  F8: the cache holds E4M3 codes (else QC).  WHOLE: 16 consecutive tokens are always on one page (page_size % 16 == 0), so a tile needs
// two page numbers, which are the wave's (scalar); else every lane looks up the pages of its tokens, a tile ahead.
template <int QC, int D, bool F8, bool WHOLE, int STEP = kWaves>
__device__ __forceinline__ void paged_tiles(const PagedRows& a, const PagedTiles& vis, const v4u (&q)[D / 32], float to_log2,
                                            float (&lo)[kWaves][D][17], float (&lm)[kWaves][16], float (&ll)[kWaves][16]) {
    using L = Lay<D, F8>;
    constexpr int ES = L::ES;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, c = lane >> 4;
    const int t0 = vis.t0, t1 = vis.t1;
    const int* table = a.table;
    const uint8_t *kbase = a.k, *vbase = a.v;

    struct Tile {
        uint32_t k[2][L::NK * L::KD], v[8][L::VD];
        int base, lo, hi;  // tokens base .. base + 31, of which lo .. hi - 1 are visible
    };
    const auto place_tile = [&](Tile& t, int i) {
        const int j = min(i, t1 - 1);
        const bool sink = j < vis.sink_tiles;
        t.base = (sink ? j : (vis.start >> 5) + j - vis.sink_tiles) * 32;
        t.lo = sink ? 0 : vis.start;
        t.hi = sink ? vis.sink_end : vis.len;
    };
    // Without whole pages: a lane's tokens in a tile (two of K, eight of V), taken into the visible
    // ones, and their pages, which are looked up a tile ahead of the rows they lead to.
    const auto token = [&](const Tile& t, int n) {
        const int tk = t.base + (n < 2 ? n * 16 + r16 : ((n - 2) >> 2) * 16 + 4 * c + ((n - 2) & 3));
        return max(t.lo, min(tk, t.hi - 1));
    };
    int page_of[WHOLE ? 1 : 10];
    const auto look_up = [&](int i) {
        if constexpr (!WHOLE) {
            Tile t;
            place_tile(t, i);
#pragma unroll
            for (int n = 0; n < 10; ++n) page_of[n] = table[a.by_page.div(token(t, n))];
        }
    };
    // Tile i's loads; past the chunk's end they read nothing (or the last tile again).
    const auto load = [&](Tile& t, int i) {
        const bool live = i < t1;
        place_tile(t, i);
        if constexpr (WHOLE) {
            __amdgpu_buffer_rsrc_t rk[2], rv[2];
            uint32_t ko[2], vo[8];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int tb = t.base + h * 16;
                const bool some = live && tb < t.hi && tb + 16 > t.lo;
                const int pi = a.by_page.div(tb), slot = tb - pi * a.page_size;
                const int page = some ? min(static_cast<uint32_t>(table[pi]), static_cast<uint32_t>(a.pages - 1)) : 0;
                rk[h] = buffer_rsrc(kbase + (page * a.k_page + slot * a.k_tok) * ES, some ? 0x7fffffffu : 0u);
                rv[h] = buffer_rsrc(vbase + (page * a.v_page + slot * a.v_tok) * ES, some ? 0x7fffffffu : 0u);
                ko[h] = r16 * static_cast<uint32_t>(a.k_tok * ES) + c * L::KW * ES;
#pragma unroll
                for (int e = 0; e < 4; ++e) vo[h * 4 + e] = (4 * c + e) * static_cast<uint32_t>(a.v_tok * ES);
            }
            if (t.base < t.lo || t.base + 32 > t.hi) {  // tokens that are not visible read zeros
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int tk = t.base + h * 16 + r16;
                    ko[h] = tk >= t.lo && tk < t.hi ? ko[h] : kOut;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int tv = t.base + h * 16 + 4 * c + e;
                        vo[h * 4 + e] = tv >= t.lo && tv < t.hi ? vo[h * 4 + e] : kOut;
                    }
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int n = 0; n < L::NK; ++n) fetch<L::KD, false>(t.k[h] + n * L::KD, rk[h], ko[h] + n * 4 * L::KW * ES);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                fetch<L::words(0), L::width(0) * ES == 2>(t.v[e], rv[e >> 2], vo[e] + r16 * L::width(0) * ES);
                if constexpr (L::SETS > 1)
                    fetch<L::words(1), L::width(1) * ES == 2>(t.v[e] + L::at(1), rv[e >> 2],
                                                              vo[e] + (L::base(1) + r16 * L::width(1)) * ES);
            }
        } else {
            const auto row = [&](int n, const uint8_t* base, int64_t page_stride, int64_t tok_stride) {
                const int tk = token(t, n), slot = tk - a.by_page.div(tk) * a.page_size;
                const int64_t page = min(static_cast<uint32_t>(page_of[n]), static_cast<uint32_t>(a.pages - 1));
                return base + (page * page_stride + slot * tok_stride) * ES;
            };
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint8_t* p = row(h, kbase, a.k_page, a.k_tok) + c * L::KW * ES;
#pragma unroll
                for (int n = 0; n < L::NK; ++n) fetch<L::KD, false>(t.k[h] + n * L::KD, p + n * 4 * L::KW * ES);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint8_t* p = row(2 + e, vbase, a.v_page, a.v_tok);
                fetch<L::words(0), L::width(0) * ES == 2>(t.v[e], p + r16 * L::width(0) * ES);
                if constexpr (L::SETS > 1)
                    fetch<L::words(1), L::width(1) * ES == 2>(t.v[e] + L::at(1), p + (L::base(1) + r16 * L::width(1)) * ES);
            }
            look_up(i + STEP);
        }
    };

    v4f acc[D / 16];
#pragma unroll
    for (int n = 0; n < D / 16; ++n) acc[n] = v4f{0, 0, 0, 0};
    float m = -1e30f, l = 0.0f;

    const auto use = [&](Tile& t) {
        float s[8];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            v4f x = v4f{0, 0, 0, 0};
#pragma unroll
            for (int n = 0; n < D / 32; ++n) {
                v4u kf;
                if constexpr (F8) {
                    const uint32_t w0 = t.k[h][n * 2], w1 = t.k[h][n * 2 + 1];
                    kf = v4u{widen_e4m3<QC, false>(w0), widen_e4m3<QC, true>(w0), widen_e4m3<QC, false>(w1),
                             widen_e4m3<QC, true>(w1)};
                } else {
                    kf = v4u{t.k[h][n * 4], t.k[h][n * 4 + 1], t.k[h][n * 4 + 2], t.k[h][n * 4 + 3]};
                }
                x = mfma16<QC>(kf, q[n], x);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) s[h * 4 + i] = x[i] * to_log2;
        }
        const bool edge = t.base < t.lo || t.base + 32 > t.hi;
        if (edge) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int tk = t.base + (e >> 2) * 16 + 4 * c + (e & 3);
                if (tk < t.lo || tk >= t.hi) {
                    s[e] = -__builtin_inff();
                    if constexpr (!WHOLE) {  // what was read in its place does not count, not even as NaN
#pragma unroll
                        for (int w = 0; w < L::VD; ++w) t.v[e][w] = 0;
                    }
                }
            }
        }
        float top = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
        if (__any(top > m + kLift<QC> + 8.0f)) {
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            const float to = fmaxf(m, top - kLift<QC>);
            const float f = exp2_hw(m - to);
            m = to;
            l *= f;
#pragma unroll
            for (int n = 0; n < D / 16; ++n) acc[n] *= f;
        }
        float p[8], sum = 0.0f;  // the tile's own: single small weights would be lost in a large l
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            p[e] = exp2_hw(s[e] - m);
            sum += p[e];
        }
        l += sum;
        // (rounded to the values' 16-bit type, as the product takes them: half a step of each weight, of unlike signs)
        const v4u pb = v4u{pack2<QC>(p[0], p[1]), pack2<QC>(p[2], p[3]), pack2<QC>(p[4], p[5]), pack2<QC>(p[6], p[7])};
        int n = 0;
#pragma unroll
        for (int st = 0; st < L::SETS; ++st) {
            const int w0 = st ? L::at(1) : 0, nw = st ? L::words(1) : L::words(0);
#pragma unroll
            for (int w = 0; w < nw; ++w) {
                if constexpr (!F8) {
                    v4u x, y;  // two d of 8 tokens
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        x[e] = __builtin_amdgcn_perm(t.v[2 * e + 1][w0 + w], t.v[2 * e][w0 + w], 0x05040100u);
                        y[e] = __builtin_amdgcn_perm(t.v[2 * e + 1][w0 + w], t.v[2 * e][w0 + w], 0x07060302u);
                    }
                    acc[n] = mfma16<QC>(x, pb, acc[n]);
                    acc[n + 1] = mfma16<QC>(y, pb, acc[n + 1]);
                    n += 2;
                } else {
#pragma unroll
                    for (int half = 0; half < (L::width(st) == 2 ? 1 : 2); ++half) {
                        v4u x, y;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {  // token pairs of two d, then widened
                            const uint32_t z = __builtin_amdgcn_perm(t.v[2 * e + 1][w0 + w], t.v[2 * e][w0 + w],
                                                                     half ? 0x07030602u : 0x05010400u);
                            x[e] = widen_e4m3<QC, false>(z);
                            y[e] = widen_e4m3<QC, true>(z);
                        }
                        acc[n] = mfma16<QC>(x, pb, acc[n]);
                        acc[n + 1] = mfma16<QC>(y, pb, acc[n + 1]);
                        n += 2;
                    }
                }
            }
        }
    };

    int i = t0 + (STEP > 1 ? wave : 0);
    if (i < t1) {
        Tile x, y;
        look_up(i);
        load(x, i);
        for (;;) {
            load(y, i + STEP);
            use(x);
            i += STEP;
            if (i >= t1) break;
            load(x, i + STEP);
            use(y);
            i += STEP;
            if (i >= t1) break;
        }
    }

    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (c == 0) {
        lm[wave][r16] = m;
        ll[wave][r16] = l;
    }
    {
        int n = 0;
#pragma unroll
        for (int st = 0; st < L::SETS; ++st)
#pragma unroll
            for (int e = 0; e < L::width(st); ++e, ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) lo[wave][L::base(st) + (4 * c + i) * L::width(st) + e][r16] = acc[n][i];
    }
}

}  // namespace attn
}  // namespace ckh
