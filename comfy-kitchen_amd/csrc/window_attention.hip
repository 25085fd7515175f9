// Causal attention of prompts with a sliding window and a few first tokens that stay visible
// (sinks), for gfx950.  Query i of a sequence stands at position p = i + keys - queries and sees
// key j if j <= p, j < lengths[b], and p - j < window or j < sinks:
//   out[b, i, h] = sum_j softmax_j(scale q[b, i, h] . k_j) v_j.
//
// Bound by the matrix units, and next to them by the softmax's exponentials (one a score, at a
// quarter of the rate of other instructions: about as many cycles as the score's MFMAs at
// head_dim 128).
//   - A row is a query and one of the query heads of a key-value head, the heads of a query next
//     to each other: a workgroup's rows then are few positions wide, so few tiles have masked
//     pairs, and a shared head's K and V are read once for its query heads.
//   - A wave owns 32 rows, which are the columns of 32x32x16 MFMAs (attn.h): running maximum and
//     sum are the lane's own, P stays in registers.  Tiles of keys go from memory to LDS without
//     passing registers, the next while this one is used; one barrier a tile.
//   - V is stored by token, its operand holds 4 + 4 tokens of one d: the transposing LDS read
//     delivers that (16 lanes give 4 tokens by 16 d).  16-byte pieces are placed so that neither
//     it nor K's reads meet on a bank.
//   - Tiles without a visible pair are not visited; only tiles with masked pairs pay for masks, and
//     only for the bounds that cut them (777 tokens of 24 heads, head_dim 64, window 256: 13.1 us,
//     16.8 with one test of the whole condition).
//     16384 tokens of 40 heads over 8, head_dim 128, window 4096: 1.18-1.34 ms (the clock varies),
//     0.9-1.03 PF, against 1.33 PF of a 16384^3 product.
//   - Where there are fewer workgroups than CUs, a workgroup's tiles are split over several, which
//     leave their fp32 sums to a second launch that joins them in order (2 x 3 queries of 40 heads
//     over 6000 keys: 28 us, 150 by one workgroup a block).
//   - A third buffer of tiles, the compiler's wait for the next tile before V is read taken away:
//     slower (4096 tokens, 16 heads: 152 us against 129).
//   - The maximum is only raised when a weight would pass 2^8 (in f16 2^15, attn.h), P is rounded to
//     the 16-bit type for the second product after its fp32 sum was taken.
//   - A masked pair's weight is zero, but zero times an infinity is not: if a result is not
//     finite, the workgroup runs again and keeps values that are not finite out of the
//     products of tiles with masked pairs, adding them to the rows that see them one by one.
#include <algorithm>
#include <type_traits>

#include "attn.h"

namespace ckh {
namespace attn {

typedef __attribute__((address_space(3))) void lds_void;
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s lds_v4s;

constexpr int kTileKeys = 64;

struct WindowArgs {
    const uint8_t *q, *k, *v;
    const int* lengths;  // null: all keys
    uint8_t* out;
    int64_t q_b, q_s, q_h, k_b, k_s, k_h, v_b, v_s, v_h;  // bytes
    int queries, keys, heads, kv_heads, group;
    int window, sinks;  // window INT32_MAX: none
    int row_blocks;     // blocks of rows of a key-value head
    int splits;         // workgroups that share a block's tiles
    float* part;        // their unnormalised outputs [splits][row][D], then maxima and sums [splits][row][2]
    int64_t all_rows;   // rows of the call
    float scale;
    FastDiv by_group;
};

// LDS rows are D (96: 128) values; 16-byte piece c of token t's row is at piece c ^ swizzle(t).
template <int D>
struct Rows {
    static constexpr int kPieces = D == 96 ? 16 : D / 8;
    static constexpr int kBytes = kPieces * 16;
    static constexpr int kMask = kPieces < 16 ? kPieces - 1 : 15;
    static __device__ __forceinline__ int k_swizzle(int t) { return t & 7; }
    static __device__ __forceinline__ int v_swizzle(int t) { return (2 * t) & kMask; }
};

// 16 bytes a lane from off (its own) to 16 consecutive bytes a lane from `to` (the wave's).
__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t rs, uint8_t* to, uint32_t off) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void*)to, 16, off, 0, 0, 0);
}

// W: waves (32 rows each) of a workgroup.
template <int C, int D, int W>
__global__ __launch_bounds__(W * 64, D == 256 ? 1 : 2) void window_kernel(WindowArgs a) {
    using R = Rows<D>;
    constexpr int kTile = kTileKeys * R::kBytes;          // bytes of a tile of K or V
    constexpr int kLoads = kTile / (W * 1024);    // 1 KB loads of a wave
    __shared__ __attribute__((aligned(1024))) uint8_t lds[4 * kTile];  // two buffers of K, V
    __shared__ int redo;

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r32 = lane & 31, g = lane >> 5;

    // the workgroups of one XCD take neighbouring blocks of rows, the longest first
    const int total = gridDim.x, x = blockIdx.x & 7;
    const int id = x * (total >> 3) + min(x, total & 7) + (blockIdx.x >> 3);
    const int bh = id / a.row_blocks, rb = a.row_blocks - 1 - (id - bh * a.row_blocks);
    const int b = bh / a.kv_heads, kvh = bh - b * a.kv_heads;

    const int rows = a.queries * a.group;
    const int row0 = (rb * W + wave) * 32;
    const int row = min(row0 + r32, rows - 1);
    const int qi = a.by_group.div(row), hq = kvh * a.group + row - qi * a.group;
    const int off = a.keys - a.queries;
    const int pos = qi + off;
    // positions of the wave's first and last row, of the workgroup's
    const int w_lo = static_cast<int>(a.by_group.div(min(row0, rows - 1))) + off;
    const int w_hi = static_cast<int>(a.by_group.div(min(row0 + 31, rows - 1))) + off;
    const int g_lo = static_cast<int>(a.by_group.div(rb * W * 32)) + off;
    const int g_hi = static_cast<int>(a.by_group.div(min((rb + 1) * W * 32, rows) - 1)) + off;
    const int len = a.lengths ? max(0, min(a.lengths[b], a.keys)) : a.keys;

    // visible tiles: the sinks' before the window's first
    const int key_end = min(g_hi + 1, len);
    const int win_from = max(0, g_lo - a.window + 1) / kTileKeys;
    const int win_to = (max(key_end, 0) + kTileKeys - 1) / kTileKeys;
    const int sink_tiles = min((min(a.sinks, max(key_end, 0)) + kTileKeys - 1) / kTileKeys, win_from);
    const int all = sink_tiles + max(0, win_to - win_from);
    const int tile0 = all * blockIdx.y / gridDim.y, tiles = all * (blockIdx.y + 1) / gridDim.y;  // this workgroup's

    float c = a.scale * kLog2e;
    const uint32_t flip = c < 0.0f ? 0x80008000u : 0u;
    c = fmaxf(fabsf(c), 1e-37f);
    v4u q[D / 16];
    {
        const uint8_t* qp = a.q + b * a.q_b + qi * a.q_s + hq * a.q_h + g * 16;
#pragma unroll
        for (int n = 0; n < D / 16; ++n) q[n] = *reinterpret_cast<const v4u*>(qp + n * 32) ^ flip;
    }

    // a lane's places in the loads of a tile: its token's row and piece
    uint32_t ko[kLoads], vo[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        const int at = (wave * kLoads + i) * 64 + lane;  // 16-byte piece of the tile
        const int t = at / R::kPieces, p = at % R::kPieces;
        const int kp = p ^ R::k_swizzle(t), vp = p ^ R::v_swizzle(t);
        ko[i] = kp < D / 8 ? t * static_cast<uint32_t>(a.k_s) + kp * 16 : 0x80000000u;
        vo[i] = vp < D / 8 ? t * static_cast<uint32_t>(a.v_s) + vp * 16 : 0x80000000u;
    }
    const uint8_t* kb = a.k + b * a.k_b + kvh * a.k_h;
    const uint8_t* vb = a.v + b * a.v_b + kvh * a.v_h;
    const auto key_of = [&](int i) { return (i < sink_tiles ? i : win_from + i - sink_tiles) * kTileKeys; };
    const auto stage = [&](int i, uint8_t* to) __attribute__((always_inline)) {  // keys past the sequence's end arrive as zeros
        const int k0 = key_of(i);
        const int64_t left = len - k0;
        const __amdgpu_buffer_rsrc_t rk = buffer_rsrc(kb + k0 * a.k_s, static_cast<uint32_t>(min(left * a.k_s, static_cast<int64_t>(0x7fffffff))));
        const __amdgpu_buffer_rsrc_t rv = buffer_rsrc(vb + k0 * a.v_s, static_cast<uint32_t>(min(left * a.v_s, static_cast<int64_t>(0x7fffffff))));
#pragma unroll
        for (int n = 0; n < kLoads; ++n)
            load_to_lds(rk, to + (wave * kLoads + n) * 1024, ko[n]);
#pragma unroll
        for (int n = 0; n < kLoads; ++n)
            load_to_lds(rv, to + kTile + (wave * kLoads + n) * 1024, vo[n]);
    };

    v16f acc[D / 32];
    float m, l;
    const auto use = [&](int i, const uint8_t* kt, const uint8_t* vt, auto careful_c) __attribute__((always_inline)) {
        constexpr bool careful = decltype(careful_c)::value;
        const int k0 = key_of(i);
        // no row of the wave sees the tile
        if (k0 > w_hi || k0 >= len || (k0 + kTileKeys - 1 < w_lo - a.window + 1 && k0 >= a.sinks)) return;
        v16f s[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int e = 0; e < 16; ++e) s[h][e] = 0.0f;
            const int t = h * 32 + r32;
            const uint8_t* kr = kt + t * R::kBytes;
#pragma unroll
            for (int n = 0; n < D / 16; ++n)
                s[h] = mfma32<C>(*reinterpret_cast<const v4u*>(kr + (((2 * n + g) ^ R::k_swizzle(t)) << 4)), q[n], s[h]);
        }
        const bool edge = k0 + kTileKeys - 1 > w_lo || k0 + kTileKeys > len ||
                          !(k0 > w_hi - a.window || k0 + kTileKeys <= a.sinks);
        if (edge) {
            // element e's key is at + its constant place: compared with the lane's bounds from there
            const int at = k0 + 4 * g;
            const int high = min(pos, len - 1) - at, low = pos - a.window + 1 - at, sink = a.sinks - at;
            if (k0 + kTileKeys - 1 > w_lo || k0 + kTileKeys > len) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int e = 0; e < 16; ++e) s[h][e] = h * 32 + 8 * (e >> 2) + (e & 3) <= high ? s[h][e] : -__builtin_inff();
            }
            if (k0 <= w_hi - a.window) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const int j = h * 32 + 8 * (e >> 2) + (e & 3);
                        s[h][e] = j >= low || j < sink ? s[h][e] : -__builtin_inff();
                    }
            }
        }
        float top = s[0][0];
#pragma unroll
        for (int e = 1; e < 16; ++e) top = fmaxf(top, s[0][e]);
#pragma unroll
        for (int e = 0; e < 16; ++e) top = fmaxf(top, s[1][e]);
        top *= c;
        if (__any(top > m + kLift<C> + 8.0f)) {
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            const float to = fmaxf(m, top - kLift<C>);
            const float f = exp2_hw(m - to);
            m = to;
            l *= f;
#pragma unroll
            for (int n = 0; n < D / 32; ++n) acc[n] *= f;
        }
        v4u p[4];
        float sum = 0.0f;  // the tile's own: single small weights would be lost in a large l
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                s[h][e] = exp2_hw(__fmaf_rn(s[h][e], c, -m));
                sum += s[h][e];
            }
        l += sum;
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                p[w][e] = pack2<C>(s[w >> 1][(w & 1) * 8 + 2 * e], s[w >> 1][(w & 1) * 8 + 2 * e + 1]);

        // tokens w * 16 + half * 8 + 4 g + 0..3: the lane gives a piece of one token and 4 d, and
        // gets one d of the four tokens
        const int sub = lane & 15, db = (lane >> 4) & 1;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
#pragma unroll
            for (int n = 0; n < D / 32; ++n) {
                v4u f;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int t = w * 16 + half * 8 + 4 * g + (sub >> 2);
                    const int piece = n * 4 + db * 2 + ((sub >> 1) & 1);
                    const uint8_t* at = vt + t * R::kBytes + ((piece ^ R::v_swizzle(t)) << 4) + (sub & 1) * 8;
                    const v4s got = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(at));
                    const v2u two = __builtin_bit_cast(v2u, got);
                    f[half * 2] = two[0];
                    f[half * 2 + 1] = two[1];
                }
                if constexpr (careful) if (edge) {  // values that are not finite become zeros here
                    constexpr uint32_t kExp = C == CKH_BF16 ? 0x7f80u : 0x7c00u;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if ((f[e] & kExp) == kExp) f[e] &= 0xffff0000u;
                        if (((f[e] >> 16) & kExp) == kExp) f[e] &= 0x0000ffffu;
                    }
                }
                acc[n] = mfma32<C>(f, p[w], acc[n]);
            }
        }
        if constexpr (careful) if (edge) {  // and reach the rows that see them here
            constexpr uint32_t kExp = C == CKH_BF16 ? 0x7f80u : 0x7c00u;
            for (int t = 0; t < kTileKeys; ++t) {
                const int j = k0 + t;
                const bool see = j <= pos && j < len && (pos - j < a.window || j < a.sinks);
                // the weight of token t: register 8 (t / 32 of s), element (t % 32 / 8) * 4 + t % 4, half (t / 4) % 2
                float w = 0.0f;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (t == h * 32 + 8 * (e >> 2) + 4 * ((t >> 2) & 1) + (e & 3)) w = s[h][e];
                w = __shfl(w, r32 + 32 * ((t >> 2) & 1), 64);
#pragma unroll
                for (int n = 0; n < D / 32; ++n)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const int d = n * 32 + 8 * (e >> 2) + 4 * g + (e & 3);
                        const uint32_t bits = *reinterpret_cast<const uint16_t*>(
                            vt + t * R::kBytes + (((d >> 3) ^ R::v_swizzle(t)) << 4) + (d & 7) * 2);
                        if (see && (bits & kExp) == kExp)
                            acc[n][e] += w * (C == CKH_BF16 ? bf16_to_f(bits) : f16_to_f(bits));
                    }
            }
        }
    };

    const auto run = [&](auto careful) __attribute__((always_inline)) {
        m = -1e30f;
        l = 0.0f;
#pragma unroll
        for (int n = 0; n < D / 32; ++n)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[n][e] = 0.0f;
        // (The buffers change hands as pointers: where the compiler sees which part of LDS a load
        // writes, it waits for the load before the next LDS read.)
        uint8_t *cur = lds, *next = lds + 2 * kTile;
        if (tile0 < tiles) stage(tile0, cur);
#pragma unroll 1
        for (int i = tile0; i < tiles; ++i) {
            __asm__ volatile("" ::: "memory");
            __builtin_amdgcn_s_waitcnt(0);  // this wave's part of tile i has arrived
            __builtin_amdgcn_s_barrier();   // everyone's has, and nobody reads the other buffer
            __asm__ volatile("" ::: "memory");
            if (i + 1 < tiles) stage(i + 1, next);
            use(i, cur, cur + kTile, careful);
            uint8_t* const t = cur;
            cur = next;
            next = t;
        }
        l += __shfl_xor(l, 32, 64);
    };
    if (threadIdx.x == 0) redo = 0;
    run(std::false_type{});
    bool odd = !(fabsf(l) < __builtin_inff());
#pragma unroll
    for (int n = 0; n < D / 32; ++n)
#pragma unroll
        for (int e = 0; e < 16; ++e) odd |= !(fabsf(acc[n][e]) < __builtin_inff());
    __syncthreads();
    if (odd) redo = 1;
    __syncthreads();
    if (redo) run(std::true_type{});

    if (row0 + r32 >= rows) return;
    const int64_t out_row = (static_cast<int64_t>(b) * a.queries + qi) * a.heads + hq;
    if (a.splits > 1) {
        const int64_t at = blockIdx.y * a.all_rows + out_row;
        float* op = a.part + at * D + g * 4;
#pragma unroll
        for (int n = 0; n < D / 32; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                *reinterpret_cast<v4f*>(op + n * 32 + e * 8) = v4f{acc[n][4 * e], acc[n][4 * e + 1], acc[n][4 * e + 2], acc[n][4 * e + 3]};
        float* ml = a.part + a.splits * a.all_rows * D + at * 2;
        if (g == 0) ml[0] = m, ml[1] = l;
        return;
    }
    const float f = l == 0.0f ? 0.0f : 1.0f / l;
    uint8_t* op = a.out + out_row * (D * 2) + g * 8;
#pragma unroll
    for (int n = 0; n < D / 32; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const v2u two = v2u{pack2<C>(acc[n][4 * e] * f, acc[n][4 * e + 1] * f), pack2<C>(acc[n][4 * e + 2] * f, acc[n][4 * e + 3] * f)};
            *reinterpret_cast<v2u*>(op + n * 64 + e * 16) = two;
        }
}

// Joins a row's splits: D / 4 lanes a row, four d a lane.
template <int C, int D>
__global__ __launch_bounds__(256) void window_join_kernel(WindowArgs a) {
    constexpr int kLanes = D / 4, kRows = 256 / kLanes;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / kLanes;
    if (threadIdx.x >= kRows * kLanes || row >= a.all_rows) return;
    const int d = threadIdx.x % kLanes * 4;
    const float* ml = a.part + a.splits * a.all_rows * D;
    float top = -1e30f, sum = 0.0f;
    for (int s = 0; s < a.splits; ++s) top = fmaxf(top, ml[(s * a.all_rows + row) * 2]);
    v4f o = v4f{0, 0, 0, 0};
#pragma unroll 4
    for (int s = 0; s < a.splits; ++s) {
        const int64_t at = s * a.all_rows + row;
        const float f = exp2_hw(ml[at * 2] - top);
        sum += f * ml[at * 2 + 1];
        o += f * *reinterpret_cast<const v4f*>(a.part + at * D + d);
    }
    const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
    *reinterpret_cast<v2u*>(a.out + (row * D + d) * 2) = v2u{pack2<C>(o[0] * f, o[1] * f), pack2<C>(o[2] * f, o[3] * f)};
}

// Waves of a workgroup: two where four would leave CUs without one (777 tokens of 24 heads over 8:
// 11.0 us against 13.2), else four (2048 tokens of 32 heads over 8: 44 against 61).
int window_waves(int64_t batch, int64_t queries, int64_t heads, int64_t kv_heads) {
    return batch * kv_heads * cdiv(queries * (heads / kv_heads), 128) < device_cus() ? 2 : 4;
}

// Workgroups that share a block's tiles: enough for two a CU, of four tiles at least.
int window_splits(int64_t batch, int64_t queries, int64_t keys, int64_t heads, int64_t kv_heads, int64_t window, int64_t sinks) {
    const int64_t group = heads / kv_heads, rows = 32 * window_waves(batch, queries, heads, kv_heads);
    const int64_t grid = batch * kv_heads * cdiv(queries * group, rows);
    const int64_t span = std::min(queries, cdiv(rows, group) + 1);  // positions of a workgroup's rows
    const int64_t seen = window > 0 ? std::min(keys, window + span + std::min(sinks, keys)) : keys;
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({32, 2 * device_cus() / grid, seen / (4 * kTileKeys)})));
}

template <int C, int D>
void launch_window(const WindowArgs& a, int64_t blocks, int waves, hipStream_t st) {
    const dim3 grid(static_cast<unsigned>(blocks), a.splits);
    if (waves == 2) window_kernel<C, D, 2><<<grid, 128, 0, st>>>(a);
    else window_kernel<C, D, 4><<<grid, 256, 0, st>>>(a);
    if (a.splits > 1) window_join_kernel<C, D><<<static_cast<unsigned>(cdiv(a.all_rows, 256 / (D / 4))), 256, 0, st>>>(a);
}

template <int C>
void launch_window(int dim, const WindowArgs& a, int64_t blocks, int waves, hipStream_t st) {
    if (dim == 64) launch_window<C, 64>(a, blocks, waves, st);
    else if (dim == 96) launch_window<C, 96>(a, blocks, waves, st);
    else if (dim == 128) launch_window<C, 128>(a, blocks, waves, st);
    else launch_window<C, 256>(a, blocks, waves, st);
}

}  // namespace attn
}  // namespace ckh

using namespace ckh;

extern "C" int64_t ckh_window_attention_workspace_bytes(int64_t batch, int64_t queries, int64_t keys, int64_t heads,
                                                        int64_t kv_heads, int64_t dim, int64_t window, int64_t sinks) {
    if (batch <= 0 || queries <= 0 || keys <= 0 || kv_heads <= 0 || heads < kv_heads || dim <= 0) return 0;
    const int64_t s = attn::window_splits(batch, queries, keys, heads, kv_heads, window, sinks);
    return s > 1 ? s * batch * queries * heads * (dim + 2) * 4 : 0;
}

extern "C" int ckh_window_attention(const void* q, const void* k, const void* v, const void* lengths, void* out,
                                    int64_t batch, int64_t queries, int64_t keys, int64_t heads, int64_t kv_heads,
                                    int64_t dim, const int64_t* strides, int64_t window, int64_t sinks, float scale,
                                    int code, void* workspace, int64_t workspace_bytes, uintptr_t stream) {
    CKH_REQUIRE(code == CKH_F16 || code == CKH_BF16, "window_attention: unsupported dtype %d", code);
    CKH_REQUIRE(dim == 64 || dim == 96 || dim == 128 || dim == 256, "window_attention: head_dim %lld is not 64, 96, 128 or 256",
                static_cast<long long>(dim));
    CKH_REQUIRE(batch >= 0 && heads >= 0 && kv_heads > 0 && heads % kv_heads == 0 && heads <= 65535,
                "window_attention: %lld heads over %lld key-value heads", static_cast<long long>(heads),
                static_cast<long long>(kv_heads));
    CKH_REQUIRE(queries >= 0 && keys >= 0 && queries <= (1 << 30) && keys <= (1 << 30) && queries * heads <= (1 << 30),
                "window_attention: %lld queries, %lld keys", static_cast<long long>(queries), static_cast<long long>(keys));
    CKH_REQUIRE(window >= 0 && sinks >= 0, "window_attention: window %lld, sinks %lld", static_cast<long long>(window),
                static_cast<long long>(sinks));
    if (batch == 0 || queries == 0 || heads == 0) return CKH_OK;
    CKH_REQUIRE(q && out && strides && (keys == 0 || (k && v)), "window_attention: null pointer");
    // q, k, v: batch, token, head each (elements)
    for (int i = 0; i < 9; ++i)
        CKH_REQUIRE(strides[i] >= 0 && strides[i] % 8 == 0, "window_attention: stride %d (%lld) is not a multiple of 16 bytes", i,
                    static_cast<long long>(strides[i]));
    CKH_REQUIRE((strides[4] >= dim && strides[7] >= dim) || keys <= 1, "window_attention: keys overlap");
    CKH_REQUIRE(strides[4] < (1 << 23) && strides[7] < (1 << 23), "window_attention: token stride too large");
    CKH_REQUIRE(aligned(q, 16) && aligned(k, 16) && aligned(v, 16) && aligned(out, 8) && aligned(lengths, 4),
                "window_attention: misaligned pointer");
    attn::WindowArgs a{};
    a.q = static_cast<const uint8_t*>(q), a.k = static_cast<const uint8_t*>(k), a.v = static_cast<const uint8_t*>(v);
    a.lengths = static_cast<const int*>(lengths);
    a.out = static_cast<uint8_t*>(out);
    a.q_b = strides[0] * 2, a.q_s = strides[1] * 2, a.q_h = strides[2] * 2;
    a.k_b = strides[3] * 2, a.k_s = std::max(strides[4], dim) * 2, a.k_h = strides[5] * 2;
    a.v_b = strides[6] * 2, a.v_s = std::max(strides[7], dim) * 2, a.v_h = strides[8] * 2;
    a.queries = static_cast<int>(queries), a.keys = static_cast<int>(keys);
    a.heads = static_cast<int>(heads), a.kv_heads = static_cast<int>(kv_heads), a.group = static_cast<int>(heads / kv_heads);
    a.window = window > 0 && window < (1 << 30) ? static_cast<int>(window) : (1 << 30);
    a.sinks = static_cast<int>(std::min<int64_t>(sinks, 1 << 30));
    const int waves = attn::window_waves(batch, queries, heads, kv_heads);
    a.row_blocks = static_cast<int>(cdiv(queries * a.group, waves * 32));
    a.scale = scale;
    a.by_group = fast_div(static_cast<uint32_t>(a.group));
    const int64_t grid = batch * kv_heads * a.row_blocks;
    CKH_REQUIRE(grid <= INT32_MAX, "window_attention: too many rows");
    const int64_t need = ckh_window_attention_workspace_bytes(batch, queries, keys, heads, kv_heads, dim, window, sinks);
    a.splits = need > 0 && workspace && workspace_bytes >= need && aligned(workspace, 16)
                   ? attn::window_splits(batch, queries, keys, heads, kv_heads, window, sinks) : 1;
    a.part = static_cast<float*>(workspace);
    a.all_rows = batch * queries * heads;
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (code == CKH_BF16) attn::launch_window<CKH_BF16>(static_cast<int>(dim), a, grid, waves, st);
    else attn::launch_window<CKH_F16>(static_cast<int>(dim), a, grid, waves, st);
    return check_launch("window_attention");
}
