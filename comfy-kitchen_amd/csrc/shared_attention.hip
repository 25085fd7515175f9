// Attention of one new token per sequence over a key-value cache held in pages, for sequences that begin
// with the same tokens, for gfx950:
//   out[b, h] = sum_t softmax_t(scale q[b, h] . k_t) v_t,  t < lengths[b],
// where the first shared[g] tokens of a group's sequences are the same rows of the cache.
//
// A span is a run of tokens that some sequences see: what a group shares, seen by all its sequences, and what
// lies behind it, seen by one.  Its rows are these sequences' query heads of a key-value head; so the common
// tokens are a matrix product of many rows, read once for each 128 of them, and bound by the matrix units
// from some 300 rows on, by HBM below.
//   - A small first launch (of a small call, every workgroup for itself) turns lengths and groups, which only the device
//     knows, into a list of pieces of work: a span's tokens in chunks of one size for the whole call, chosen so that there
//     are about two a CU, times its blocks of 128 rows and the key-value heads.
//   - The second works on one piece a workgroup.  Spans of up to 16 rows (a sequence's own tokens, mostly) are read
//     by the wave, each wave its own tiles, as ckh_paged_attention does (paged_tiles.h).  Wider ones go as prompts do:
//     a wave owns 32 rows, the columns of 32x32x16 MFMAs, with running maximum and sum; tiles of 64 tokens go to
//     LDS, the next while this one is used, each token's row found by its page, which is looked up a tile before.  A
//     16-bit cache goes there without passing registers; E4M3 codes are widened on the way, once for all rows.
//   - The third joins each row's chunks, those of its group and its own, in their order: results do not
//     depend on timing.
//
// Measured: 64 sequences of 40 heads on 8 over a common 16384 tokens and 1 .. 512 of their own, D 128, E4M3 pages: 4.5 +
// 48 + 8 us, 0.46 PF of the 22 GF (bf16 pages: 56 us in all); a tile's products, exponentials and LDS reads take a third of
// its time each, two workgroups a CU overlap them in part, and 480 pieces on 256 CUs leave some idle.  Six groups of 12
// sequences of 24 heads on 24 over 9001 and 700, D 64, f16: 4.5 + 86 + 5, 4.2 TB/s (rows of 128 bytes: ckh_paged_attention
// reads such a cache at the same rate).  Four sequences over 777 and 100: 11 + 4 us, nearly all of it steps that wait for
// each other.
// Against ckh_paged_attention over the same cache: 64 sequences over a common 32768 tokens in bf16, 73 us for 575;
// 16 over 8192, 27 for 52; 4 over 8192, 22 for 23; 4 over 2048, 16 for 15.  It pays from some 80 MB of keys and values that are not read again.
#include <algorithm>

#include "dispatch.h"
#include "paged_tiles.h"

namespace ckh {
namespace attn {

typedef __attribute__((address_space(3))) void lds_void;
typedef const __attribute__((address_space(1))) void global_void;
typedef const __attribute__((address_space(4))) int constant_int;
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s lds_v4s;

constexpr int kTileTokens = 64;
constexpr int kWideRows = 128;  // of a piece
constexpr int kThinRows = 16;
constexpr int kMinTiles = 2;    // of a chunk, where a span has several
constexpr int kMinThinTiles = 1;  // (4 sequences over 777 and 100, replayed: 16.7 us; of 4 and 2 tiles 19.7)
constexpr int kThinChunks = 8;  // of few rows, for one of many: they follow these and end the launch (64 sequences over a common 16384
                                // and 512 of their own in bf16: 56 us; 4: 68, 16: 58)
constexpr int kMaxSpans = 4096; // sequences and groups of a call

struct Span {
    int first, chunks;   // its first workgroup; chunks of each row
    int seq, sequences;  // the sequences that see it
    int from, to;        // tokens
    int group;           // of a sequence's own span: its group's span, or -1
    int size;            // tiles of a chunk
    int pieces;          // of work
    int pad;
    int64_t part;        // row of the partial results that chunk 0 of its first row has
};

struct SharedArgs {
    const uint8_t *q, *k, *v;
    const int *table, *lengths, *starts, *shared;
    const float *k_scale, *v_scale;
    uint8_t* out;
    Span* spans;  // [groups + batch]
    int* firsts;  // [groups + batch + 1]: their first workgroups, the workgroups of all
    float *part, *stat;  // [row][D], [row][2]: unnormalised outputs; maxima and sums
    int64_t q_b, q_h, k_page, k_tok, k_head, v_page, v_tok, v_head;  // bytes
    int64_t table_stride;
    int batch, heads, kv_heads, group, groups;  // group: query heads of a key-value head
    int pages, page_size, capacity, target;
    bool plans;  // shared_kernel makes the plan
    float scale;
    FastDiv by_page, by_group;
};

// Blocks of rows.  (16 rows by the wave: 16 groups of two sequences of 8 heads to a key-value head, D 128, bf16, 128 us and 158 by the
// workgroup's 128; one such group over 32768 tokens 43 and 36.)
__host__ __device__ __forceinline__ int64_t blocks_of(int64_t rows) {
    return rows <= kThinRows ? (rows > 0) : (rows + kWideRows - 1) / kWideRows;
}

template <int T>
__device__ __forceinline__ void plan_sync() {
    if constexpr (T > 64) __syncthreads();
    else __asm__ volatile("" ::: "memory");  // (one wave: LDS keeps its order)
}

// Inclusive sums over T threads; `total`: of all.
template <int T>
__device__ __forceinline__ void plan_scan(int64_t (&v)[2], int64_t (&total)[2], int64_t (*sums)[2]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1)
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const int64_t u = __shfl_up(static_cast<long long>(v[n]), d, 64);
            if (lane >= d) v[n] += u;
        }
    plan_sync<T>();
    if (lane == 63) sums[wave][0] = v[0], sums[wave][1] = v[1];
    plan_sync<T>();
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        total[n] = 0;
#pragma unroll
        for (int w = 0; w < T / 64; ++w) {
            if (w < wave) v[n] += sums[w][n];
            total[n] += sums[w][n];
        }
    }
}

template <int T>
struct PlanSpace {
    static constexpr int kSpans = T == 1024 ? kMaxSpans : T;
    int64_t sums[T / 64][2];
    int start[kSpans + 1], common[kSpans], top[T / 64];
};

// T threads (64: one wave, which needs no barriers) call put(i, span i), each for its own.  Returns the workgroups of all.
template <int T, typename Put>
__device__ __forceinline__ int64_t plan(const SharedArgs& a, PlanSpace<T>& space, Put put) {
    int *const start = space.start, *const common = space.common, *const top = space.top;
    auto& sums = space.sums;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int spans = a.groups + a.batch;
    const auto length = [&](int b) { return max(0, min(a.lengths[b], a.capacity)); };
    const int own_length = t < a.batch ? length(t) : 0;  // (the first T sequences': read ahead)

    for (int g = t; g < a.groups; g += T) common[g] = max(0, a.shared[g]);
    // group bounds, within the batch and ascending (whatever they are, groups do not overlap)
    int before = 0;
    for (int i0 = 0; i0 <= a.groups; i0 += T) {
        int v = i0 + t <= a.groups ? max(0, min(a.starts[i0 + t], a.batch)) : 0;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int u = __shfl_up(v, d, 64);
            if (lane >= d) v = max(v, u);
        }
        plan_sync<T>();
        if (lane == 63) top[wave] = v;
        plan_sync<T>();
        v = max(v, before);
        for (int w = 0; w < T / 64; ++w) {
            if (w < wave) v = max(v, top[w]);
            before = max(before, top[w]);
        }
        if (i0 + t <= a.groups) start[i0 + t] = v;
    }
    plan_sync<T>();
    const auto group_of = [&](int b) {  // the last group that begins at or before b, if b is in it
        int lo = 0, hi = a.groups;      // groups lo .. hi - 1
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (start[mid] <= b) lo = mid + 1;
            else hi = mid;
        }
        return lo > 0 && b < start[lo] ? lo - 1 : -1;
    };
    for (int b = t; b < a.batch; b += T) {
        const int g = group_of(b);
        if (g >= 0) atomicMin(&common[g], start[g + 1] - start[g] > 1 ? (b == t ? own_length : length(b)) : 0);
    }
    plan_sync<T>();

    const auto span = [&](int i) {
        Span s{};
        if (i < a.groups) {
            s.seq = start[i], s.sequences = start[i + 1] - start[i];
            s.to = s.sequences ? common[i] : 0;
            s.group = -1;
        } else {
            s.seq = i - a.groups, s.sequences = 1;
            s.group = group_of(s.seq);
            s.from = s.group < 0 ? 0 : common[s.group];
            s.to = length(s.seq);
        }
        return s;
    };
    // chunks begin at multiples of a tile
    const auto tiles_of = [&](const Span& s) { return s.to > s.from ? (s.to + kTileTokens - 1) / kTileTokens - s.from / kTileTokens : 0; };
    const auto rows_of = [&](const Span& s) { return static_cast<int64_t>(s.sequences) * a.group; };
    int64_t tiles = 0;
    Span held{};  // the thread's span, where there are no more than threads
    for (int i0 = 0; i0 < spans; i0 += T) {
        int64_t work[2] = {0, 0}, total[2];
        if (i0 + t < spans) {
            const Span s = span(i0 + t);
            if (i0 == 0) held = s;
            work[0] = tiles_of(s) * blocks_of(rows_of(s)) * a.kv_heads;
        }
        plan_scan<T>(work, total, sums);
        tiles += total[0];
    }
    // (no span has 2^26 tiles)
    const int64_t size = min(max((tiles + a.target - 1) / a.target, static_cast<int64_t>(kMinTiles)), static_cast<int64_t>(1) << 26);

    int64_t slot = 0, row = 0;
    for (int i0 = 0; i0 < spans; i0 += T) {
        int64_t n[2] = {0, 0}, total[2];  // pieces, rows of partial results
        Span s{};
        if (i0 + t < spans) {
            s = i0 == 0 ? held : span(i0 + t);
            // a workgroup works on one block of many rows, or on the few rows of kWaves chunks or heads
            const bool thin = rows_of(s) <= kThinRows;
            s.size = static_cast<int>(thin ? max((size + kThinChunks - 1) / kThinChunks, static_cast<int64_t>(kMinThinTiles)) : size);
            s.chunks = (tiles_of(s) + s.size - 1) / s.size;
            n[0] = s.chunks * blocks_of(rows_of(s)) * a.kv_heads;
            s.pieces = static_cast<int>(n[0]);
            if (thin) n[0] = (n[0] + kWaves - 1) / kWaves;
            n[1] = s.chunks * rows_of(s) * a.kv_heads;
        }
        int64_t end[2] = {n[0], n[1]};
        plan_scan<T>(end, total, sums);
        s.first = static_cast<int>(slot + end[0] - n[0]);
        s.part = row + end[1] - n[1];
        slot += total[0];
        row += total[1];
        if (i0 + t < spans) put(i0 + t, s);
    }
    return slot;
}

template <int T>
__global__ __launch_bounds__(T) void plan_kernel(SharedArgs a) {
    __shared__ PlanSpace<T> space;
    const int64_t slots = plan<T>(a, space, [&](int i, const Span& s) {
        a.firsts[i] = s.first;
        a.spans[i] = s;
    });
    if (threadIdx.x == 0) a.firsts[a.groups + a.batch] = static_cast<int>(slots);
}


// LDS rows are D (96: 128) values of 16 bits; 16-byte piece c of token t's row is at piece c ^ swizzle(t), so that the
// 16 lanes that read K at once (16 tokens' pieces), and the 32 that read V (4 tokens', 4 pieces of each), touch all 64 banks.
template <int D>
struct TileRows {
    static constexpr int kPieces = D == 96 ? 16 : D / 8;
    static constexpr int kBytes = kPieces * 16;
    static __device__ __forceinline__ int k_swizzle(int t) { return D == 64 ? (t >> 1) & 7 : t & 15; }
    static __device__ __forceinline__ int v_swizzle(int t) { return D == 64 ? (t & 2) * 2 : (t & 3) * 4; }
};

// What a workgroup, or a wave of one, works on.
struct Piece {
    int kv_head, row0, rows;  // its first row, the span's rows
    int from, to, seq;        // tokens; the span's first sequence
    int64_t part;             // of the span's row 0 in this chunk and head
    // The at-th of the span's: chunk by chunk, block of rows by block, and the heads of a token's rows side by side.
    __device__ __forceinline__ Piece(const SharedArgs& a, const Span& s, int at) {
        rows = s.sequences * a.group;
        const int blocks = static_cast<int>(blocks_of(rows)), in = at / a.kv_heads, chunk = in / blocks;
        const int64_t tile = s.from / kTileTokens + static_cast<int64_t>(chunk) * s.size;
        kv_head = at - in * a.kv_heads;
        row0 = (in - chunk * blocks) * kWideRows;
        from = static_cast<int>(max(static_cast<int64_t>(s.from), tile * kTileTokens));
        to = static_cast<int>(min(static_cast<int64_t>(s.to), (tile + s.size) * kTileTokens));
        seq = s.seq;
        part = s.part + (static_cast<int64_t>(chunk) * a.kv_heads + kv_head) * rows;
    }
};

// A wave, up to 16 rows: their tokens are read once, and what counts is loads in flight.
template <int C, int D, bool F8, bool WHOLE>
__device__ __forceinline__ void thin_piece(const SharedArgs& a, const Piece& p, uint8_t* lds) {
    using L = Lay<D, F8>;
    auto& lo = *reinterpret_cast<float(*)[kWaves][D][17]>(lds);
    auto& lm = *reinterpret_cast<float(*)[kWaves][16]>(lds + sizeof(lo));
    auto& ll = *reinterpret_cast<float(*)[kWaves][16]>(lds + sizeof(lo) + sizeof(lm));
    const int lane = threadIdx.x & 63, r16 = lane & 15, c = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    v4u q[D / 32];
    {
        const int row = min(r16, p.rows - 1), s = a.by_group.div(row);
        const uint8_t* qp = a.q + (p.seq + s) * a.q_b + (p.kv_head * a.group + row - s * a.group) * a.q_h;
#pragma unroll
        for (int n = 0; n < D / 32; ++n) {
            const int d = L::KW == 8 ? n * 32 + c * 8 : (n >> 1) * 64 + c * 16 + (n & 1) * 8;
            q[n] = *reinterpret_cast<const v4u*>(qp + d * 2);
        }
    }
    const float to_log2 = a.scale * kLog2e * (a.k_scale ? *a.k_scale : 1.0f);
    constexpr int ES = L::ES;
    const PagedRows rows{a.k + p.kv_head * a.k_head, a.v + p.kv_head * a.v_head, a.table + p.seq * a.table_stride,
                         a.k_page / ES, a.k_tok / ES, a.v_page / ES, a.v_tok / ES, a.pages, a.page_size, a.by_page};
    paged_tiles<C, D, F8, WHOLE, 1>(rows, PagedTiles{0, 0, p.from, p.to, 0, ((p.to + 31) >> 5) - (p.from >> 5)}, q, to_log2, lo, lm, ll);
    __asm__ volatile("" ::: "memory");  // (one wave: LDS keeps its order)
    for (int e = lane; e < p.rows * D; e += 64) a.part[p.part * D + e] = lo[wave][e % D][e / D];
    if (lane < p.rows) *reinterpret_cast<float2*>(a.stat + (p.part + lane) * 2) = make_float2(lm[wave][lane], ll[wave][lane]);
}

// A workgroup, up to 128 of more rows.  A wave fetches 16 tokens of a tile: with WHOLE they lie on one page, whose number
// and place are the wave's (scalar), and what is not to be seen is out of the buffer's bounds, which arrives as zeros;
// else every lane finds its tokens' places.
template <int C, int D, bool F8, bool WHOLE>
__device__ __forceinline__ void wide_piece(const SharedArgs& a, const Piece& piece, uint8_t* lds) {
    using R = TileRows<D>;
    constexpr int kTile = kTileTokens * R::kBytes;  // two buffers of K, V
    // loads of a lane for a tile of K or V: 16 bytes, of a row's kRow
    constexpr int kRow = F8 ? D / 16 : R::kPieces;
    constexpr int kLoads = (16 * kRow + 63) / 64;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r32 = lane & 31, g = lane >> 5;
    const int from = piece.from, to = piece.to, kvh = piece.kv_head, rows = piece.rows, seq = piece.seq;
    const int row0 = piece.row0 + wave * 32;
    const int first = from / kTileTokens * kTileTokens;  // of the first tile
    const int tiles = (to - first + kTileTokens - 1) / kTileTokens;
    const int* table = a.table + seq * a.table_stride;
    const bool busy = row0 < rows;  // this wave has rows

    float c = a.scale * kLog2e * (a.k_scale ? *a.k_scale : 1.0f);
    const uint32_t flip = c < 0.0f ? 0x80008000u : 0u;
    c = fmaxf(fabsf(c), 1e-37f);
    v4u q[D / 16];
    {
        const int row = min(row0 + r32, rows - 1), s = a.by_group.div(row);
        const uint8_t* qp = a.q + (seq + s) * a.q_b + (kvh * a.group + row - s * a.group) * a.q_h + g * 16;
#pragma unroll
        for (int n = 0; n < D / 16; ++n) q[n] = *reinterpret_cast<const v4u*>(qp + n * 32) ^ flip;
    }

    // a lane's load n of a tile: piece (n * 64 + lane) % kRow of the wave's token (n * 64 + lane) / kRow
    const auto tok = [&](int n) { return min((n * 64 + lane) / kRow, 15); };
    const auto col = [&](int n) { return (n * 64 + lane) % kRow; };
    const auto k_at = [&](int n) { return F8 ? col(n) : min(col(n) ^ R::k_swizzle(wave * 16 + tok(n)), D / 8 - 1); };
    const auto v_at = [&](int n) { return F8 ? col(n) : min(col(n) ^ R::v_swizzle(wave * 16 + tok(n)), D / 8 - 1); };
    const uint8_t* kb = a.k + kvh * a.k_head;
    const uint8_t* vb = a.v + kvh * a.v_head;
    // Whether any of the wave's tokens of tile i are to be seen.
    const auto some = [&](int i) { return first + i * kTileTokens + wave * 16 < to && first + i * kTileTokens + wave * 16 + 16 > from; };
    const auto token = [&](int i, int n) { return max(from, min(first + i * kTileTokens + wave * 16 + tok(n), to - 1)); };
    int page_of[WHOLE ? 1 : kLoads];  // of the next tile's tokens
    const auto look_up = [&](int i) __attribute__((always_inline)) {
        if constexpr (WHOLE) {
            // (a scalar load: a vector one would be waited for, and with it the fetches before it)
            page_of[0] = some(i) ? ((constant_int*)table)[a.by_page.div(first + i * kTileTokens + wave * 16)] : 0;
        } else {
#pragma unroll
            for (int n = 0; n < kLoads; ++n) page_of[n] = table[a.by_page.div(token(i, n))];
        }
    };
    v4u held[F8 ? 2 * kLoads : 1];  // codes on their way to LDS
    uint32_t ko[WHOLE ? kLoads : 1], vo[WHOLE ? kLoads : 1];
    if constexpr (WHOLE) {
#pragma unroll
        for (int n = 0; n < kLoads; ++n) {
            ko[n] = tok(n) * static_cast<uint32_t>(a.k_tok) + k_at(n) * 16;
            vo[n] = tok(n) * static_cast<uint32_t>(a.v_tok) + v_at(n) * 16;
        }
    }
    // Begins to fetch tile i.
    const auto fetch = [&](int i, uint8_t* at) __attribute__((always_inline)) {
        if constexpr (WHOLE) {
            const int t0 = first + i * kTileTokens + wave * 16, slot = t0 - a.by_page.div(t0) * a.page_size;
            const int64_t page = min(static_cast<uint32_t>(page_of[0]), static_cast<uint32_t>(a.pages - 1));
            const __amdgpu_buffer_rsrc_t rk = buffer_rsrc(kb + page * a.k_page + slot * a.k_tok, some(i) ? 0x7fffffffu : 0u);
            const __amdgpu_buffer_rsrc_t rv = buffer_rsrc(vb + page * a.v_page + slot * a.v_tok, some(i) ? 0x7fffffffu : 0u);
            const bool edge = first + i * kTileTokens < from || first + (i + 1) * kTileTokens > to;
#pragma unroll
            for (int n = 0; n < kLoads; ++n) {
                uint32_t kn = ko[n], vn = vo[n];
                if (edge && (t0 + tok(n) < from || t0 + tok(n) >= to)) kn = vn = kOut;
                if constexpr (F8) {
                    held[n] = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(rk, kn, 0, 0));
                    held[kLoads + n] = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(rv, vn, 0, 0));
                } else {
                    __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, (lds_void*)(at + (wave * kLoads + n) * 1024), 16, kn, 0, 0, 0);
                    __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, (lds_void*)(at + kTile + (wave * kLoads + n) * 1024), 16, vn, 0, 0, 0);
                }
            }
        } else {
#pragma unroll
            for (int n = 0; n < kLoads; ++n) {
                const int tk = token(i, n), slot = tk - a.by_page.div(tk) * a.page_size;
                const int64_t page = min(static_cast<uint32_t>(page_of[n]), static_cast<uint32_t>(a.pages - 1));
                const uint8_t* kp = kb + page * a.k_page + slot * a.k_tok + k_at(n) * 16;
                const uint8_t* vp = vb + page * a.v_page + slot * a.v_tok + v_at(n) * 16;
                if constexpr (F8) {
                    held[n] = *reinterpret_cast<const v4u*>(kp);
                    held[kLoads + n] = *reinterpret_cast<const v4u*>(vp);
                } else {
                    __builtin_amdgcn_global_load_lds((global_void*)kp, (lds_void*)(at + (wave * kLoads + n) * 1024), 16, 0, 0);
                    __builtin_amdgcn_global_load_lds((global_void*)vp, (lds_void*)(at + kTile + (wave * kLoads + n) * 1024), 16, 0, 0);
                }
            }
        }
    };
    // What of tile i the fetch does not bring to LDS at `at` by itself: widened codes; zeros for values that are not to be seen.
    const auto settle = [&](int i, uint8_t* at) __attribute__((always_inline)) {
        const int t0 = first + i * kTileTokens;
#pragma unroll
        for (int n = 0; n < kLoads; ++n) {
            const int t = wave * 16 + tok(n);
            const bool out = !WHOLE && (t0 + t < from || t0 + t >= to);
            if constexpr (F8) {
                if (16 * kRow % 64 != 0 && n * 64 + lane >= 16 * kRow) continue;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint32_t k0 = held[n][2 * half], k1 = held[n][2 * half + 1];
                    uint32_t v0 = held[kLoads + n][2 * half], v1 = held[kLoads + n][2 * half + 1];
                    if (out) v0 = v1 = 0u;
                    const int piece = 2 * col(n) + half;
                    *reinterpret_cast<v4u*>(at + t * R::kBytes + ((piece ^ R::k_swizzle(t)) << 4)) =
                        v4u{widen_e4m3<C, false>(k0), widen_e4m3<C, true>(k0), widen_e4m3<C, false>(k1), widen_e4m3<C, true>(k1)};
                    *reinterpret_cast<v4u*>(at + kTile + t * R::kBytes + ((piece ^ R::v_swizzle(t)) << 4)) =
                        v4u{widen_e4m3<C, false>(v0), widen_e4m3<C, true>(v0), widen_e4m3<C, false>(v1), widen_e4m3<C, true>(v1)};
                }
            } else if (out) {
                *reinterpret_cast<v4u*>(at + kTile + (wave * kLoads + n) * 1024 + lane * 16) = v4u{0u, 0u, 0u, 0u};
            }
        }
    };

    v16f acc[D / 32];
#pragma unroll
    for (int n = 0; n < D / 32; ++n)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[n][e] = 0.0f;
    float m = -1e30f, l = 0.0f;

    const auto use = [&](int i, const uint8_t* kt, const uint8_t* vt) __attribute__((always_inline)) {
        // (the two halves in turn: a product that adds to the one before it waits for it)
        v16f s[2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int e = 0; e < 16; ++e) s[h][e] = 0.0f;
#pragma unroll
        for (int n = 0; n < D / 16; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int t = h * 32 + r32;
                const uint8_t* kr = kt + t * R::kBytes;
                s[h] = mfma32<C>(*reinterpret_cast<const v4u*>(kr + (((2 * n + g) ^ R::k_swizzle(t)) << 4)), q[n], s[h]);
            }
        // two steps' keys are read ahead of the products (left to the compiler: 64 spans of 16 rows over a prefix of 4096, 46.3 us instead of 44.8)
        __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);  // LDS reads
#pragma unroll
        for (int n = 0; n < D / 16; ++n) {
            __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);  // products
            __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        }
        const int t0 = first + i * kTileTokens;
        if (t0 < from || t0 + kTileTokens > to) {
            const int low = from - t0 - 4 * g, high = to - t0 - 4 * g;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int j = h * 32 + 8 * (e >> 2) + (e & 3);
                    s[h][e] = j >= low && j < high ? s[h][e] : -__builtin_inff();
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
            const float high = fmaxf(m, top - kLift<C>);
            const float f = exp2_hw(m - high);
            m = high;
            l *= f;
#pragma unroll
            for (int n = 0; n < D / 32; ++n) acc[n] *= f;
        }
        // The weights of 16 tokens are made while the matrix units multiply those of the 16 before with their values.  They are
        // rounded to the values' 16-bit type, as the product takes them and as ckh_paged_attention does; their sum is taken before that.
        float sum = 0.0f;  // the tile's own: single small weights would be lost in a large l
        const auto weigh = [&](int w) __attribute__((always_inline)) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] = exp2_hw(__fmaf_rn(s[w >> 1][(w & 1) * 8 + e], c, -m));
                sum += x[e];
            }
            return v4u{pack2<C>(x[0], x[1]), pack2<C>(x[2], x[3]), pack2<C>(x[4], x[5]), pack2<C>(x[6], x[7])};
        };
        // tokens w * 16 + half * 8 + 4 g + 0..3: the lane gives a piece of one token and 4 d, and
        // gets one d of the four tokens
        const int sub = lane & 15, db = (lane >> 4) & 1;
        const auto values = [&](int w, v4u (&f)[D / 32]) __attribute__((always_inline)) {
#pragma unroll
            for (int n = 0; n < D / 32; ++n)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int t = w * 16 + half * 8 + 4 * g + (sub >> 2);
                    const int piece = n * 4 + db * 2 + ((sub >> 1) & 1);
                    const uint8_t* at = vt + t * R::kBytes + ((piece ^ R::v_swizzle(t)) << 4) + (sub & 1) * 8;
                    const v2u two = __builtin_bit_cast(v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(at)));
                    f[n][half * 2] = two[0];
                    f[n][half * 2 + 1] = two[1];
                }
        };
        v4u f[D / 32], p = weigh(0);
        values(0, f);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            v4u next = p;
            if (w < 3) next = weigh(w + 1);
#pragma unroll
            for (int n = 0; n < D / 32; ++n) acc[n] = mfma32<C>(f[n], p, acc[n]);
            if (w < 3) values(w + 1, f);
            p = next;
        }
        l += sum;
    };

    // (The buffers change hands as pointers: where the compiler sees which part of LDS a load
    // writes, it waits for the load before the next LDS read.)
    uint8_t *cur = lds, *next = lds + 2 * kTile;
    look_up(0);
    fetch(0, cur);
    if (tiles > 1) look_up(1);
    if constexpr (F8) settle(0, cur);
#pragma unroll 1
    for (int i = 0; i < tiles; ++i) {
        __asm__ volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0);  // this wave's part of tile i has arrived
        if constexpr (!F8 && !WHOLE) {
            if (i == 0 || i + 1 == tiles) {
                __asm__ volatile("" ::: "memory");
                settle(i, cur);
                __asm__ volatile("" ::: "memory");
                __builtin_amdgcn_s_waitcnt(0);
            }
        }
        __builtin_amdgcn_s_barrier();   // everyone's has, and nobody reads the other buffer
        __asm__ volatile("" ::: "memory");
        if (i + 1 < tiles) {
            fetch(i + 1, next);
            if (i + 2 < tiles) look_up(i + 2);
        }
        if (busy) use(i, cur, cur + kTile);
        if constexpr (F8) {
            if (i + 1 < tiles) settle(i + 1, next);
        }
        uint8_t* const t = cur;
        cur = next;
        next = t;
    }
    l += __shfl_xor(l, 32, 64);

    if (row0 + r32 >= rows) return;
    const int64_t at = piece.part + row0 + r32;
    float* op = a.part + at * D + g * 4;
#pragma unroll
    for (int n = 0; n < D / 32; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            *reinterpret_cast<v4f*>(op + n * 32 + e * 8) = v4f{acc[n][4 * e], acc[n][4 * e + 1], acc[n][4 * e + 2], acc[n][4 * e + 3]};
    if (g == 0) *reinterpret_cast<float2*>(a.stat + at * 2) = make_float2(m, l);
}

template <int C, int D, bool F8, bool WHOLE>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void shared_kernel(SharedArgs a) {
    constexpr int kLds = std::max<int>(4 * kTileTokens * TileRows<D>::kBytes, kWaves * (D * 17 + 32) * 4);
    __shared__ __attribute__((aligned(1024))) uint8_t lds[kLds];
    // the span of this workgroup: the last that begins at or before it
    const int spans = a.groups + a.batch, id = blockIdx.x;
    Span s;
    if (a.plans) {  // no launch before this one: each workgroup makes the plan for itself, the first also for the join
        auto& space = *reinterpret_cast<PlanSpace<64>*>(lds);
        Span& found = *reinterpret_cast<Span*>(lds + 2048);
        int& all = *reinterpret_cast<int*>(lds + 2048 + sizeof(Span));
        static_assert(sizeof(PlanSpace<64>) <= 2048 && 2048 + sizeof(Span) + 4 <= kLds, "both fit");
        if (threadIdx.x < 64) {
            Span mine{};
            const int64_t slots = plan<64>(a, space, [&](int i, const Span& x) {
                mine = x;
                if (id == 0) a.spans[i] = x;
            });
            const int lane = threadIdx.x;
            const uint64_t here = __ballot(lane < spans && mine.first <= id);
            if (lane == __popcll(here) - 1) found = mine;
            if (lane == 0) all = static_cast<int>(slots);
        }
        __syncthreads();
        if (id >= all) return;
        s = found;
        int* const w = reinterpret_cast<int*>(&s);
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(Span) / 4); ++i) w[i] = __builtin_amdgcn_readfirstlane(w[i]);
        __syncthreads();
    } else {
        if (id >= a.firsts[spans]) return;
        int before = 0;
        for (int i0 = 0; i0 < spans; i0 += 64) {
            const int i = i0 + static_cast<int>(threadIdx.x & 63);
            const uint64_t here = __ballot(i < spans && a.firsts[i] <= id);
            before += __popcll(here);
            if (here != ~0ull) break;
        }
        s = a.spans[__builtin_amdgcn_readfirstlane(before) - 1];
    }
    if (s.sequences * a.group <= kThinRows) {
        const int at = (id - s.first) * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        if (at < s.pieces) thin_piece<C, D, F8, WHOLE>(a, Piece(a, s, at), lds);
    } else {
        wide_piece<C, D, F8, WHOLE>(a, Piece(a, s, id - s.first), lds);
    }
}

// A row by W waves: its chunks' maxima and sums first, 64 a wave at a time, then four d a lane of as many chunks at once as
// lanes allow.
template <int C, int D, int W>
__global__ __launch_bounds__(256) void shared_join_kernel(SharedArgs a) {
    constexpr int kLanes = D / 4, kSets = 64 / kLanes;  // lanes of a chunk's row; chunks at once
    __shared__ __attribute__((aligned(16))) float outs[W > 1 ? W : 1][D];
    __shared__ float tops[W], sums[W];
    const int wave = W > 1 ? threadIdx.x >> 6 : 0;
    const int64_t row = W > 1 ? blockIdx.x : static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (row >= static_cast<int64_t>(a.batch) * a.heads) return;
    const int lane = threadIdx.x & 63, set = lane / kLanes, d = (lane - set * kLanes) * 4;
    const int b = static_cast<int>(row / a.heads), h = static_cast<int>(row - static_cast<int64_t>(b) * a.heads);
    const int kvh = h / a.group, in = h - kvh * a.group;
    const Span own = a.spans[a.groups + b];
    const Span group = own.group >= 0 ? a.spans[own.group] : Span{};
    // chunk i of the group's, then of the sequence's own: its row of the partial results
    const int64_t group_step = static_cast<int64_t>(a.kv_heads) * group.sequences * a.group, own_step = static_cast<int64_t>(a.kv_heads) * a.group;
    const int64_t group_at = group.part + (static_cast<int64_t>(kvh) * group.sequences + (b - group.seq)) * a.group + in;
    const int64_t own_at = own.part + static_cast<int64_t>(kvh) * a.group + in;
    const int chunks = group.chunks + own.chunks;
    const auto place = [&](int i) { return i < group.chunks ? group_at + i * group_step : own_at + (i - group.chunks) * own_step; };

    float top = -1e30f, sum = 0.0f;
    v4f o = v4f{0, 0, 0, 0};
    for (int i0 = wave * 64; i0 < chunks; i0 += W * 64) {
        const int i = i0 + lane;
        float2 st = make_float2(-1e30f, 0.0f);
        if (i < chunks) st = *reinterpret_cast<const float2*>(a.stat + place(i) * 2);
        float high = st.x;
#pragma unroll
        for (int s = 32; s >= 1; s >>= 1) high = fmaxf(high, __shfl_xor(high, s, 64));
        high = fmaxf(high, top);
        const float f = exp2_hw(st.x - high), old = exp2_hw(top - high);
        top = high;
        float part = f * st.y;
#pragma unroll
        for (int s = 32; s >= 1; s >>= 1) part += __shfl_xor(part, s, 64);
        sum = sum * old + part;
        o *= old;
        const int n = min(64, chunks - i0);
        constexpr int U = 8;  // loads of a lane in flight
        for (int j0 = 0; j0 < n; j0 += U * kSets) {
            v4f x[U];
            float g[U];
#pragma unroll
            for (int e = 0; e < U; ++e) {  // past the last chunk (and in lanes without a set): the last one again, with no weight
                const int j = j0 + e * kSets + set;
                const bool live = set < kSets && j < n;
                x[e] = *reinterpret_cast<const v4f*>(a.part + place(i0 + min(j, n - 1)) * D + d);
                g[e] = __shfl(f, live ? j : 0, 64);
                g[e] = live ? g[e] : 0.0f;
            }
#pragma unroll
            for (int e = 0; e < U; ++e) o += g[e] != 0.0f ? g[e] * x[e] : v4f{0, 0, 0, 0};
        }
    }
    // the sets' sums, in order
    v4f all = o;
#pragma unroll
    for (int n = 1; n < kSets; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) all[e] += __shfl(o[e], lane + n * kLanes, 64);
    if constexpr (W > 1) {
        if (set == 0) *reinterpret_cast<v4f*>(&outs[wave][d]) = all;
        if (lane == 0) tops[wave] = top, sums[wave] = sum;
        __syncthreads();
        if (wave != 0) return;
        all = v4f{0, 0, 0, 0};
        sum = 0.0f;
        for (int w = 0; w < W; ++w) top = fmaxf(top, tops[w]);
        for (int w = 0; w < W; ++w) {
            const float g = exp2_hw(tops[w] - top);
            sum += g * sums[w];
            if (set == 0 && g != 0.0f) all += g * *reinterpret_cast<const v4f*>(&outs[w][d]);
        }
    }
    if (set != 0) return;
    const float f = sum == 0.0f ? 0.0f : (a.v_scale ? *a.v_scale : 1.0f) / sum;
    *reinterpret_cast<v2u*>(a.out + (row * D + d) * 2) = v2u{pack2<C>(all[0] * f, all[1] * f), pack2<C>(all[2] * f, all[3] * f)};
}

template <int C, int D>
void launch_shared(const SharedArgs& a, int64_t slots, bool f8, hipStream_t st) {
    // A span a thread, and barriers only where there are several waves (5 spans: 3.8 us by one wave, 4.8 by sixteen).
    if (a.plans) {
    } else if (a.batch + a.groups <= kOneWaveSpans) plan_kernel<64><<<1, 64, 0, st>>>(a);
    else if (a.batch + a.groups <= 128) plan_kernel<128><<<1, 128, 0, st>>>(a);
    else if (a.batch + a.groups <= 256) plan_kernel<256><<<1, 256, 0, st>>>(a);
    else plan_kernel<1024><<<1, 1024, 0, st>>>(a);
    // 16 tokens lie on one page (64 sequences over a common 16384 in bf16, pages of 64: 53 us; of 72: 59).
    const bool whole = a.page_size % 16 == 0;
    const unsigned grid = static_cast<unsigned>(slots);
    if (f8 && whole) shared_kernel<C, D, true, true><<<grid, 256, 0, st>>>(a);
    else if (f8) shared_kernel<C, D, true, false><<<grid, 256, 0, st>>>(a);
    else if (whole) shared_kernel<C, D, false, true><<<grid, 256, 0, st>>>(a);
    else shared_kernel<C, D, false, false><<<grid, 256, 0, st>>>(a);
    const int64_t rows = static_cast<int64_t>(a.batch) * a.heads;
    // Few rows have many chunks (2 sequences over 32768 tokens, 80 rows of some 128 chunks: 15 us by a wave a row, 7.5 by four).
    if (rows <= 4 * device_cus()) shared_join_kernel<C, D, 4><<<static_cast<unsigned>(rows), 256, 0, st>>>(a);
    else shared_join_kernel<C, D, 1><<<static_cast<unsigned>(cdiv(rows, 4)), 256, 0, st>>>(a);
}

template <int C>
void launch_shared(int dim, const SharedArgs& a, int64_t slots, bool f8, hipStream_t st) {
    if (dim == 64) launch_shared<C, 64>(a, slots, f8, st);
    else if (dim == 96) launch_shared<C, 96>(a, slots, f8, st);
    else if (dim == 128) launch_shared<C, 128>(a, slots, f8, st);
    else launch_shared<C, 256>(a, slots, f8, st);
}

// Places in the workspace.
struct SharedSpace {
    int64_t target, slots, rows, firsts, part, stat, bytes;  // slots: pieces of work at most; rows: of partial results
    SharedSpace(int64_t batch, int64_t heads, int64_t kv_heads, int64_t dim, int64_t groups, int64_t capacity) {
        const int64_t group = heads / kv_heads, all = batch * group;  // rows of a key-value head
        const int64_t tiles = cdiv(capacity, kTileTokens);            // of a span
        target = 2 * device_cus();  // (64 over 16384 and 512, bf16: 56 us; one a CU 64, three 63)
        // workgroups for a chunk of every span (one more where they share it out), and `target` for those that have several: the
        // plan's chunks are at least tiles / target long, those of few rows, one a wave, a part of that
        slots = std::max(1, kThinChunks / kWaves) * target + kv_heads * (batch * blocks_of(group) + groups + all / kWideRows) + 2 * (batch + groups);
        rows = target * std::max(std::min<int64_t>(kWideRows, all), kThinChunks * std::min<int64_t>(kThinRows, all)) + 2 * kv_heads * all;
        // nor are there more chunks than tiles
        const int64_t own = group <= kThinRows ? cdiv(tiles * kv_heads, kWaves) : tiles * kv_heads * blocks_of(group);
        slots = std::max<int64_t>(std::min(slots, batch * own + tiles * kv_heads * (groups + all / kWideRows)), 1);
        rows = std::min(rows, 2 * kv_heads * all * tiles);
        firsts = rup((batch + groups) * sizeof(Span), 256);
        part = firsts + rup((batch + groups + 1) * 4, 256);
        stat = part + rup(rows * dim * 4, 256);
        bytes = stat + rows * 8;
    }
};

}  // namespace attn
}  // namespace ckh

using namespace ckh;

extern "C" int64_t ckh_shared_attention_workspace_bytes(int64_t batch, int64_t heads, int64_t kv_heads, int64_t dim, int64_t groups,
                                                        int64_t page_size, int64_t max_pages) {
    if (batch <= 0 || kv_heads <= 0 || heads < kv_heads || dim <= 0 || groups < 0 || page_size <= 0 || max_pages < 0) return 0;
    return attn::SharedSpace(batch, heads, kv_heads, dim, groups, max_pages * page_size).bytes;
}

extern "C" int ckh_shared_attention(const void* q, const void* k_cache, const void* v_cache, const void* page_table,
                                    const void* lengths, const void* group_starts, const void* shared, const void* k_scale,
                                    const void* v_scale, void* out, int64_t batch, int64_t heads, int64_t kv_heads, int64_t dim,
                                    int64_t groups, int64_t pages, int64_t page_size, int64_t max_pages, int64_t table_stride,
                                    const int64_t* strides, float scale, int q_code, int cache_code, void* workspace,
                                    int64_t workspace_bytes, uintptr_t stream) {
    CKH_REQUIRE(q_code == CKH_F16 || q_code == CKH_BF16, "shared_attention: unsupported query dtype %d", q_code);
    CKH_REQUIRE(cache_code == q_code || cache_code == CKH_E4M3, "shared_attention: cache dtype %d with query dtype %d",
                cache_code, q_code);
    CKH_REQUIRE(dim == 64 || dim == 96 || dim == 128 || dim == 256, "shared_attention: head_dim %lld is not 64, 96, 128 or 256",
                static_cast<long long>(dim));
    CKH_REQUIRE(batch >= 0 && heads >= 0 && kv_heads > 0 && heads % kv_heads == 0 && heads <= 65535,
                "shared_attention: %lld heads over %lld key-value heads", static_cast<long long>(heads),
                static_cast<long long>(kv_heads));
    CKH_REQUIRE(groups >= 0 && batch + groups <= attn::kMaxSpans, "shared_attention: %lld sequences in %lld groups (%d together at most)",
                static_cast<long long>(batch), static_cast<long long>(groups), attn::kMaxSpans);
    CKH_REQUIRE(pages > 0 && pages <= INT32_MAX && page_size > 0 && max_pages >= 0 && page_size <= INT32_MAX &&
                    max_pages <= INT32_MAX && max_pages * page_size <= INT32_MAX - 64,
                "shared_attention: %lld pages of %lld tokens, %lld a sequence", static_cast<long long>(pages),
                static_cast<long long>(page_size), static_cast<long long>(max_pages));
    if (batch == 0 || heads == 0) return CKH_OK;
    CKH_REQUIRE(q && k_cache && v_cache && (page_table || max_pages == 0) && lengths && group_starts && (shared || groups == 0) && out &&
                    strides && workspace,
                "shared_attention: null pointer");
    const int es = cache_code == CKH_E4M3 ? 1 : 2;
    // q: batch, head; k: page, token, head; v: page, token, head (elements)
    for (int i = 0; i < 8; ++i)
        CKH_REQUIRE(strides[i] >= 0 && strides[i] * (i < 2 ? 2 : es) % 16 == 0, "shared_attention: stride %d (%lld) is not a multiple of 16 bytes",
                    i, static_cast<long long>(strides[i]));
    CKH_REQUIRE(strides[3] * es < (int64_t(1) << 25) && strides[6] * es < (int64_t(1) << 25), "shared_attention: token stride too large");
    CKH_REQUIRE(aligned(q, 16) && aligned(k_cache, 16) && aligned(v_cache, 16) && aligned(out, 8) && aligned(page_table, 4) &&
                    aligned(lengths, 4) && aligned(group_starts, 4) && aligned(shared, 4) && aligned(k_scale, 4) && aligned(v_scale, 4) &&
                    aligned(workspace, 16),
                "shared_attention: misaligned pointer");
    const attn::SharedSpace space(batch, heads, kv_heads, dim, groups, max_pages * page_size);
    CKH_REQUIRE(space.slots <= (1 << 24), "shared_attention: too many heads and sequences");
    CKH_REQUIRE(workspace_bytes >= space.bytes, "shared_attention: a workspace of %lld bytes, needs %lld",
                static_cast<long long>(workspace_bytes), static_cast<long long>(space.bytes));
    attn::SharedArgs a{};
    a.q = static_cast<const uint8_t*>(q);
    a.k = static_cast<const uint8_t*>(k_cache), a.v = static_cast<const uint8_t*>(v_cache);
    a.table = static_cast<const int*>(page_table), a.lengths = static_cast<const int*>(lengths);
    a.starts = static_cast<const int*>(group_starts), a.shared = static_cast<const int*>(shared);
    a.k_scale = static_cast<const float*>(k_scale), a.v_scale = static_cast<const float*>(v_scale);
    a.out = static_cast<uint8_t*>(out);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    a.spans = reinterpret_cast<attn::Span*>(ws);
    a.firsts = reinterpret_cast<int*>(ws + space.firsts);
    a.part = reinterpret_cast<float*>(ws + space.part);
    a.stat = reinterpret_cast<float*>(ws + space.stat);
    a.q_b = strides[0] * 2, a.q_h = strides[1] * 2;
    a.k_page = strides[2] * es, a.k_tok = strides[3] * es, a.k_head = strides[4] * es;
    a.v_page = strides[5] * es, a.v_tok = strides[6] * es, a.v_head = strides[7] * es;
    a.table_stride = table_stride;
    a.batch = static_cast<int>(batch), a.heads = static_cast<int>(heads), a.kv_heads = static_cast<int>(kv_heads);
    a.group = static_cast<int>(heads / kv_heads), a.groups = static_cast<int>(groups);
    a.pages = static_cast<int>(pages), a.page_size = static_cast<int>(page_size);
    a.capacity = static_cast<int>(max_pages * page_size);
    a.target = static_cast<int>(space.target);
    a.scale = scale;
    a.by_page = fast_div(static_cast<uint32_t>(page_size)), a.by_group = fast_div(static_cast<uint32_t>(a.group));
    a.plans = shared_plans_itself(batch + groups, space.slots, static_cast<int>(dim), device_cus());
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (q_code == CKH_BF16) attn::launch_shared<CKH_BF16>(static_cast<int>(dim), a, space.slots, es == 1, st);
    else attn::launch_shared<CKH_F16>(static_cast<int>(dim), a, space.slots, es == 1, st);
    return check_launch("shared_attention");
}
