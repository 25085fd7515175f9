// Attention of one new token per sequence over a key-value cache held in pages, for gfx950:
//   out[b, h] = sum_t softmax_t(scale q[b, h] . k_t) v_t
// over the tokens t of sequence b that are visible: all of its lengths[b] tokens, or with a window
// its last `window` tokens and its first `sinks`.  Token t is row t % page_size of page
// table[b][t / page_size].
//
// The call is bound by reading K and V once (with 8 query heads to a key-value head it does 8
// flops a byte), so everything serves loads in flight:
//   - A wave takes tiles of 32 tokens and needs no other wave until its end: the running maximum
//     and sum of its softmax are its own, and so is its output, merged once in LDS.
//   - K and V go straight to registers, the next tile's while this one is computed.  The query
//     heads of a key-value head are the columns of 16x16x32 MFMAs (attn.h), so a shared
//     head's K and V are read once for all of them.
//   - V's operand holds 8 tokens of one d in a lane, memory 8 d of one token: a lane loads whole
//     runs of d for its 8 tokens (16 lanes a token row, whole lines) and transposes them in
//     its registers, one permute for two values; which tokens and which d a lane holds is free,
//     since P's layout fixes the tokens and the output's rows may be any order of d.
//   - The visible tiles of all sequences and key-value heads are dealt out in chunks of one size,
//     found on the device from the lengths (they are not known on the host), so sequences of
//     unlike lengths load the chip evenly and one long sequence fills it.  A sequence in several
//     chunks leaves fp32 partial results, which a second small launch joins in chunk order:
//     results do not depend on timing.
//   - Measured: 80003 tokens of 30 heads, f16 (1.23 GB): 211-220 us by card, 5.6-5.8 TB/s; 48
//     sequences of 8192 tokens and fewer, 8 heads, bf16 (823 MB): 168 us, 4.9 TB/s; the same as E4M3
//     (412 MB): 107 us, 3.9 TB/s, for its rows are 128 bytes; 333 tokens: 7.3-8.2 us, loads that
//     wait for each other.
//   - The maximum is only raised when a weight would pass 2^8 (in f16 2^15, attn.h): that costs
//     fp32 sums nothing and saves most rescaling.  P is rounded to the 16-bit type for the
//     second product, as its other operand is; its sum is taken before that.
#include <algorithm>

#include "paged_tiles.h"

namespace ckh {
namespace attn {

constexpr int kMaxChunks = 1024;  // of a unit: the join's factors are in LDS

struct PagedArgs {
    const uint8_t *q, *k, *v;
    const int* table;
    const int* lengths;
    const float *k_scale, *v_scale;  // null: 1
    void* out;
    float* part;  // [chunk][16][D + 2]: unnormalised output, maximum, sum
    int2* plan;   // [unit]: its first chunk, its chunks (null: one each)
    int64_t q_b, q_h, k_page, k_tok, k_head, v_page, v_tok, v_head;  // strides in elements
    int64_t table_stride;
    int batch, heads, kv_heads, group, head_tiles;  // group: query heads of a key-value head
    int pages, page_size, max_pages, window, sinks;
    int target;     // chunks wanted, at most kMaxChunks, which no unit then passes; 1: no splitting
    int min_tiles;  // least tiles of a chunk, where a unit has several
    float scale;
    FastDiv by_page;
};

// The visible tokens of a sequence as tiles of 32: those of the sinks, then those of the window.
struct Visible {
    int len, start, sink_end, sink_tiles, tiles;
    __device__ __forceinline__ Visible(const PagedArgs& a, int length) {
        len = static_cast<int>(min(static_cast<int64_t>(max(length, 0)), static_cast<int64_t>(a.max_pages) * a.page_size));
        start = a.window > 0 ? max(0, len - a.window) : 0;
        sink_end = min(a.sinks, start);
        sink_tiles = (sink_end + 31) >> 5;
        tiles = sink_tiles + ((len + 31) >> 5) - (start >> 5);
    }
};

__device__ __forceinline__ int wave_scan(int v, int lane) {  // inclusive
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const int u = __shfl_up(v, s, 64);
        if (lane >= s) v += u;
    }
    return v;
}

// Chunks.  A unit is a sequence, a key-value head and 16 of its query heads; a unit's tiles go in
// chunks of one size, chosen so that there are about `target` chunks.  Chunks are numbered sequence by
// sequence, then chunk by chunk, then unit by unit: workgroups that run together then read the
// heads of the same tokens, which lie next to each other in memory.
struct Place {
    int b, unit, chunk, count;  // count: chunks of each of the sequence's units; b -1: no such chunk
    int length, size;           // of the sequence; tiles of a chunk
};
__device__ __forceinline__ Place find_chunk(const PagedArgs& a, int at, int units, int lane) {
    Place p{-1, 0, 0, 1, 0, 1 << 30};
    if (a.target == 1) {  // every unit is one chunk
        p.b = at / units;
        p.unit = at - p.b * units;
        p.length = a.lengths[p.b];
        return p;
    }
    // the lane's sequences: the first 64 stay in registers
    const int length = lane < a.batch ? a.lengths[lane] : 0;
    const int tiles = lane < a.batch ? Visible(a, length).tiles : 0;
    int64_t total = __shfl(wave_scan(tiles, lane), 63, 64);
    for (int i = 64; i < a.batch; i += 64)
        total += __shfl(wave_scan(i + lane < a.batch ? Visible(a, a.lengths[i + lane]).tiles : 0, lane), 63, 64);
    const int64_t want = (total * units + a.target - 1) / a.target;
    p.size = static_cast<int>(min(max(want, static_cast<int64_t>(a.min_tiles)), static_cast<int64_t>(1) << 30));
    int before = 0;
    for (int i = 0; i < a.batch; i += 64) {
        const int n = i == 0 ? length : i + lane < a.batch ? a.lengths[i + lane] : 0;
        const int t = i == 0 ? tiles : Visible(a, n).tiles;
        const int per = i + lane < a.batch ? max(1, (t + p.size - 1) / p.size) : 0;
        const int end = before + wave_scan(per * units, lane);
        const uint64_t past = __ballot(end > at);
        if (past) {
            const int l = __builtin_ctzll(past);
            p.b = i + l;
            p.count = __builtin_amdgcn_readlane(per, l);
            p.length = __builtin_amdgcn_readlane(n, l);
            const int in = at - (__builtin_amdgcn_readlane(end, l) - p.count * units);
            p.chunk = in / units;
            p.unit = in - p.chunk * units;
            return p;
        }
        before = __builtin_amdgcn_readlane(end, 63);
    }
    return p;
}

// QC: type of q and out.  F8: the cache holds E4M3 codes (else QC).  WHOLE: 16 consecutive tokens
// are always on one page (page_size % 16 == 0), so a tile needs two page numbers, which are the
// wave's (scalar); else every lane looks up the pages of its tokens, a tile ahead.  4
// sequences of up to 9000 tokens, 8 heads, bf16, pages of 16: 30.4 us WHOLE, 32.1 not; 48 of up to 8192,
// E4M3: 109 us by pages of 64, 117 by pages of 8.  Without the look-up ahead pages of 8 took 44.5 for 32.3.
template <int QC, int D, bool F8, bool WHOLE>
__global__ __launch_bounds__(kWaves * 64, D == 256 ? 1 : 2) void paged_kernel(PagedArgs a) {
    using L = Lay<D, F8>;
    constexpr int ES = L::ES;
    __shared__ float lo[kWaves][D][17];
    __shared__ float lm[kWaves][16], ll[kWaves][16];

    const int lane = threadIdx.x & 63;
    const int r16 = lane & 15, c = lane >> 4;

    const int units = a.kv_heads * a.head_tiles;
    const Place place = find_chunk(a, blockIdx.x, units, lane);
    if (place.b < 0) return;  // the whole workgroup
    const int b = __builtin_amdgcn_readfirstlane(place.b), unit = __builtin_amdgcn_readfirstlane(place.unit);
    const int kvh = unit / a.head_tiles, h0 = (unit - kvh * a.head_tiles) * 16;
    const int nh = min(16, a.group - h0);  // query heads of this unit
    const Visible vis(a, __builtin_amdgcn_readfirstlane(place.length));
    const int size = __builtin_amdgcn_readfirstlane(place.size);
    const int t0 = __builtin_amdgcn_readfirstlane(place.chunk) * size, t1 = min(vis.tiles, t0 + size);
    const int* table = a.table + b * a.table_stride;

    v4u q[D / 32];
    {
        const uint8_t* qp = a.q + (b * a.q_b + static_cast<int64_t>(kvh * a.group + h0 + min(r16, nh - 1)) * a.q_h) * 2;
#pragma unroll
        for (int n = 0; n < D / 32; ++n) {
            const int d = L::KW == 8 ? n * 32 + c * 8 : (n >> 1) * 64 + c * 16 + (n & 1) * 8;
            q[n] = *reinterpret_cast<const v4u*>(qp + d * 2);
        }
    }
    const float to_log2 = a.scale * kLog2e * (a.k_scale ? *a.k_scale : 1.0f);

    const uint8_t* kbase = a.k + kvh * a.k_head * ES;
    const uint8_t* vbase = a.v + kvh * a.v_head * ES;

    const PagedRows rows{kbase, vbase, table, a.k_page, a.k_tok, a.v_page, a.v_tok, a.pages, a.page_size, a.by_page};
    paged_tiles<QC, D, F8, WHOLE>(rows, PagedTiles{vis.sink_tiles, vis.sink_end, vis.start, vis.len, t0, t1}, q, to_log2, lo, lm, ll);
    __syncthreads();
    if (a.plan && place.chunk == 0 && threadIdx.x == 0) a.plan[b * units + unit] = make_int2(blockIdx.x, place.count);
    const float vs = a.v_scale ? *a.v_scale : 1.0f;
    for (int e = threadIdx.x; e < nh * D; e += kWaves * 64) {
        const int h = e / D, d = e % D;
        float top = lm[0][h];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) top = fmaxf(top, lm[w][h]);
        float o = 0.0f, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float f = exp2_hw(lm[w][h] - top);
            o += f * lo[w][d][h];
            sum += f * ll[w][h];
        }
        if (place.count == 1) {
            const float y = sum == 0.0f ? 0.0f : o / sum * vs;
            const int64_t at = (static_cast<int64_t>(b) * a.heads + kvh * a.group + h0 + h) * D + d;
            static_cast<uint16_t*>(a.out)[at] = static_cast<uint16_t>(QC == CKH_BF16 ? f_to_bf16_rne(y) : f_to_f16(y));
        } else {
            float* part = a.part + (static_cast<int64_t>(blockIdx.x) * 16 + h) * (D + 2);
            part[d] = o;
            if (d == 0) {
                part[D] = top;
                part[D + 1] = sum;
            }
        }
    }
}

// Joins the chunks of the sequences that have several: a workgroup per sequence and query head.
// The chunks' factors go to LDS first, so that their outputs are read without waiting for them.
template <int QC, int D>
__global__ __launch_bounds__(256) void join_kernel(PagedArgs a) {
    constexpr int N = 256 / D;  // chunks taken at a time
    __shared__ float so[N][D], factor[kMaxChunks], red[8];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int b = blockIdx.y, h = blockIdx.x;
    const int units = a.kv_heads * a.head_tiles;
    const int kvh = h / a.group, in = h - kvh * a.group;
    const int2 plan = a.plan[b * units + kvh * a.head_tiles + (in >> 4)];
    const int count = plan.y;
    if (count == 1) return;
    const float* part = a.part + (static_cast<int64_t>(plan.x) * 16 + (in & 15)) * (D + 2);
    const int64_t step = static_cast<int64_t>(units) * 16 * (D + 2);
    float top = -1e30f;
    for (int i = threadIdx.x; i < count; i += 256) top = fmaxf(top, part[i * step + D]);
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) top = fmaxf(top, __shfl_xor(top, s, 64));
    if (lane == 0) red[wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const int d = threadIdx.x % D, g = threadIdx.x / D;
    float o = 0.0f, sum = 0.0f;
    for (int i = threadIdx.x; i < count; i += 256) {
        const float f = exp2_hw(part[i * step + D] - top);
        factor[i] = f;
        sum += f * part[i * step + D + 1];
    }
    __syncthreads();
    if (g < N) {
#pragma unroll 8
        for (int i = g; i < count; i += N) o += factor[i] * part[i * step + d];
    }
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) sum += __shfl_xor(sum, s, 64);
    if (lane == 0) red[4 + wave] = sum;
    if (g < N) so[g][d] = o;
    __syncthreads();
    if (threadIdx.x < D) {
        o = so[0][d];
#pragma unroll
        for (int i = 1; i < N; ++i) o += so[i][d];
        sum = red[4] + red[5] + red[6] + red[7];
        const float y = sum == 0.0f ? 0.0f : o / sum * (a.v_scale ? *a.v_scale : 1.0f);
        static_cast<uint16_t*>(a.out)[(static_cast<int64_t>(b) * a.heads + h) * D + d] =
            static_cast<uint16_t>(QC == CKH_BF16 ? f_to_bf16_rne(y) : f_to_f16(y));
    }
}

// How a call is split, from what the host knows: the units and the tokens their tables can hold.
struct Split {
    int target, min_tiles;  // as in PagedArgs
    int64_t slots;          // workgroups that the call may need
};
Split paged_split(int64_t units, int64_t capacity) {
    const int64_t tiles = cdiv(capacity, 32) + 2;  // a unit's at most, with the sinks'
    // Chunks of 16 tiles at least, four a wave: with 8 the joins cost more than the shorter chunks
    // gain (4 x 30000 tokens of one head 24.5 us against 23.1) unless even chunks of 16 leave most of
    // the CUs idle (4000 tokens of 8 heads: 11.9 against 15.5).
    const int min_tiles = units * tiles < 8 * device_cus() && tiles > 32 ? 8 : 16;
    if (tiles <= min_tiles) return {1, min_tiles, units};
    // Two or three workgroups are resident on a CU; four a CU even out their ends (48 ragged
    // sequences in bf16: 168 us; three 175; eight 165, but 64 windows of 1024 tokens 68 for 60).
    // Each unit may have one chunk more for its ragged end.
    const int target = std::clamp(4 * device_cus(), 2, kMaxChunks);
    return {target, min_tiles, std::min(units * cdiv(tiles, min_tiles), units + target)};
}

template <int QC, int D, bool F8>
void launch_paged(const PagedArgs& a, int64_t slots, bool join, hipStream_t st) {
    if (a.page_size % 16 == 0) paged_kernel<QC, D, F8, true><<<static_cast<unsigned>(slots), kWaves * 64, 0, st>>>(a);
    else paged_kernel<QC, D, F8, false><<<static_cast<unsigned>(slots), kWaves * 64, 0, st>>>(a);
    if (join) join_kernel<QC, D><<<dim3(a.heads, a.batch), 256, 0, st>>>(a);
}

template <int QC, bool F8>
void launch_paged(int dim, const PagedArgs& a, int64_t slots, bool join, hipStream_t st) {
    if (dim == 64) launch_paged<QC, 64, F8>(a, slots, join, st);
    else if (dim == 96) launch_paged<QC, 96, F8>(a, slots, join, st);
    else if (dim == 128) launch_paged<QC, 128, F8>(a, slots, join, st);
    else launch_paged<QC, 256, F8>(a, slots, join, st);
}

}  // namespace attn
}  // namespace ckh

using namespace ckh;

static int64_t paged_units(int64_t batch, int64_t heads, int64_t kv_heads) {
    return batch * kv_heads * cdiv(heads / kv_heads, 16);
}

extern "C" int64_t ckh_paged_attention_workspace_bytes(int64_t batch, int64_t heads, int64_t kv_heads, int64_t dim,
                                                       int64_t page_size, int64_t max_pages) {
    if (batch <= 0 || heads <= 0 || kv_heads <= 0 || dim <= 0 || page_size <= 0 || max_pages < 0) return 0;
    const int64_t units = paged_units(batch, heads, kv_heads);
    const attn::Split split = attn::paged_split(units, page_size * max_pages);
    return split.target == 1 ? 0 : split.slots * 16 * (dim + 2) * 4 + units * 8;
}

extern "C" int ckh_paged_attention(const void* q, const void* k_cache, const void* v_cache, const void* page_table,
                                   const void* lengths, const void* k_scale, const void* v_scale, void* out,
                                   int64_t batch, int64_t heads, int64_t kv_heads, int64_t dim, int64_t pages,
                                   int64_t page_size, int64_t max_pages, int64_t table_stride, const int64_t* strides,
                                   int64_t window, int64_t sinks, float scale, int q_code, int cache_code,
                                   void* workspace, int64_t workspace_bytes, uintptr_t stream) {
    CKH_REQUIRE(q_code == CKH_F16 || q_code == CKH_BF16, "paged_attention: unsupported query dtype %d", q_code);
    CKH_REQUIRE(cache_code == q_code || cache_code == CKH_E4M3, "paged_attention: cache dtype %d with query dtype %d",
                cache_code, q_code);
    CKH_REQUIRE(dim == 64 || dim == 96 || dim == 128 || dim == 256, "paged_attention: head_dim %lld is not 64, 96, 128 or 256",
                static_cast<long long>(dim));
    CKH_REQUIRE(batch >= 0 && heads >= 0 && kv_heads > 0 && heads % kv_heads == 0 && batch <= 65535 && heads <= 65535,
                "paged_attention: %lld heads over %lld key-value heads, batch %lld", static_cast<long long>(heads),
                static_cast<long long>(kv_heads), static_cast<long long>(batch));
    CKH_REQUIRE(pages > 0 && pages <= INT32_MAX && page_size > 0 && max_pages >= 0 && page_size <= INT32_MAX &&
                    max_pages <= INT32_MAX && max_pages * page_size <= INT32_MAX - 64,
                "paged_attention: %lld pages of %lld tokens, %lld a sequence", static_cast<long long>(pages),
                static_cast<long long>(page_size), static_cast<long long>(max_pages));
    // find_chunk sums the tiles of 64 sequences in 32 bits
    CKH_REQUIRE(std::min<int64_t>(batch, 64) * (cdiv(max_pages * page_size, 32) + 1) <= INT32_MAX,
                "paged_attention: page tables of %lld tokens for %lld sequences", static_cast<long long>(max_pages * page_size),
                static_cast<long long>(batch));
    CKH_REQUIRE(window >= 0 && window <= INT32_MAX && sinks >= 0 && sinks <= INT32_MAX, "paged_attention: window %lld, sinks %lld",
                static_cast<long long>(window), static_cast<long long>(sinks));
    if (batch == 0 || heads == 0) return CKH_OK;
    CKH_REQUIRE(q && k_cache && v_cache && (page_table || max_pages == 0) && lengths && out && strides, "paged_attention: null pointer");
    const int es = cache_code == CKH_E4M3 ? 1 : 2;
    // q: batch, head; k: page, token, head; v: page, token, head (elements)
    for (int i = 0; i < 8; ++i)
        CKH_REQUIRE(strides[i] >= 0 && strides[i] * (i < 2 ? 2 : es) % 16 == 0, "paged_attention: stride %d (%lld) is not a multiple of 16 bytes",
                    i, static_cast<long long>(strides[i]));
    CKH_REQUIRE(strides[3] * es < (int64_t(1) << 25) && strides[6] * es < (int64_t(1) << 25), "paged_attention: token stride too large");
    CKH_REQUIRE(aligned(q, 16) && aligned(k_cache, 16) && aligned(v_cache, 16) && aligned(out, 2) && aligned(page_table, 4) &&
                    aligned(lengths, 4) && aligned(k_scale, 4) && aligned(v_scale, 4),
                "paged_attention: misaligned pointer");
    const int64_t units = paged_units(batch, heads, kv_heads);
    CKH_REQUIRE(units <= (1 << 28), "paged_attention: too many heads and sequences");
    const int64_t need = ckh_paged_attention_workspace_bytes(batch, heads, kv_heads, dim, page_size, max_pages);
    // without a workspace every sequence is one chunk
    attn::Split split = attn::paged_split(units, page_size * max_pages);
    if (need > 0 && !(workspace && workspace_bytes >= need && aligned(workspace, 8))) split = {1, 16, units};
    attn::PagedArgs a{};
    a.q = static_cast<const uint8_t*>(q);
    a.k = static_cast<const uint8_t*>(k_cache);
    a.v = static_cast<const uint8_t*>(v_cache);
    a.table = static_cast<const int*>(page_table);
    a.lengths = static_cast<const int*>(lengths);
    a.k_scale = static_cast<const float*>(k_scale);
    a.v_scale = static_cast<const float*>(v_scale);
    a.out = out;
    a.part = static_cast<float*>(workspace);
    a.q_b = strides[0], a.q_h = strides[1];
    a.k_page = strides[2], a.k_tok = strides[3], a.k_head = strides[4];
    a.v_page = strides[5], a.v_tok = strides[6], a.v_head = strides[7];
    a.table_stride = table_stride;
    a.batch = static_cast<int>(batch), a.heads = static_cast<int>(heads), a.kv_heads = static_cast<int>(kv_heads);
    a.group = static_cast<int>(heads / kv_heads), a.head_tiles = static_cast<int>(cdiv(a.group, 16));
    a.pages = static_cast<int>(pages), a.page_size = static_cast<int>(page_size), a.max_pages = static_cast<int>(max_pages);
    a.window = static_cast<int>(window), a.sinks = static_cast<int>(sinks);
    a.target = split.target, a.min_tiles = split.min_tiles;
    a.scale = scale;
    a.by_page = fast_div(static_cast<uint32_t>(page_size));
    const int64_t slots = split.slots;
    const bool join = split.target > 1;
    if (join) a.plan = reinterpret_cast<int2*>(static_cast<uint8_t*>(workspace) + slots * 16 * (dim + 2) * 4);
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const int d = static_cast<int>(dim);
    if (q_code == CKH_BF16) {
        if (es == 1) attn::launch_paged<CKH_BF16, true>(d, a, slots, join, st);
        else attn::launch_paged<CKH_BF16, false>(d, a, slots, join, st);
    } else {
        if (es == 1) attn::launch_paged<CKH_F16, true>(d, a, slots, join, st);
        else attn::launch_paged<CKH_F16, false>(d, a, slots, join, st);
    }
    return check_launch("paged_attention");
}
