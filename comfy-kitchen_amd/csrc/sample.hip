// The next token of each row of logits, drawn with a given random number, for gfx950.
//
// Tokens stand in the order of their logits, the largest first, equal ones by their number.  With
// w = exp((l - max) / temperature), the first tokens of that order are kept that
//   are among the first top_k,
//   are needed to reach top_p of the weight of those,
//   have w >= min_p,
// and the first is; the result is the first token whose running weight exceeds u times the weight of
// all that are kept.  What lies 32 temperatures or more (kBins bins: 31.94 to 32, by where in its bin the largest lies) under the
// largest logit is not kept: e^-31.94 each, 2^-22 of the row where 2^24 logits lie there.
//
// Nothing is sorted.  Logits fall into bins of 1/16 temperature, and
//   - a first launch (a workgroup for 8192 logits, which it holds in registers) counts and sums the
//     weights of its logits by bin, from its own largest logit down;
//   - a second (a workgroup a row) adds these up, which gives the bins that the borders of top_k, top_p,
//     min_p and the drawn token lie in; reads the row again for the few logits of those bins; and finds
//     the places in them: one wave where there are at most 64, else by counting over ever narrower ranges of
//     (logit, number).  Bins that do not fit LDS are narrowed over the row in memory.
// What bounds them: the first, instructions and LDS atomics, 18 of 64 bits for a logit (256 rows of 128000 in f32, 131 MB:
// 29 us); the second, one CU's loads and instructions for a row, and some 8 us of steps that wait for each other (40 us of
// that case; 64 rows of 150001 in bf16: 12 + 26; one row of 32000: 4.4 + 12.6).  A row of the second by several workgroups
// would need a launch more, or workgroups that wait for each other, for less than the 8 us that stay.
//
// A weight is a 32-bit fixed-point number relative to its bin's upper end, taken from the logit in 64 bits;
// sums of them are whole numbers, so they do not depend on the order in which atomics add them.  The
// 2^-33 by which a weight is rounded is nothing to u's 2^-24.  Running sums are compared with 2^-36 of
// slack, so that sums which are equal by definition (equal logits, u = 1/2) compare as equal.
#include "ckh_common.h"

namespace ckh {
namespace sample {

constexpr int kBins = 512;
constexpr double kPer = 16.0;     // bins of a temperature
constexpr int kChunk = 8192;      // logits of a workgroup of the first launch
constexpr int kFirst = 512;       // its threads
constexpr int kThreads = 512;     // of the second launch's workgroup
constexpr int kList = 4096;       // logits that it holds
constexpr int kQueue = 3008;      // 16-byte pieces of the row that it looks at twice
constexpr int kSubBits = 9, kSub = 1 << kSubBits;  // ranges that it counts by
static_assert(kSub == kThreads && kBins <= kThreads, "a range and a bin a thread");
constexpr int kMaxChunks = 2048;
constexpr double kSlack = 0x1p-36;

struct Args {
    const uint8_t* logits;
    const float* u;
    const float *temperature, *top_p, *min_p;  // one a row, or null: the values below
    const int* top_k;
    double temperature_all, top_p_all, min_p_all;
    int64_t* out;
    uint64_t* bins;    // [row][chunk][kBins]: count << 48 | weight
    int2* top;         // [row][chunk]: the largest logit's bits, its number
    int64_t row_bytes;
    int rows, vocab, chunks, top_k_all;
    __device__ __forceinline__ double temperature_of(int r) const { return temperature ? temperature[r] : temperature_all; }
    __device__ __forceinline__ int top_k_of(int r) const { return top_k ? top_k[r] : top_k_all; }
    // the largest logit is all that counts
    __device__ __forceinline__ bool greedy(int r) const { return !(temperature_of(r) > 0.0) || top_k_of(r) == 1; }
};

struct __attribute__((packed, aligned(2))) Piece16 {
    uint32_t w[4];
};

// 8 logits of a row from the place `begin` on.
template <int C>
__device__ __forceinline__ void load_logits(const uint8_t* row, int begin, float (&v)[8]) {
    if constexpr (C == CKH_F32) {
        struct __attribute__((packed, aligned(4))) Piece32 {
            float f[8];
        };
        const Piece32 p = *reinterpret_cast<const Piece32*>(row + static_cast<int64_t>(begin) * 4);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = p.f[e];
    } else {
        const Piece16 p = *reinterpret_cast<const Piece16*>(row + static_cast<int64_t>(begin) * 2);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t h = (p.w[e >> 1] >> (16 * (e & 1))) & 0xffffu;
            v[e] = C == CKH_BF16 ? bf16_to_f(h) : f16_to_f(h);
        }
    }
}

// A row of 8 logits or more in pieces of 8: the one from i on begins at begin(i), and what it holds before i is another's.
// (Where the row ends inside a piece, the piece lies at the row's end, so that all loads are whole ones.)
template <int C>
struct Pieces {
    const uint8_t* row;
    int vocab;
    __device__ __forceinline__ int begin(int i) const { return min(i, vocab - 8); }
    __device__ __forceinline__ void load(int i, float (&v)[8]) const { load_logits<C>(row, begin(i), v); }
};

// Bins under a largest logit `top`.
struct Scale {
    double per, top_bin, top_at;  // bins of a unit; the bin and place of `top`
    float top;
    __device__ __forceinline__ Scale(float t, double temperature) : top(t) {
        per = fmin(kPer / temperature, 1e200);
        top_at = t == __builtin_inff() ? 0.0 : static_cast<double>(t) * per;
        top_bin = floor(top_at);
    }
    // A finite logit's bin, counted down from the top's (or kBins and more); y: its place in the bin, 0 .. 1.
    __device__ __forceinline__ uint32_t finite_bin(float l, double& y) const {
        const double at = static_cast<double>(l) * per, b = floor(at);
        y = at - b;
        return static_cast<uint32_t>(fmin(top_bin - b, static_cast<double>(kBins)));
    }
    __device__ __forceinline__ int bin(float l, double& y) const {
        if (top == __builtin_inff()) {  // infinities alone count, all alike
            y = 0.0;
            return l == top ? 0 : kBins;
        }
        return static_cast<int>(finite_bin(l, y));
    }
};

// a b + c with c in scalar registers (left to itself the compiler copies every constant to vector ones first).
__device__ __forceinline__ double fma_const(double a, double b, double c) {
    double r;
    __asm__("v_fma_f64 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "s"(c));
    return r;
}

// 2^32 exp((y - 1) / 16), 0 <= y <= 1, as a whole number: a polynomial through five Chebyshev points, 2^-35 off.
__device__ __forceinline__ uint64_t weight(double y) {
    double e = __fma_rn(y, 6.162469714203124e-07, 3.820811450174273e-05);
    e = fma_const(y, e, 0.0018347971173092148);
    e = fma_const(y, e, 0.05871331567765126);
    e = fma_const(y, e, 0.9394130628284427);
    // 2^20 has steps of 2^-32: the sum's low bits are the rounded number
    return static_cast<uint64_t>(__double_as_longlong(e + 0x1p20)) & 0x1ffffffffull;
}

// ---------------------------------------------------------------- first launch
template <int C>
__global__ __launch_bounds__(kFirst) void bins_kernel(Args a) {
    constexpr int N = kChunk / (kFirst * 8);
    __shared__ uint64_t bins[kBins];
    __shared__ float top_of[kFirst / 64];
    __shared__ int first;
    const int chunk = blockIdx.x, row = blockIdx.y;
    const Pieces<C> pieces{a.logits + row * a.row_bytes, a.vocab};
    float v[N][8];
    float top = -__builtin_inff();
    const auto place = [&](int n) { return chunk * kChunk + (n * kFirst + static_cast<int>(threadIdx.x)) * 8; };
    const bool whole = a.vocab >= 8;
    if (whole) {
#pragma unroll
        for (int n = 0; n < N; ++n) pieces.load(place(n), v[n]);
    } else {
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[n][e] = place(n) + e < a.vocab ? load1<C>(pieces.row, place(n) + e) : -__builtin_inff();
    }
    for (int i = threadIdx.x; i < kBins; i += kFirst) bins[i] = 0;
    if (whole && (chunk + 1) * kChunk > a.vocab) {  // the row's end: what a piece there holds of another's does not count
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < place(n) - pieces.begin(place(n))) v[n][e] = -__builtin_inff();
    }
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, v[n][e]);  // a NaN is not taken
#pragma unroll
    for (int s = 32; s >= 1; s >>= 1) top = fmaxf(top, __shfl_xor(top, s, 64));
    if ((threadIdx.x & 63) == 0) top_of[threadIdx.x >> 6] = top;
    if (threadIdx.x == 0) first = INT32_MAX;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kFirst / 64; ++w) top = fmaxf(top, top_of[w]);
    bool here = false;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int e = 0; e < 8; ++e) here |= v[n][e] == top;
    if (here && top > -__builtin_inff()) {
        int at = INT32_MAX;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (v[n][e] == top) at = min(at, (whole ? pieces.begin(place(n)) : place(n)) + e);
        atomicMin(&first, at);
    }
    const int64_t slot = static_cast<int64_t>(row) * a.chunks + chunk;
    if (a.greedy(row) || top == -__builtin_inff()) {
        __syncthreads();
        if (threadIdx.x == 0) a.top[slot] = make_int2(static_cast<int>(as_u(top)), first);
        return;
    }
    const float largest = top;
    if (top == __builtin_inff()) {  // infinities alone count, all alike
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[n][e] = v[n][e] == top ? 0.0f : -__builtin_inff();
        top = 0.0f;
    }
    const Scale scale(top, a.temperature_of(row));
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            double y;
            const uint32_t b = scale.finite_bin(v[n][e], y);  // -inf: kBins
            const uint64_t one = (1ull << 48) | weight(y);
            if (b < kBins) atomicAdd(reinterpret_cast<unsigned long long*>(&bins[b]), static_cast<unsigned long long>(one));
        }
    __syncthreads();
    if (threadIdx.x == 0) a.top[slot] = make_int2(static_cast<int>(as_u(largest)), first);
    for (int i = threadIdx.x; i < kBins; i += kFirst) a.bins[slot * kBins + i] = bins[i];
}

// --------------------------------------------------------------- second launch
// A token's place in the order as one number: its logit's bits, turned so that the larger logit is the
// smaller number (16-bit types have no more bits than that), then the token's own number.
template <int C>
struct Order {
    static constexpr int kDrop = C == CKH_F32 ? 0 : C == CKH_F16 ? 13 : 16;  // zeros in a widened logit
    int bits;  // of a token's number
    __device__ __forceinline__ uint64_t key(float l) const {
        const uint32_t u = as_u(l + 0.0f);  // one zero
        return (u & 0x80000000u ? u : ~u & 0x7fffffffu) >> kDrop;
    }
    __device__ __forceinline__ uint64_t of(float l, int token) const { return key(l) << bits | static_cast<uint32_t>(token); }
    __device__ __forceinline__ float logit(uint64_t order) const {
        const uint32_t up = static_cast<uint32_t>(order >> bits) << kDrop;
        return as_f(up & 0x80000000u ? up : ~up & 0x7fffffffu & ~((1u << kDrop) - 1u));
    }
    __device__ __forceinline__ int64_t token(uint64_t order) const { return static_cast<int64_t>(order & ((1ull << bits) - 1)); }
};

enum Ask { kRank, kReach, kPass };  // the r-th token; the first whose running weight reaches, or passes, a target

// What the bins' sums tell of the borders.
struct Found {
    double low_k, high_k, low, high;  // the weight that top_k leaves, that is kept: at least and at most
    int bin_k, bin_m;                 // the bins of top_k's and min_p's borders
    bool by_k, by_p, by_min;          // which borders have to be looked for
};

struct Shared {
    double below[kBins];          // weight of the bins up to and with this one
    uint32_t counts[kBins];       // their tokens
    uint16_t under[kMaxChunks];   // by how many bins a chunk's largest logit is under the row's
    int queue[kQueue];            // pieces of the row that hold some of them
    uint64_t list[kList];         // places of the tokens of the bins that are looked into
    uint64_t sub_weight[kSub], few[64];
    uint32_t sub_count[kSub];
    float low[3], high[3];        // logits of these bins: of top_k's border, of the tighter of top_p's and min_p's, of the draw
    uint32_t listed, queued, fews;
    int bin, sub;
    Found found;
    unsigned long long above_weight, sum;
    uint32_t above_count, sub_n;
    double running;
    uint64_t place;
};

template <int C>
struct Row {
    const Args& a;
    Shared& s;
    Pieces<C> pieces;
    Scale scale;
    Order<C> order;
    int lane;
    bool whole;  // the list does not hold the bins that are looked into: the row itself is read

    __device__ __forceinline__ double unit(int bin) const {  // a weight's 2^-32 in this bin, relative to the largest logit's weight
        return exp((scale.top_bin - scale.top_at + 1.0 - bin) * (1.0 / kPer)) * 0x1p-32;
    }
    __device__ __forceinline__ bool is(Ask ask, double running, double target) const {
        return ask == kPass ? running > target * (1.0 + kSlack) : running >= target * (1.0 - kSlack);
    }
    __device__ __forceinline__ double base(int bin) const { return bin ? s.below[bin - 1] : 0.0; }

    // Logits that a bin's lie between (a little more than the bin).
    __device__ __forceinline__ float lower(int bin) const {
        if (scale.top == __builtin_inff()) return scale.top;
        const float f = static_cast<float>((scale.top_bin - bin) / scale.per);
        return fmaxf(f - fabsf(f) * 0x1p-22f - 1e-37f, -3.402823466e38f);
    }
    __device__ __forceinline__ float upper(int bin) const {
        if (scale.top == __builtin_inff()) return scale.top;
        const float f = static_cast<float>((scale.top_bin - bin + 1.0) / scale.per);
        return fminf(f + fabsf(f) * 0x1p-22f + 1e-37f, scale.top);
    }

    // The workgroup: lists the tokens whose logits lie in one of the ranges low .. high.  What bounds it is instructions, so
    // 16-byte pieces are looked at as they lie in memory: a range of logits of one sign is a range of their bits, and x is
    // in it where x - first, as an unsigned number, is at most its width; the least of these over a piece tells of the piece,
    // and the few pieces that hold something are looked at again logit by logit.  (Widened and compared as floats the row
    // took three times as long: 64 rows of 150001 in bf16 24 us of the launch.)
    static constexpr int kPiece = C == CKH_F32 ? 4 : 8;  // logits of a piece
    static __device__ __forceinline__ uint32_t code(float l) {  // a logit's bits in its own type, rounded towards zero
        if constexpr (C == CKH_F32) return as_u(l);
        else if constexpr (C == CKH_BF16) return as_u(l) >> 16;
        else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(l, 0.0f)) & 0xffffu;
    }
    // Q ranges of bits at most.
    template <int Q>
    __device__ __forceinline__ void scan(const uint32_t (&first)[6], const uint32_t (&width)[6]) const {
        constexpr int U = 8;  // pieces of a thread in flight
        typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
        struct __attribute__((packed, aligned(C == CKH_F32 ? 4 : 2))) Words {
            uint32_t w[4];
        };
        const auto load = [&](Words (&x)[U], int i0) {
#pragma unroll
            for (int n = 0; n < U; ++n) {
                const int i = min(i0 + (n * kThreads + static_cast<int>(threadIdx.x)) * kPiece, a.vocab - kPiece);
                x[n] = *reinterpret_cast<const Words*>(pieces.row + static_cast<int64_t>(i) * (16 / kPiece));
            }
        };
        Words x[U], next[U];
        load(x, 0);
        constexpr int kStep = kThreads * kPiece * U;
        for (int i0 = 0; i0 < a.vocab; i0 += kStep) {
            if (i0 + kStep < a.vocab) load(next, i0 + kStep);
#pragma unroll
            for (int n = 0; n < U; ++n) {
                bool hit = false;
#pragma unroll
                for (int q = 0; q < Q; ++q) {
                    if constexpr (C == CKH_F32) {
                        uint32_t least = x[n].w[0] - first[q];
#pragma unroll
                        for (int e = 1; e < 4; ++e) {
                            const uint32_t d = x[n].w[e] - first[q];
                            least = d < least ? d : least;
                        }
                        hit |= least <= width[q];
                    } else {
                        const u16x2 from = __builtin_bit_cast(u16x2, first[q] * 0x10001u);
                        u16x2 least = __builtin_bit_cast(u16x2, x[n].w[0]) - from;
#pragma unroll
                        for (int e = 1; e < 4; ++e) least = __builtin_elementwise_min(least, static_cast<u16x2>(__builtin_bit_cast(u16x2, x[n].w[e]) - from));
                        hit |= (least.x < least.y ? least.x : least.y) <= width[q];
                    }
                }
                const int i = i0 + (n * kThreads + static_cast<int>(threadIdx.x)) * kPiece;
                if (hit && i < a.vocab) {
                    const uint32_t place = atomicAdd(&s.queued, 1u);
                    if (place < kQueue) s.queue[place] = i;
                }
            }
#pragma unroll
            for (int n = 0; n < U; ++n) x[n] = next[n];
        }
    }
    __device__ __forceinline__ void gather() const {
        const float low0 = s.low[0], high0 = s.high[0], low1 = s.low[1], high1 = s.high[1], low2 = s.low[2], high2 = s.high[2];
        const auto wanted = [&](float l) { return (l >= low0 && l <= high0) || (l >= low1 && l <= high1) || (l >= low2 && l <= high2); };
        const auto list = [&](float l, int token) {
            if (!wanted(l)) return;
            const uint32_t place = atomicAdd(&s.listed, 1u);
            if (place < kList) s.list[place] = order.of(l, token);
        };
        if (a.vocab < 8) {
            if (static_cast<int>(threadIdx.x) < a.vocab) list(load1<C>(pieces.row, threadIdx.x), threadIdx.x);
            return;
        }
        uint32_t first[6], width[6];
        int ranges = 0;
#pragma unroll
        for (int n = 0; n < 6; ++n) first[n] = code(-__builtin_nanf("")) | (C == CKH_F32 ? 0x7fffffu : 0x7fu), width[n] = 0;  // NaN
        const auto add = [&](uint32_t from, uint32_t to) {
#pragma unroll
            for (int n = 0; n < 6; ++n)
                if (n == ranges) first[n] = from, width[n] = to - from;
            ++ranges;
        };
#pragma unroll
        for (int n = 0; n < 3; ++n) {
            const float lo = s.low[n], hi = s.high[n];
            if (lo > hi) continue;
            if (lo <= 0.0f) add(code(hi < 0.0f ? hi : -0.0f), code(lo < 0.0f ? lo : -0.0f));
            if (hi >= 0.0f) add(code(lo > 0.0f ? lo : 0.0f), code(hi > 0.0f ? hi : 0.0f));
        }
        if (ranges == 1) scan<1>(first, width);
        else if (ranges == 2) scan<2>(first, width);
        else if (ranges == 3) scan<3>(first, width);
        else scan<6>(first, width);
        __syncthreads();
        const int n = min(s.queued, static_cast<uint32_t>(kQueue));
        for (int j = threadIdx.x; j < n; j += kThreads) {
            const int i = s.queue[j], begin = min(i, a.vocab - kPiece);
#pragma unroll
            for (int e = 0; e < kPiece; ++e)
                if (begin + e >= i) list(load1<C>(pieces.row, begin + e), begin + e);
        }
    }

    // f(place in the order, fixed-point weight) for the tokens of a bin
    template <typename F>
    __device__ __forceinline__ void each(int bin, F f) const {
        if (!whole) {
            const uint32_t n = min(s.listed, static_cast<uint32_t>(kList));
            for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
                const uint64_t o = s.list[i];
                double y;
                if (scale.bin(order.logit(o), y) == bin) f(o, weight(y));
            }
        } else {
            for (int i = threadIdx.x * 8; i < a.vocab; i += kThreads * 8) {
                float v[8];
                pieces.load(i, v);
                const int begin = pieces.begin(i);
                for (int e = 0; e < 8; ++e) {
                    double y;
                    if (v[e] > -__builtin_inff() && begin + e >= i && scale.bin(v[e], y) == bin) f(order.of(v[e], begin + e), weight(y));
                }
            }
        }
    }

    // One wave: the first bin that is not empty and whose running weight is (or count reaches) what is asked, or the
    // last that is not empty.
    __device__ __forceinline__ int find(Ask ask, double target, uint32_t rank) const {
        // the first of 64 runs of bins that ends there, then the bin in it
        constexpr int N = kBins / 64;
        const uint32_t all = s.counts[kBins - 1];
        uint64_t hit = 0;
        int i = lane * N + N - 1;
#pragma unroll
        for (int step = 0; step < 2; ++step) {
            const uint32_t n = s.counts[i];
            const double w = s.below[i];
            hit = __ballot(ask == kRank ? n >= rank : is(ask, w, target));
            if (!hit) hit = __ballot(n >= all);
            if (step == 0) i = __builtin_ctzll(hit) * N + min(lane, N - 1);
        }
        return (i - min(lane, N - 1)) + min(static_cast<int>(__builtin_ctzll(hit)), N - 1);
    }

    // One wave, a token a lane (n of them): the one that is asked for, with `above` weight and tokens of its bin before these.
    __device__ __forceinline__ uint64_t pick(uint64_t o, uint64_t w, bool live, int bin, Ask ask, double target, uint32_t rank,
                                             uint64_t above_weight, uint32_t above_count, double& running) const {
        uint64_t sum = 0;
        uint32_t n = 0;
        for (uint64_t left = __ballot(live); left; left &= left - 1) {
            const int j = __builtin_ctzll(left);
            const uint64_t oj = lane_of(o, j), wj = lane_of(w, j);
            if (oj <= o) sum += wj, ++n;
        }
        const double begin = base(bin), one = unit(bin);
        const uint32_t count = (bin ? s.counts[bin - 1] : 0) + above_count + n;
        const double to = begin + static_cast<double>(above_weight + sum) * one;
        const bool here = live && (ask == kRank ? count >= rank : is(ask, to, target));
        // the first of these in the order, or the last of all
        const uint64_t all = __ballot(live), those = __ballot(here);
        uint64_t best = 0;
        int lane_at = -1;
        for (uint64_t left = those ? those : all; left; left &= left - 1) {
            const int j = __builtin_ctzll(left);
            const uint64_t oj = lane_of(o, j);
            if (lane_at < 0 || (those ? oj < best : oj > best)) best = oj, lane_at = j;
        }
        running = __shfl(to, lane_at < 0 ? 0 : lane_at, 64);
        return best;
    }
    static __device__ __forceinline__ uint64_t lane_of(uint64_t v, int j) {
        const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(v), j);
        const uint32_t hi = __builtin_amdgcn_readlane(static_cast<uint32_t>(v >> 32), j);
        return static_cast<uint64_t>(hi) << 32 | lo;
    }

    // One wave, where the list has at most 64 tokens: the one that is asked for in a bin.
    __device__ __forceinline__ uint64_t in_wave(int bin, Ask ask, double target, uint32_t rank, double& running) const {
        const uint64_t o = lane < static_cast<int>(s.listed) ? s.list[lane] : 0;
        double y = 0.0;
        const bool live = lane < static_cast<int>(s.listed) && scale.bin(order.logit(o), y) == bin;
        return pick(o, weight(y), live, bin, ask, target, rank, 0, 0, running);
    }

    // The workgroup: the same in a bin of any size.
    __device__ uint64_t in_group(int bin, Ask ask, double target, uint32_t rank, double& running) {
        uint64_t from = order.of(upper(bin), 0), to = order.of(lower(bin), 0) | ((1ull << order.bits) - 1);
        uint64_t above_weight = 0;
        uint32_t above_count = 0, n = s.counts[bin] - (bin ? s.counts[bin - 1] : 0);
        const uint32_t rank_base = bin ? s.counts[bin - 1] : 0;
        const double begin = base(bin), one = unit(bin);
        while (n > 64) {
            const int shift = max(0, 64 - __clzll(static_cast<long long>(to - from)) - kSubBits);
            s.sub_weight[threadIdx.x] = 0;
            s.sub_count[threadIdx.x] = 0;
            __syncthreads();
            each(bin, [&](uint64_t o, uint64_t w) {
                if (o >= from && o <= to) {
                    const uint32_t i = static_cast<uint32_t>((o - from) >> shift);
                    atomicAdd(reinterpret_cast<unsigned long long*>(&s.sub_weight[i]), static_cast<unsigned long long>(w));
                    atomicAdd(&s.sub_count[i], 1u);
                }
            });
            __syncthreads();
            if (threadIdx.x < 64) {  // a lane's ranges one after the other
                constexpr int N = kSub / 64;
                uint64_t w = 0;
                uint32_t c = 0;
#pragma unroll
                for (int e = 0; e < N; ++e) w += s.sub_weight[lane * N + e], c += s.sub_count[lane * N + e];
                uint64_t end_w = w;
                uint32_t end_c = c;
#pragma unroll
                for (int d = 1; d < 64; d <<= 1) {
                    const uint64_t u = __shfl_up(static_cast<unsigned long long>(end_w), d, 64);
                    const uint32_t m = __shfl_up(end_c, d, 64);
                    if (lane >= d) end_w += u, end_c += m;
                }
                w = above_weight + end_w - w;
                c = above_count + end_c - c;
                int at = kSub, last = -1;
                uint64_t at_w = 0, last_w = 0;
                uint32_t at_c = 0, last_c = 0;
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    const int i = lane * N + e;
                    const uint64_t ow = s.sub_weight[i];
                    const uint32_t oc = s.sub_count[i];
                    if (oc) {
                        last = i, last_w = w, last_c = c;
                        if (at == kSub && (ask == kRank ? rank_base + c + oc >= rank : is(ask, begin + static_cast<double>(w + ow) * one, target)))
                            at = i, at_w = w, at_c = c;
                    }
                    w += ow, c += oc;
                }
                const uint64_t found = __ballot(at < kSub), any = __ballot(last >= 0);
                const int l = found ? __builtin_ctzll(found) : 63 - __builtin_clzll(any | 1);
                if (lane == l) {
                    s.sub = found ? at : last;
                    s.above_weight = found ? at_w : last_w;
                    s.above_count = found ? at_c : last_c;
                    s.sub_n = s.sub < 0 ? 0 : s.sub_count[s.sub];
                }
            }
            __syncthreads();
            above_weight = s.above_weight, above_count = s.above_count, n = s.sub_n;
            from += static_cast<uint64_t>(max(s.sub, 0)) << shift;
            if ((to - from) >> shift) to = from + ((1ull << shift) - 1);
            __syncthreads();
        }
        if (threadIdx.x == 0) s.fews = 0;
        __syncthreads();
        each(bin, [&](uint64_t o, uint64_t) {
            if (o >= from && o <= to) {
                const uint32_t i = atomicAdd(&s.fews, 1u);
                if (i < 64) s.few[i] = o;
            }
        });
        __syncthreads();
        if (threadIdx.x < 64) {
            const bool live = lane < static_cast<int>(s.fews);
            const uint64_t o = live ? s.few[lane] : 0;
            double y = 0.0, r;
            if (live) scale.bin(order.logit(o), y);
            const uint64_t place = pick(o, weight(y), live, bin, ask, target, rank, above_weight, above_count, r);
            if (lane == 0) s.place = place, s.running = r;
        }
        __syncthreads();
        running = s.running;
        const uint64_t place = s.place;
        __syncthreads();
        return place;
    }
};

template <int C>
__global__ __launch_bounds__(kThreads) void pick_kernel(Args a) {
    __shared__ Shared s;
    const int row = blockIdx.x, lane = threadIdx.x & 63;
    const int2* tops = a.top + static_cast<int64_t>(row) * a.chunks;

    // the row's largest logit, the first of equal ones
    float top = -__builtin_inff();
    int at = INT32_MAX;
    for (int c = lane; c < a.chunks; c += 64) {
        const int2 t = tops[c];
        if (as_f(t.x) > top) top = as_f(t.x), at = t.y;
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
        const float t = __shfl_xor(top, d, 64);
        const int i = __shfl_xor(at, d, 64);
        if (t > top || (t == top && i < at)) top = t, at = i;
    }
    if (at == INT32_MAX) at = -1;
    if (a.greedy(row) || at < 0) {  // at -1: no token to draw
        if (threadIdx.x == 0) a.out[row] = at;
        return;
    }
    const double temperature = a.temperature_of(row);
    Row<C> r{a, s, {a.logits + row * a.row_bytes, a.vocab}, Scale(top, temperature), Order<C>{32 - __clz(a.vocab - 1 | 1)}, lane, false};

    // weights and counts of the bins
    for (int c = threadIdx.x; c < a.chunks; c += kThreads) {
        const float t = as_f(tops[c].x);
        double under = kBins;
        if (t == top) under = 0.0;
        else if (t > -__builtin_inff() && top < __builtin_inff()) under = fmin(under, r.scale.top_bin - Scale(t, temperature).top_bin);
        s.under[c] = static_cast<uint16_t>(under);
    }
    if (threadIdx.x == 0) s.listed = s.queued = 0;
    __syncthreads();
    if (threadIdx.x < kBins) {
        uint64_t w = 0;
        uint32_t n = 0;
        const uint64_t* bins = a.bins + static_cast<int64_t>(row) * a.chunks * kBins;
#pragma unroll 8
        for (int c = 0; c < a.chunks; ++c) {
            const int i = static_cast<int>(threadIdx.x) - s.under[c];
            const uint64_t x = i >= 0 ? bins[static_cast<int64_t>(c) * kBins + i] : 0;
            w += x & 0xffffffffffffull;
            n += static_cast<uint32_t>(x >> 48);
        }
        s.below[threadIdx.x] = static_cast<double>(w) * r.unit(threadIdx.x);
        s.counts[threadIdx.x] = n;
    }
    __syncthreads();

    const int top_k = a.top_k_of(row);
    const double top_p = a.top_p ? a.top_p[row] : a.top_p_all;
    const double min_p = fmin(a.min_p ? a.min_p[row] : a.min_p_all, 1.0);
    const double u = fmin(fmax(static_cast<double>(a.u[row]), 0.0), 1.0 - 0x1p-24);  // (fp32 numbers, 0 <= u < 1)
    const bool by_p = top_p < 1.0, by_min = min_p > 0.0;
    if (threadIdx.x < 64) {
        // running sums
        constexpr int N = kBins / 64;
        double f[N], sum = 0.0;
        uint32_t c[N], count = 0;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            f[e] = sum += s.below[lane * N + e];
            c[e] = count += s.counts[lane * N + e];
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const double g = __shfl_up(sum, d, 64);
            const uint32_t k = __shfl_up(count, d, 64);
            if (lane >= d) sum += g, count += k;
        }
        const double before = sum - f[N - 1];
#pragma unroll
        for (int e = 0; e < N; ++e) {
            s.below[lane * N + e] = e + 1 < N ? before + f[e] : sum;
            s.counts[lane * N + e] = count - c[N - 1] + c[e];
        }
        __asm__ volatile("" ::: "memory");  // (one wave: LDS keeps its order)
        // the bins in which the borders can lie: each border's range follows from the one before it
        const double all = s.below[kBins - 1];
        const bool by_k = top_k > 0 && static_cast<uint32_t>(top_k) < s.counts[kBins - 1];
        Found f0{};
        f0.low_k = f0.high_k = all;
        int from[3] = {0, 0, 0}, to[3] = {-1, -1, -1};
        if (by_k) {
            f0.bin_k = r.find(kRank, 0.0, top_k);
            f0.low_k = r.base(f0.bin_k), f0.high_k = s.below[f0.bin_k];
        }
        f0.low = f0.low_k, f0.high = f0.high_k;
        f0.by_k = by_k, f0.by_p = by_p, f0.by_min = by_min;
        if (by_p) {
            from[1] = r.find(kReach, top_p * f0.low_k, 0), to[1] = r.find(kReach, top_p * f0.high_k, 0);
            f0.low = fmin(f0.low, r.base(from[1])), f0.high = fmin(f0.high, s.below[to[1]]);
        }
        if (by_min) {
            // the last bin with a part at min_p or over it (the one behind that, by rounding, does no harm)
            const double under = ceil(r.scale.top_bin - r.scale.top_at - log(min_p) * kPer);
            f0.bin_m = static_cast<int>(fmin(fmax(under, 0.0), kBins - 1.0));
            f0.low = fmin(f0.low, r.base(f0.bin_m)), f0.high = fmin(f0.high, s.below[f0.bin_m]);
            // a border that lies behind another does not count
            if (by_p && f0.bin_m < from[1]) f0.by_p = false;
            if ((by_p && f0.bin_m > to[1]) || (by_k && f0.bin_m > f0.bin_k)) f0.by_min = false;
            if (f0.by_min && !f0.by_p) from[1] = to[1] = f0.bin_m;
            if (by_k && f0.by_min && !f0.by_p && f0.bin_m < f0.bin_k) f0.by_k = false;
        }
        if (f0.by_k) from[0] = to[0] = f0.bin_k;
        from[2] = r.find(kPass, u * f0.low, 0), to[2] = r.find(kPass, u * f0.high, 0);
        if (lane == 0) {
            s.found = f0;
#pragma unroll
            for (int i = 0; i < 3; ++i) {
                s.low[i] = to[i] < 0 ? __builtin_inff() : r.lower(to[i]);
                s.high[i] = to[i] < 0 ? -__builtin_inff() : r.upper(from[i]);
            }
        }
    }
    __syncthreads();

    // their tokens
    r.gather();
    __syncthreads();

    // the places of the borders, and the token
    r.whole = s.listed > kList || s.queued > kQueue;
    const bool few = !r.whole && s.listed <= 64;
    if (few && threadIdx.x >= 64) return;
    const Found f = s.found;
    const auto find = [&](Ask ask, double target) {
        if (few) return r.find(ask, target, 0);
        if (threadIdx.x < 64) {
            const int bin = r.find(ask, target, 0);
            if (lane == 0) s.bin = bin;
        }
        __syncthreads();
        return s.bin;  // (in_group has barriers before the next write)
    };
    const auto look = [&](int bin, Ask ask, double target, double& running) {
        return few ? r.in_wave(bin, ask, target, top_k, running) : r.in_group(bin, ask, target, top_k, running);
    };
    double kept = s.below[kBins - 1], running;
    if (f.by_k) {
        look(f.bin_k, kRank, 0.0, running);
        kept = fmin(fmax(running, f.low_k), f.high_k);  // (sums of the same in another order)
    }
    if (f.by_p) {
        const double target = top_p * kept;
        look(find(kReach, target), kReach, target, running);
        kept = fmin(kept, running);
    }
    if (f.by_min) {
        uint64_t sum = 0;
        const auto add = [&](uint64_t o, uint64_t w) {
            const float l = r.order.logit(o);
            if (r.order.key(l) == r.order.key(top) || exp((static_cast<double>(l) - static_cast<double>(top)) / temperature) >= min_p) sum += w;
        };
        if (few) {
            const uint64_t o = lane < static_cast<int>(s.listed) ? s.list[lane] : 0;
            double y;
            if (lane < static_cast<int>(s.listed) && r.scale.bin(r.order.logit(o), y) == f.bin_m) add(o, weight(y));
        } else {
            if (threadIdx.x == 0) s.sum = 0;
            __syncthreads();
            r.each(f.bin_m, add);
        }
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1) sum += __shfl_xor(static_cast<unsigned long long>(sum), d, 64);
        if (!few) {
            if (lane == 0) atomicAdd(&s.sum, static_cast<unsigned long long>(sum));
            __syncthreads();
            sum = s.sum;
        }
        kept = fmin(kept, r.base(f.bin_m) + static_cast<double>(sum) * r.unit(f.bin_m));
    }
    kept = fmin(fmax(kept, f.low), f.high);
    const uint64_t o = look(find(kPass, u * kept), kPass, u * kept, running);
    if (threadIdx.x == 0) a.out[row] = r.order.token(o);
}

template <int C>
void launch(const Args& a, hipStream_t st) {
    bins_kernel<C><<<dim3(a.chunks, a.rows), kFirst, 0, st>>>(a);
    pick_kernel<C><<<a.rows, kThreads, 0, st>>>(a);
}

}  // namespace sample
}  // namespace ckh

using namespace ckh;

extern "C" int64_t ckh_sample_workspace_bytes(int64_t rows, int64_t vocab) {
    if (rows <= 0 || vocab <= 0) return 0;
    return rows * cdiv(vocab, sample::kChunk) * (sample::kBins * 8 + 8);
}

extern "C" int ckh_sample(const void* logits, const void* u, const void* temperature, const void* top_k, const void* top_p,
                          const void* min_p, double temperature_all, int64_t top_k_all, double top_p_all, double min_p_all,
                          void* out, int64_t rows, int64_t vocab, int64_t row_stride, int code, void* workspace,
                          int64_t workspace_bytes, uintptr_t stream) {
    CKH_REQUIRE(code == CKH_F32 || code == CKH_F16 || code == CKH_BF16, "sample: unsupported dtype %d", code);
    CKH_REQUIRE(rows >= 0 && rows <= 65535 && vocab >= 1 && vocab <= sample::kChunk * sample::kMaxChunks && row_stride >= 0, "sample: %lld rows of %lld logits",
                static_cast<long long>(rows), static_cast<long long>(vocab));
    CKH_REQUIRE(temperature || temperature_all >= 0.0, "sample: temperature %g", temperature_all);
    CKH_REQUIRE(top_k || top_k_all >= 0, "sample: top_k %lld", static_cast<long long>(top_k_all));
    CKH_REQUIRE(top_p || (top_p_all >= 0.0), "sample: top_p %g", top_p_all);
    CKH_REQUIRE(min_p || (min_p_all >= 0.0 && min_p_all <= 1.0), "sample: min_p %g", min_p_all);
    if (rows == 0) return CKH_OK;
    const int es = code == CKH_F32 ? 4 : 2;
    CKH_REQUIRE(logits && u && out && workspace, "sample: null pointer");
    CKH_REQUIRE(aligned(logits, es) && aligned(u, 4) && aligned(temperature, 4) && aligned(top_k, 4) && aligned(top_p, 4) &&
                    aligned(min_p, 4) && aligned(out, 8) && aligned(workspace, 8),
                "sample: misaligned pointer");
    const int64_t need = ckh_sample_workspace_bytes(rows, vocab);
    CKH_REQUIRE(workspace_bytes >= need, "sample: a workspace of %lld bytes, needs %lld", static_cast<long long>(workspace_bytes),
                static_cast<long long>(need));
    sample::Args a{};
    a.logits = static_cast<const uint8_t*>(logits);
    a.u = static_cast<const float*>(u);
    a.temperature = static_cast<const float*>(temperature), a.top_p = static_cast<const float*>(top_p);
    a.min_p = static_cast<const float*>(min_p), a.top_k = static_cast<const int*>(top_k);
    a.temperature_all = temperature_all, a.top_p_all = top_p_all, a.min_p_all = min_p_all;
    a.top_k_all = static_cast<int>(top_k_all < vocab ? top_k_all : 0);
    a.out = static_cast<int64_t*>(out);
    a.rows = static_cast<int>(rows), a.vocab = static_cast<int>(vocab);
    a.chunks = static_cast<int>(cdiv(vocab, sample::kChunk));
    a.row_bytes = row_stride * es;
    a.bins = static_cast<uint64_t*>(workspace);
    a.top = reinterpret_cast<int2*>(a.bins + rows * a.chunks * sample::kBins);
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (code == CKH_F32) sample::launch<CKH_F32>(a, st);
    else if (code == CKH_F16) sample::launch<CKH_F16>(a, st);
    else sample::launch<CKH_BF16>(a, st);
    return check_launch("sample");
}
