// The next token of each row of logits, drawn with a given random number, for gfx950.
//
// Tokens stand in the order of their logits, the largest first, equal ones by their number.  With
// w = exp((l - max) / temperature), the first tokens of that order are kept that
//   are among the first top_k,
//   are needed to reach top_p of the weight of those,
//   have w >= min_p,
// and the first is; the result is the first token whose running weight exceeds u times the weight of
// all that are kept.  What lies more than 32 temperatures (kBins bins) under the largest logit is not kept.
//
// Nothing is sorted.  Logits fall into bins of 1/16 temperature, and
//   - a first launch (a workgroup for 8192 logits, which it holds in registers) counts and sums the
//     weights of its logits by bin, from its own largest logit down;
//   - a second (a workgroup a row) adds these up, which gives the bins that the borders of top_k, top_p,
//     min_p and the drawn token lie in; reads the row again for the few logits of those bins; and finds
//     the places in them by counting over ever narrower ranges of (logit, number).
// Both read the row once (the second mostly from a cache), whatever is asked of them; a bin that does not fit
// LDS is narrowed over the row in memory.
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
constexpr int kThreads = 1024;    // of the second launch's workgroup
constexpr int kList = 4096;       // logits that it holds
constexpr int kSub = kThreads;    // ranges that it counts by
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

// The 8 logits from i on (i a multiple of 8) of a row; NaN, and what lies past the row's end, as -inf.
template <int C>
__device__ __forceinline__ void load_logits(const uint8_t* row, int i, int vocab, float (&v)[8]) {
    const float none = -__builtin_inff();
    if (i + 8 <= vocab) {
        if constexpr (C == CKH_F32) {
            struct __attribute__((packed, aligned(4))) Piece32 {
                float f[8];
            };
            const Piece32 p = *reinterpret_cast<const Piece32*>(row + static_cast<int64_t>(i) * 4);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = p.f[e];
        } else {
            const Piece16 p = *reinterpret_cast<const Piece16*>(row + static_cast<int64_t>(i) * 2);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t h = (p.w[e >> 1] >> (16 * (e & 1))) & 0xffffu;
                v[e] = C == CKH_BF16 ? bf16_to_f(h) : f16_to_f(h);
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = i + e < vocab ? load1<C>(row, i + e) : none;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = v[e] == v[e] ? v[e] : none;
}

// Bins under a largest logit `top`.
struct Scale {
    double per, top_bin, top_at;  // bins of a unit; the bin and place of `top`
    float top;
    __device__ __forceinline__ Scale(float t, double temperature) : top(t) {
        per = fmin(kPer / temperature, 1e200);
        top_at = t == __builtin_inff() ? 0.0 : static_cast<double>(t) * per;
        top_bin = floor(top_at);
    }
    // A logit's bin, counted down from the top's, or kBins; x: how far under its bin's upper end, in bins.
    __device__ __forceinline__ int bin(float l, double& x) const {
        const double at = static_cast<double>(l) * per, b = floor(at);
        x = b + 1.0 - at;
        if (top == __builtin_inff()) {  // infinities alone count, all alike
            x = 1.0;
            return l == top ? 0 : kBins;
        }
        const double rel = top_bin - b;
        return rel < kBins ? static_cast<int>(rel) : kBins;
    }
};

// 2^32 exp(-x / 16), 0 <= x <= 1, as a whole number: the terms up to the sixth power, 10^-12 off.
__device__ __forceinline__ uint64_t weight(double x) {
    const double y = x * (-1.0 / kPer);
    double e = __fma_rn(y, 1.0 / 720.0, 1.0 / 120.0);
    e = __fma_rn(y, e, 1.0 / 24.0);
    e = __fma_rn(y, e, 1.0 / 6.0);
    e = __fma_rn(y, e, 0.5);
    e = __fma_rn(y, e, 1.0);
    e = __fma_rn(y, e, 1.0);
    return static_cast<uint64_t>(e * 0x1p32 + 0.5);
}

// ---------------------------------------------------------------- first launch
template <int C>
__global__ __launch_bounds__(kFirst) void bins_kernel(Args a) {
    constexpr int N = kChunk / (kFirst * 8);
    __shared__ uint64_t bins[kBins];
    __shared__ float top_of[kFirst / 64];
    __shared__ int at_of[kFirst / 64];
    const int chunk = blockIdx.x, row = blockIdx.y;
    const uint8_t* logits = a.logits + row * a.row_bytes;
    float v[N][8];
    float top = -__builtin_inff();
    int at = INT32_MAX;
#pragma unroll
    for (int n = 0; n < N; ++n) load_logits<C>(logits, chunk * kChunk + (n * kFirst + threadIdx.x) * 8, a.vocab, v[n]);
    for (int i = threadIdx.x; i < kBins; i += kFirst) bins[i] = 0;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (v[n][e] > top) {
                top = v[n][e];
                at = chunk * kChunk + (n * kFirst + threadIdx.x) * 8 + e;
            }
#pragma unroll
    for (int s = 32; s >= 1; s >>= 1) {
        const float t = __shfl_xor(top, s, 64);
        const int i = __shfl_xor(at, s, 64);
        if (t > top || (t == top && i < at)) top = t, at = i;
    }
    if ((threadIdx.x & 63) == 0) {
        top_of[threadIdx.x >> 6] = top;
        at_of[threadIdx.x >> 6] = at;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kFirst / 64; ++w)
        if (top_of[w] > top || (top_of[w] == top && at_of[w] < at)) top = top_of[w], at = at_of[w];
    const int64_t place = static_cast<int64_t>(row) * a.chunks + chunk;
    if (threadIdx.x == 0) a.top[place] = make_int2(static_cast<int>(as_u(top)), at);
    if (a.greedy(row) || top == -__builtin_inff()) return;
    const Scale scale(top, a.temperature_of(row));
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (v[n][e] == -__builtin_inff()) continue;
            double x;
            const int b = scale.bin(v[n][e], x);
            if (b < kBins) atomicAdd(reinterpret_cast<unsigned long long*>(&bins[b]), (1ull << 48) | weight(x));
        }
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kFirst) a.bins[place * kBins + i] = bins[i];
}

// --------------------------------------------------------------- second launch
// Orders tokens: the larger logit first, then the smaller number.
__device__ __forceinline__ uint64_t order_of(float l, int i) {
    const uint32_t u = as_u(l + 0.0f);  // one zero
    const uint32_t up = u & 0x80000000u ? u : ~u & 0x7fffffffu;
    return static_cast<uint64_t>(up) << 32 | static_cast<uint32_t>(i);
}
__device__ __forceinline__ float logit_of(uint64_t order) {
    const uint32_t up = static_cast<uint32_t>(order >> 32);
    return as_f(up & 0x80000000u ? up : ~up & 0x7fffffffu);
}

struct Shared {
    double below[kBins];     // weight of the bins up to and with this one
    uint32_t count[kBins], sum_count[kBins];
    uint64_t list[kList];
    uint64_t sub_weight[kSub];
    uint32_t sub_count[kSub];
    uint8_t wanted[kBins];
    uint16_t under[kMaxChunks];  // by how many bins a chunk's largest logit is under the row's
    double wave_weight[kThreads / 64];
    uint64_t wave_sum[kThreads / 64];
    uint32_t wave_count[kThreads / 64];
    unsigned long long lo, hi, above_weight;
    uint32_t above_count, listed;
    int found, first;
};

enum Ask { kRank, kReach, kPass };  // the r-th token; the first whose running weight reaches, or passes, a target

// All threads of the workgroup call its members together.
template <int C>
struct Row {
    const Args& a;
    Shared& s;
    const uint8_t* logits;
    Scale scale;
    bool whole;  // the list does not hold the bins that are asked for: the row itself is read

    __device__ __forceinline__ double unit(int bin) const {  // weight of a bin's upper end / 2^32, relative to the largest logit's
        return exp((scale.top_bin - scale.top_at + 1.0 - bin) * (1.0 / kPer)) * 0x1p-32;
    }
    __device__ __forceinline__ bool is(Ask ask, double running, double target) const {
        return ask == kPass ? running > target * (1.0 + kSlack) : running >= target * (1.0 - kSlack);
    }
    // f(order, fixed-point weight) for the tokens of a bin
    template <typename F>
    __device__ __forceinline__ void each(int bin, F f) const {
        if (!whole) {
            for (uint32_t i = threadIdx.x; i < min(s.listed, static_cast<uint32_t>(kList)); i += kThreads) {
                const uint64_t o = s.list[i];
                double x;
                if (scale.bin(logit_of(o), x) == bin) f(o, weight(x));
            }
        } else {
            for (int i = threadIdx.x * 8; i < a.vocab; i += kThreads * 8) {
                float v[8];
                load_logits<C>(logits, i, a.vocab, v);
                for (int e = 0; e < 8; ++e) {
                    double x;
                    if (v[e] != -__builtin_inff() && scale.bin(v[e], x) == bin) f(order_of(v[e], i + e), weight(x));
                }
            }
        }
    }

    // The first bin whose running weight is (or count reaches) what is asked, or the last that is not empty.
    __device__ int find(Ask ask, double target, uint32_t rank) {
        __syncthreads();
        if (threadIdx.x == 0) s.first = 0;
        __syncthreads();
        const int i = threadIdx.x;
        if (i < kBins && s.count[i]) {
            const bool here = ask == kRank ? s.sum_count[i] >= rank : is(ask, s.below[i], target);
            const bool before = i > 0 && (ask == kRank ? s.sum_count[i - 1] >= rank : s.sum_count[i - 1] > 0 && is(ask, s.below[i - 1], target));
            // an order of its own for the last one: it stands where nothing is found
            if (!before && (here || s.sum_count[i] == s.sum_count[kBins - 1])) s.first = i;
        }
        __syncthreads();
        return s.first;
    }

    // The token that is asked for within a bin that holds it: its order, and the weight of the tokens up to and with it.
    __device__ uint64_t within(int bin, Ask ask, double target, uint32_t rank, double& running) {
        const double base = bin ? s.below[bin - 1] : 0.0, one = unit(bin);
        const uint32_t rank_base = bin ? s.sum_count[bin - 1] : 0;
        __syncthreads();
        if (threadIdx.x == 0) {
            s.lo = 0, s.hi = ~0ull;
            s.above_weight = 0, s.above_count = 0;
        }
        __syncthreads();
        for (;;) {
            // the range's first and last token
            const uint64_t lo = s.lo, hi = s.hi;
            uint64_t least = ~0ull, most = 0;
            __syncthreads();
            if (threadIdx.x == 0) s.lo = ~0ull, s.hi = 0;
            s.sub_weight[threadIdx.x] = 0;
            s.sub_count[threadIdx.x] = 0;
            __syncthreads();
            each(bin, [&](uint64_t o, uint64_t) {
                if (o >= lo && o <= hi) least = o < least ? o : least, most = o > most ? o : most;
            });
            if (least <= most) {
                atomicMin(&s.lo, static_cast<unsigned long long>(least));
                atomicMax(&s.hi, static_cast<unsigned long long>(most));
            }
            __syncthreads();
            const uint64_t from = s.lo, to = s.hi;
            if (from >= to) break;
            const uint64_t span = to - from;
            const int shift = max(0, 64 - __clzll(static_cast<long long>(span)) - 10);
            each(bin, [&](uint64_t o, uint64_t w) {
                if (o >= from && o <= to) {
                    const uint32_t i = static_cast<uint32_t>((o - from) >> shift);
                    atomicAdd(reinterpret_cast<unsigned long long*>(&s.sub_weight[i]), static_cast<unsigned long long>(w));
                    atomicAdd(&s.sub_count[i], 1u);
                }
            });
            __syncthreads();
            uint64_t w = s.sub_weight[threadIdx.x];
            uint32_t n = s.sub_count[threadIdx.x];
            const uint64_t own_w = w;
            const uint32_t own_n = n;
            scan(w, n);
            w += s.above_weight;
            n += s.above_count;
            const bool here = ask == kRank ? rank_base + n >= rank : is(ask, base + static_cast<double>(w) * one, target);
            const bool before = ask == kRank ? rank_base + n - own_n >= rank
                                             : n - own_n > s.above_count && is(ask, base + static_cast<double>(w - own_w) * one, target);
            __syncthreads();
            const int last = static_cast<int>(span >> shift);
            const bool mine = own_n && !before && (here || static_cast<int>(threadIdx.x) == last);
            if (mine) {
                const uint64_t begin = from + (static_cast<uint64_t>(threadIdx.x) << shift);
                s.lo = begin;
                s.hi = (to - begin) >> shift ? begin + ((1ull << shift) - 1) : to;
                s.above_weight = w - own_w;
                s.above_count = n - own_n;
            }
            __syncthreads();
        }
        const uint64_t o = s.lo;
        double x;
        scale.bin(logit_of(o), x);
        running = base + static_cast<double>(s.above_weight + weight(x)) * one;
        return o;
    }

    // inclusive sums over the workgroup's threads
    __device__ __forceinline__ void scan(uint64_t& w, uint32_t& n) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint64_t u = __shfl_up(static_cast<unsigned long long>(w), d, 64);
            const uint32_t m = __shfl_up(n, d, 64);
            if (lane >= d) w += u, n += m;
        }
        if (lane == 63) s.wave_sum[wave] = w, s.wave_count[wave] = n;
        __syncthreads();
        for (int i = 0; i < wave; ++i) w += s.wave_sum[i], n += s.wave_count[i];
        __syncthreads();
    }
};

template <int C>
__global__ __launch_bounds__(kThreads) void pick_kernel(Args a) {
    __shared__ Shared s;
    const int row = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
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
    Row<C> r{a, s, a.logits + row * a.row_bytes, Scale(top, temperature), false};

    // counts and weights of the bins, and their running sums
    for (int c = threadIdx.x; c < a.chunks; c += kThreads) {
        const float t = as_f(tops[c].x);
        double under = kBins;
        if (t == top) under = 0.0;
        else if (t > -__builtin_inff() && top < __builtin_inff()) under = fmin(under, r.scale.top_bin - Scale(t, temperature).top_bin);
        s.under[c] = static_cast<uint16_t>(under);
    }
    __syncthreads();
    uint64_t w = 0;
    uint32_t n = 0;
    if (threadIdx.x < kBins) {
        const uint64_t* bins = a.bins + static_cast<int64_t>(row) * a.chunks * kBins;
#pragma unroll 8
        for (int c = 0; c < a.chunks; ++c) {
            const int i = static_cast<int>(threadIdx.x) - s.under[c];
            const uint64_t x = i >= 0 ? bins[static_cast<int64_t>(c) * kBins + i] : 0;
            w += x & 0xffffffffffffull;
            n += static_cast<uint32_t>(x >> 48);
        }
    }
    double f = static_cast<double>(w) * r.unit(threadIdx.x);
    uint32_t m = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const double g = __shfl_up(f, d, 64);
        const uint32_t k = __shfl_up(m, d, 64);
        if (lane >= d) f += g, m += k;
    }
    if (lane == 63) s.wave_weight[wave] = f, s.wave_count[wave] = m;
    __syncthreads();
    for (int i = wave - 1; i >= 0; --i) f += s.wave_weight[i], m += s.wave_count[i];
    if (threadIdx.x < kBins) {
        s.count[threadIdx.x] = n;
        s.sum_count[threadIdx.x] = m;
        s.below[threadIdx.x] = f;
        s.wanted[threadIdx.x] = 0;
    }
    if (threadIdx.x == 0) s.listed = 0;
    __syncthreads();

    const int top_k = a.top_k_of(row);
    const double top_p = a.top_p ? a.top_p[row] : a.top_p_all;
    const double min_p = fmin(a.min_p ? a.min_p[row] : a.min_p_all, 1.0);
    const double u = fmin(fmax(static_cast<double>(a.u[row]), 0.0), 1.0 - 0x1p-25);
    const uint32_t all = s.sum_count[kBins - 1];
    const bool by_k = top_k > 0 && static_cast<uint32_t>(top_k) < all, by_p = top_p < 1.0, by_min = min_p > 0.0;

    // the bins in which the borders can lie: each border's range follows from the one before it
    double low = s.below[kBins - 1], high = low;  // weight that is kept, at least and at most
    double low_k = low, high_k = high;            // the same of top_k alone
    int bin_k = -1, bin_m = -1;
    const auto want = [&](int from, int to) {
        if (static_cast<int>(threadIdx.x) >= from && static_cast<int>(threadIdx.x) <= to) s.wanted[threadIdx.x] = 1;
    };
    if (by_k) {
        bin_k = r.find(kRank, 0.0, top_k);
        low = low_k = bin_k ? s.below[bin_k - 1] : 0.0, high = high_k = s.below[bin_k];
        want(bin_k, bin_k);
    }
    if (by_p) {
        const int from = r.find(kReach, top_p * low, 0), to = r.find(kReach, top_p * high, 0);
        low = fmin(low, from ? s.below[from - 1] : 0.0), high = fmin(high, s.below[to]);
        want(from, to);
    }
    if (by_min) {
        // the last bin with a part at min_p or over it (the one behind that, by rounding, does no harm)
        const double under = ceil(r.scale.top_bin - r.scale.top_at - log(min_p) * kPer);
        bin_m = static_cast<int>(fmin(fmax(under, 0.0), kBins - 1.0));
        low = fmin(low, bin_m ? s.below[bin_m - 1] : 0.0), high = fmin(high, s.below[bin_m]);
        want(bin_m, bin_m);
    }
    want(r.find(kPass, u * low, 0), r.find(kPass, u * high, 0));
    __syncthreads();

    // their tokens
    uint32_t wanted = threadIdx.x < kBins && s.wanted[threadIdx.x] ? n : 0;
    uint64_t unused = 0;
    r.scan(unused, wanted);
    if (threadIdx.x == kThreads - 1) s.above_count = wanted;
    __syncthreads();
    r.whole = s.above_count > kList;
    if (!r.whole) {
        for (int i = threadIdx.x * 8; i < a.vocab; i += kThreads * 8) {
            float v[8];
            load_logits<C>(r.logits, i, a.vocab, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (v[e] == -__builtin_inff()) continue;
                double x;
                const int b = r.scale.bin(v[e], x);
                if (b < kBins && s.wanted[b]) {
                    const uint32_t place = atomicAdd(&s.listed, 1u);
                    if (place < kList) s.list[place] = order_of(v[e], i + e);
                }
            }
        }
    }
    __syncthreads();

    double kept = s.below[kBins - 1];
    if (by_k) {
        double running;
        r.within(bin_k, kRank, 0.0, top_k, running);
        kept = fmin(fmax(running, low_k), high_k);  // (sums of the same in another order)
    }
    const double target = top_p * kept;
    if (by_p) {
        double running;
        r.within(r.find(kReach, target, 0), kReach, target, 0, running);
        kept = fmin(kept, running);
    }
    if (by_min) {
        __syncthreads();
        if (threadIdx.x == 0) s.above_weight = 0;
        __syncthreads();
        r.each(bin_m, [&](uint64_t o, uint64_t weight) {
            const double l = logit_of(o);
            if (o >> 32 == order_of(top, 0) >> 32 || exp((l - static_cast<double>(top)) / temperature) >= min_p)
                atomicAdd(&s.above_weight, static_cast<unsigned long long>(weight));
        });
        __syncthreads();
        kept = fmin(kept, (bin_m ? s.below[bin_m - 1] : 0.0) + static_cast<double>(s.above_weight) * r.unit(bin_m));
    }
    kept = fmin(fmax(kept, low), high);
    double running;
    const uint64_t o = r.within(r.find(kPass, u * kept, 0), kPass, u * kept, 0, running);
    if (threadIdx.x == 0) a.out[row] = static_cast<int64_t>(o & 0xffffffffu);
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
