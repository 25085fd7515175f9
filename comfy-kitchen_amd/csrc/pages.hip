// Moving tokens in a key-value cache held in pages, for gfx950.  A slot is a token's place in the
// cache, page * page_size + row; a token's row is kv_heads runs of head_dim elements in K and in V.
//
//   write  keys and values of new tokens [tokens, kv_heads, head_dim] to their slots, as they are
//          or as E4M3 codes of x / scale
//   copy   rows from slots to slots, in every layer's K and V at once: the partly filled pages of
//          forked sequences, whole pages, the kept tokens of compacted sequences
//
// Both are bound by the bytes they move.  A thread moves a 16-byte piece of K and one of V, whose
// places it finds once; consecutive threads take consecutive pieces of a row and then of the next
// row, so every wave reads and writes whole lines.  A slot outside the cache is skipped.
//
// copy reads and writes past the caches (nontemporal): what is moved is not read again before
// much else is.  6001 rows of 2 KB, K and V of 20 layers (983 MB): 174 us, 5.7 TB/s; 195 with
// ordinary accesses.  write stores past the caches too (32000 tokens, 262 MB: 48.3 us, 51.3 without)
// but reads its keys and values through them, where the prompt's attention finds them.  More pieces a thread are slower (two layers' 187, four pieces of a row's
// K or V 185).
#include "pages.h"

namespace ckh {
namespace pages {

struct WriteArgs {
    const uint8_t* x[2];
    uint8_t* cache[2];
    const float* scale[2];
    int64_t x_tok[2], x_head[2];
    Strides to[2];
    Slots slots;
    int64_t pieces;  // of all tokens
    FastDiv by_row, by_head;
    int row, head;  // pieces of a row and of a head
};

// XC: type of x; F8: the cache takes E4M3 codes (else x's type).  A piece is 8 elements of x.
template <int XC, bool F8>
__global__ __launch_bounds__(256) void write_kernel(WriteArgs a) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= a.pieces) return;
    const uint32_t tok = a.by_row.div(static_cast<uint32_t>(i)), in = static_cast<uint32_t>(i) - tok * a.row;
    const uint32_t head = a.by_head.div(in), piece = in - head * a.head;
    const int64_t slot = a.slots.get(tok);
    v4u x[2];
#pragma unroll
    for (int n = 0; n < 2; ++n)
        x[n] = *reinterpret_cast<const v4u*>(a.x[n] + tok * a.x_tok[n] + head * a.x_head[n] + piece * 16);
    if (slot < 0) return;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        uint8_t* to = a.cache[n] + a.slots.offset(slot, a.to[n].page, a.to[n].tok) + head * a.to[n].head;
        if constexpr (!F8) {
            __builtin_nontemporal_store(x[n], reinterpret_cast<v4u*>(to + piece * 16));
        } else {
            const float s = a.scale[n] ? *a.scale[n] : 1.0f;
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t h = (x[n][e >> 1] >> (16 * (e & 1))) & 0xffffu;
                f[e] = __fdiv_rn(XC == CKH_BF16 ? bf16_to_f(h) : f16_to_f(h), s);
                f[e] = is_nan(f[e]) ? f[e] : fminf(fmaxf(f[e], -448.0f), 448.0f);
            }
            *reinterpret_cast<v2u*>(to + piece * 8) = v2u{hw_e4m3x4(f[0], f[1], f[2], f[3]), hw_e4m3x4(f[4], f[5], f[6], f[7])};
        }
    }
}

struct CopyArgs {
    uint8_t* cache[2];
    Strides st[2];
    int64_t layer[2];
    Slots src, dst;
    uint32_t pieces;  // of all rows of one layer
    FastDiv by_row, by_head;
    int row, head;
};

__global__ __launch_bounds__(256) void copy_kernel(CopyArgs a) {
    const uint32_t i = blockIdx.x * 256u + threadIdx.x;
    if (i >= a.pieces) return;
    const uint32_t row = a.by_row.div(i), in = i - row * a.row;
    const uint32_t head = a.by_head.div(in), piece = in - head * a.head;
    const int64_t s = a.src.get(row), d = a.dst.get(row);
    if (s < 0 || d < 0) return;
    v4u x[2];
    uint8_t* to[2];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        const Strides st = a.st[n];
        uint8_t* cache = a.cache[n] + blockIdx.y * a.layer[n] + head * st.head + piece * 16;
        x[n] = __builtin_nontemporal_load(reinterpret_cast<const v4u*>(cache + a.src.offset(s, st.page, st.tok)));
        to[n] = cache + a.dst.offset(d, st.page, st.tok);
    }
#pragma unroll
    for (int n = 0; n < 2; ++n) __builtin_nontemporal_store(x[n], reinterpret_cast<v4u*>(to[n]));
}

}  // namespace pages
}  // namespace ckh

using namespace ckh;

extern "C" int ckh_paged_write(const void* key, const void* value, void* k_cache, void* v_cache, const void* slots,
                               const void* k_scale, const void* v_scale, int64_t tokens, int64_t kv_heads, int64_t dim,
                               int64_t pages, int64_t page_size, const int64_t* strides, int x_code, int cache_code,
                               int wide_slots, uintptr_t stream) {
    CKH_REQUIRE(x_code == CKH_F16 || x_code == CKH_BF16, "paged_write: unsupported dtype %d", x_code);
    CKH_REQUIRE(cache_code == x_code || cache_code == CKH_E4M3, "paged_write: cache dtype %d with dtype %d", cache_code, x_code);
    CKH_REQUIRE(tokens >= 0 && kv_heads >= 0 && dim > 0 && dim % 16 == 0, "paged_write: head_dim %lld is not a multiple of 16",
                static_cast<long long>(dim));
    CKH_REQUIRE(pages > 0 && page_size > 0 && pages <= INT32_MAX && page_size <= INT32_MAX && pages * page_size <= INT32_MAX,
                "paged_write: %lld pages of %lld tokens", static_cast<long long>(pages), static_cast<long long>(page_size));
    CKH_REQUIRE(cache_code == CKH_E4M3 || (!k_scale && !v_scale), "paged_write: scales with a cache of dtype %d", cache_code);
    const int64_t row = kv_heads * dim / 8;
    CKH_REQUIRE(kv_heads <= 65535 && dim <= 65536 && tokens * row < INT32_MAX, "paged_write: too many elements");
    if (tokens * row == 0) return CKH_OK;
    CKH_REQUIRE(key && value && k_cache && v_cache && slots && strides, "paged_write: null pointer");
    const int es = cache_code == CKH_E4M3 ? 1 : 2;
    // key: token, head; value: token, head; k: page, token, head; v: page, token, head (elements)
    for (int i = 0; i < 10; ++i)
        CKH_REQUIRE(strides[i] >= 0 && strides[i] * (i < 4 ? 2 : es) % 16 == 0, "paged_write: stride %d (%lld) is not a multiple of 16 bytes",
                    i, static_cast<long long>(strides[i]));
    CKH_REQUIRE(aligned(key, 16) && aligned(value, 16) && aligned(k_cache, 16) && aligned(v_cache, 16) &&
                    aligned(slots, wide_slots ? 8 : 4) && aligned(k_scale, 4) && aligned(v_scale, 4),
                "paged_write: misaligned pointer");
    pages::WriteArgs a{};
    for (int n = 0; n < 2; ++n) {
        a.x[n] = static_cast<const uint8_t*>(n ? value : key);
        a.cache[n] = static_cast<uint8_t*>(n ? v_cache : k_cache);
        a.scale[n] = static_cast<const float*>(n ? v_scale : k_scale);
        a.x_tok[n] = strides[2 * n] * 2, a.x_head[n] = strides[2 * n + 1] * 2;
        a.to[n] = {strides[4 + 3 * n] * es, strides[5 + 3 * n] * es, strides[6 + 3 * n] * es};
    }
    a.slots = {slots, wide_slots != 0, pages * page_size, fast_div(static_cast<uint32_t>(page_size)), static_cast<int>(page_size)};
    a.pieces = tokens * row;
    a.row = static_cast<int>(row), a.head = static_cast<int>(dim / 8);
    a.by_row = fast_div(a.row), a.by_head = fast_div(a.head);
    const unsigned grid = static_cast<unsigned>(cdiv(a.pieces, 256));
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (es == 2) pages::write_kernel<CKH_BF16, false><<<grid, 256, 0, st>>>(a);  // 16 bits are moved as they are
    else if (x_code == CKH_BF16) pages::write_kernel<CKH_BF16, true><<<grid, 256, 0, st>>>(a);
    else pages::write_kernel<CKH_F16, true><<<grid, 256, 0, st>>>(a);
    return check_launch("paged_write");
}

extern "C" int ckh_paged_copy(void* k_cache, void* v_cache, const void* src, const void* dst, int64_t layers, int64_t rows,
                              int64_t kv_heads, int64_t dim, int64_t pages, int64_t page_size, const int64_t* strides,
                              int element_bytes, int wide_slots, uintptr_t stream) {
    CKH_REQUIRE(element_bytes == 1 || element_bytes == 2 || element_bytes == 4, "paged_copy: elements of %d bytes", element_bytes);
    CKH_REQUIRE(layers >= 0 && layers <= 65535 && rows >= 0 && kv_heads >= 0 && kv_heads <= 65535 && dim > 0 && dim <= 65536 &&
                    dim * element_bytes % 16 == 0,
                "paged_copy: %lld layers, %lld heads of %lld elements (a head must be a multiple of 16 bytes)",
                static_cast<long long>(layers), static_cast<long long>(kv_heads), static_cast<long long>(dim));
    CKH_REQUIRE(pages > 0 && page_size > 0 && pages <= INT32_MAX && page_size <= INT32_MAX && pages * page_size <= INT32_MAX,
                "paged_copy: %lld pages of %lld tokens", static_cast<long long>(pages), static_cast<long long>(page_size));
    const int64_t head = dim * element_bytes / 16, row = kv_heads * head;
    CKH_REQUIRE(row <= INT32_MAX && rows <= INT32_MAX && rows * row < INT32_MAX - 1024, "paged_copy: too many elements");
    if (layers * rows * row == 0) return CKH_OK;
    CKH_REQUIRE(k_cache && v_cache && src && dst && strides, "paged_copy: null pointer");
    // k: layer, page, token, head; v: layer, page, token, head (elements)
    for (int i = 0; i < 8; ++i)
        CKH_REQUIRE(strides[i] >= 0 && strides[i] * element_bytes % 16 == 0, "paged_copy: stride %d (%lld) is not a multiple of 16 bytes",
                    i, static_cast<long long>(strides[i]));
    CKH_REQUIRE(aligned(k_cache, 16) && aligned(v_cache, 16) && aligned(src, wide_slots ? 8 : 4) && aligned(dst, wide_slots ? 8 : 4),
                "paged_copy: misaligned pointer");
    pages::CopyArgs a{};
    for (int n = 0; n < 2; ++n) {
        a.cache[n] = static_cast<uint8_t*>(n ? v_cache : k_cache);
        a.layer[n] = strides[4 * n] * element_bytes;
        a.st[n] = {strides[4 * n + 1] * element_bytes, strides[4 * n + 2] * element_bytes, strides[4 * n + 3] * element_bytes};
    }
    a.src = {src, wide_slots != 0, pages * page_size, fast_div(static_cast<uint32_t>(page_size)), static_cast<int>(page_size)};
    a.dst = a.src;
    a.dst.at = dst;
    a.pieces = static_cast<uint32_t>(rows * row);
    a.row = static_cast<int>(row), a.head = static_cast<int>(head);
    a.by_row = fast_div(a.row), a.by_head = fast_div(a.head);
    const dim3 grid(static_cast<unsigned>(cdiv(a.pieces, 256)), static_cast<unsigned>(layers));
    pages::copy_kernel<<<grid, 256, 0, reinterpret_cast<hipStream_t>(stream)>>>(a);
    return check_launch("paged_copy");
}
