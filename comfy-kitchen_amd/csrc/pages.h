// Where a token's rows lie in a key-value cache held in pages.
#pragma once

#include "ckh_common.h"

namespace ckh {
namespace pages {

typedef unsigned v4u __attribute__((ext_vector_type(4)));
typedef unsigned v2u __attribute__((ext_vector_type(2)));

// The byte offset of a slot, or -1.
struct Slots {
    const void* at;
    bool wide;  // int64 slots
    int64_t count;
    FastDiv by_page;
    int page_size;
    __device__ __forceinline__ int64_t get(int64_t i) const {
        const int64_t s = wide ? static_cast<const int64_t*>(at)[i] : static_cast<const int*>(at)[i];
        return s >= 0 && s < count ? s : -1;
    }
    __device__ __forceinline__ int64_t offset(int64_t s, int64_t page_stride, int64_t tok_stride) const {
        const uint32_t page = by_page.div(static_cast<uint32_t>(s));
        return page * page_stride + static_cast<int64_t>(static_cast<uint32_t>(s) - page * page_size) * tok_stride;
    }
};

struct Strides {  // bytes
    int64_t page, tok, head;
};

}  // namespace pages
}  // namespace ckh
