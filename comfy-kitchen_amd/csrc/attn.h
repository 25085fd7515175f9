// Pieces shared by the attention kernels: 16-bit MFMA wrappers and the operand layouts they use.
//
// Scores are formed transposed, S^T = K Q^T, and so is the output, O^T = V^T P^T: in both a lane's
// column is its query (a head, or a prompt row), so the softmax statistics of that query, and the
// factor its output is rescaled by, are the lane's own; and the scores a lane receives are those
// of the tokens whose values it multiplies next, so P goes from one product to the other without
// leaving its registers.
#pragma once

#include "ckh_common.h"

namespace ckh {
namespace attn {

typedef unsigned v4u __attribute__((ext_vector_type(4)));
typedef unsigned v2u __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.4426950408889634f;

// The power of two that the largest weight is held at, at least: f16 has no normal numbers under 2^-14,
// and many far weights under that may together outweigh the near ones, so its weights sit at 2^7 .. 2^15.
template <int C>
constexpr float kLift = C == CKH_F16 ? 7.0f : 0.0f;

template <int C>
__device__ __forceinline__ v4f mfma16(v4u a, v4u b, v4f c) {
    if constexpr (C == CKH_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

template <int C>
__device__ __forceinline__ v16f mfma32(v4u a, v4u b, v16f c) {
    if constexpr (C == CKH_BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

// Two floats rounded to the 16-bit type, a in the low half.
template <int C>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (C == CKH_BF16) return __builtin_bit_cast(uint32_t, v2bf{static_cast<__bf16>(a), static_cast<__bf16>(b)});
    else return __builtin_bit_cast(uint32_t, v2h{static_cast<_Float16>(a), static_cast<_Float16>(b)});
}

// Codes 2 HI and 2 HI + 1 of a word of E4M3 codes, exactly, in the 16-bit type.
template <int C, bool HI>
__device__ __forceinline__ uint32_t widen_e4m3(uint32_t w) {
    if constexpr (C == CKH_BF16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HI));
    else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HI));
}

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

}  // namespace attn
}  // namespace ckh
