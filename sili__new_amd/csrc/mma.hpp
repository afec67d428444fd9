// mma.hpp -- products on the bf16 matrix cores, with E2M1 codes and with values
// in bf16 parts.
#pragma once

#include "common.hpp"

namespace sili {

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(2))) float f32x2;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;

typedef __attribute__((ext_vector_type(16))) float f32x16;

__device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ uint32_t pack_bf16(float x, float y) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){x, y}, bf16x2));
}
__device__ __forceinline__ float bf16_lo(uint32_t w) { return __builtin_bit_cast(float, w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __builtin_bit_cast(float, w & 0xFFFF0000u); }
// Two codes (byte SEL of w) to bf16.
template <int SEL>
__device__ __forceinline__ uint32_t codes(uint32_t w) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, SEL));
}
// Eight codes of a dword: eight consecutive channels.
__device__ __forceinline__ u32x4 codes8(uint32_t w) { return (u32x4){codes<0>(w), codes<1>(w), codes<2>(w), codes<3>(w)}; }
// bf16 parts of q: 24 bits of fp32, all 11 of f16, all 8 of bf16.
template <typename T>
constexpr int q_parts() { return sizeof(T) == 4 ? 3 : __is_same(T, __bf16) ? 1 : 2; }
// x, y in N parts: part k the bf16 nearest to what the parts before leave.
template <int N>
__device__ __forceinline__ void split_bf16(float x, float y, uint32_t (&part)[N]) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
        part[k] = pack_bf16(x, y);
        x -= bf16_lo(part[k]);
        y -= bf16_hi(part[k]);
    }
}

// The part of this lane's column: take[k] is all ones for part k's columns.
template <int N>
__device__ __forceinline__ uint32_t pick(const uint32_t (&part)[N], const uint32_t (&take)[N]) {
    uint32_t w = part[0] & take[0];
#pragma unroll
    for (int k = 1; k < N; ++k) w |= part[k] & take[k];
    return w;
}

}  // namespace sili
