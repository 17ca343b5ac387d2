// attention_lanes.hpp -- what the attention kernels share: maxima and sums over
// the lanes that hold one query row.
#pragma once

#include "device_common.hpp"

namespace atlas {

typedef float f32x2_t __attribute__((ext_vector_type(2)));

inline constexpr float kLog2e = 1.44269504088896340736f;

__device__ __forceinline__ float neg_inf() { return -__builtin_inff(); }

// The maximum over lanes that differ in bit 3 / 4 / 5 of their number.
__device__ __forceinline__ float max_xor8(float x) { return fmaxf(x, dpp_f32<0x128, 0xf, false>(x)); }  // row_ror:8
__device__ __forceinline__ float max_xor16(float x) {
    const uint32_t u = __float_as_uint(x);
    const auto p = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
}
__device__ __forceinline__ float max_xor32(float x) {
    const uint32_t u = __float_as_uint(x);
    const auto p = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
}
__device__ __forceinline__ float sum_xor16(float x) {
    const uint32_t u = __float_as_uint(x);
    const auto p = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return __uint_as_float(p[0]) + __uint_as_float(p[1]);
}
__device__ __forceinline__ float sum_xor32(float x) {
    const uint32_t u = __float_as_uint(x);
    const auto p = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __uint_as_float(p[0]) + __uint_as_float(p[1]);
}

}  // namespace atlas
