// exp2_f64.hpp -- probabilities of logits in 64 bits: a short exponential and
// sums over a wavefront.
#pragma once

#include "device_common.hpp"

namespace atlas {

__device__ __forceinline__ float number_or_none(float x) { return x != x ? -__builtin_inff() : x; }

// 2^(y / 32), y <= 0, by 2^(j / 32) from a table in LDS and the Taylor
// polynomial of 2^(r / 32) to the sixth degree, |r| <= 1 / 2: ((r / 32) ln 2)^7 / 7!
// is below 2^-58.  With the rounding of y and of the products, within
// 2^-51 (|y / 32| + 2) of the true value; below 2^-1022 no bits are kept, and from
// 2^-1023 down, and of a y that is no number, it is zero.
//
// Its 64-bit instructions bound the sums of rows of logits (384 rows of 262144
// 68 us without them), so it has few: with the library's exp they took 120 us, as
// plain C 105, so 98 (in the same runs; 101 to 107 in others).  Adding 1.5 2^52
// leaves the nearest whole number of thirty-seconds in the low bits of the sum,
// with 1023 ones more in front; its
// upper part is added to the exponent of a table entry, whose own is taken out;
// and the constants stay in registers, one operand of an instruction a scalar
// one, which the compiler would not hold them in by itself.
struct Exp2 {
    const uint2* table;
    double first, c[5], shift, least;

    static __device__ void fill(uint2 (&table)[32]) {
        if (threadIdx.x < 32) {
            const uint64_t bits = __builtin_bit_cast(uint64_t, exp2(threadIdx.x * (1.0 / 32.0)));
            table[threadIdx.x] = make_uint2(static_cast<uint32_t>(bits), static_cast<uint32_t>(bits >> 32) - (1023u << 20));
        }
    }
    explicit __device__ Exp2(const uint2 (&table)[32])
        : table(table),
          first(0x1.430912f86c787p-13 * 0x1p-30),  // ln2^6 / 720, of 1 / 32 each
          c{0x1.5d87fe78a6731p-10 * 0x1p-25,       // ln2^5 / 120
            0x1.3b2ab6fba4e77p-7 * 0x1p-20,        // ln2^4 / 24
            0x1.c6b08d704a0c0p-5 * 0x1p-15,        // ln2^3 / 6
            0x1.ebfbdff82c58fp-3 * 0x1p-10,        // ln2^2 / 2
            0x1.62e42fefa39efp-1 * 0x1p-5},        // ln2
          shift(0x1.8p52 + 32 * 1023), least(-32.0 * 1023.0) {
        asm("" : "+v"(first));
#pragma unroll
        for (int i = 0; i < 5; ++i) asm("" : "+s"(c[i]));
        asm("" : "+s"(shift), "+s"(least));
    }
    __device__ __forceinline__ double operator()(double y) const {
        y = fmax(y, least);
        const double t = y + shift;
        const double r = y - (t - shift);
        const uint32_t k = static_cast<uint32_t>(__builtin_bit_cast(uint64_t, t));
        double p = first;
#pragma unroll
        for (int i = 0; i < 5; ++i) p = __builtin_fma(p, r, c[i]);
        p = __builtin_fma(p, r, 1.0);
        uint2 power = table[k & 31];
        power.y += k >> 5 << 20;
        return p * __builtin_bit_cast(double, static_cast<uint64_t>(power.y) << 32 | power.x);
    }
};

template <int CTRL, int ROW_MASK, bool BOUND>
__device__ __forceinline__ double dpp_f64(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(u), CTRL, ROW_MASK, 0xf, BOUND);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(u >> 32), CTRL, ROW_MASK, 0xf, BOUND);
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
// Sum over the wavefront in a fixed tree, the result in every lane (the
// steps of wave_sum_tree_f32).
__device__ __forceinline__ double wave_sum_f64(double v) {
    v += dpp_f64<0xb1, 0xf, false>(v);
    v += dpp_f64<0x4e, 0xf, false>(v);
    v += dpp_f64<0x141, 0xf, false>(v);
    v += dpp_f64<0x140, 0xf, false>(v);
    v += __shfl_xor(v, 16, kWave);
    return v + __shfl_xor(v, 32, kWave);
}

}  // namespace atlas
