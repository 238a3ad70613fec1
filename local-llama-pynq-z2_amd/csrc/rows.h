// Rows of activations and codes of 8 bits: device helpers of the caches' kernels (internal header).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "../../include/llm_hip.h"

// Max of non-negative bit patterns over the 16 lanes of a DPP row.
__device__ __forceinline__ uint32_t umax16(uint32_t m) {
    auto get = [](uint32_t v, auto ctrl) {
        return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, decltype(ctrl)::value, 0xF, 0xF, false);
    };
    m = max(m, get(m, std::integral_constant<int, 0xB1>()));
    m = max(m, get(m, std::integral_constant<int, 0x4E>()));
    m = max(m, get(m, std::integral_constant<int, 0x141>()));
    return max(m, get(m, std::integral_constant<int, 0x140>()));
}

template <int RT>
__device__ __forceinline__ float4 row4(const uint8_t *p) { // 4 values
    if constexpr (RT == LLM_F32) return *(const float4 *)p;
    const uint2 u = *(const uint2 *)p;
    return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                       __uint_as_float(u.y & 0xffff0000u));
}
__device__ __forceinline__ uint32_t bf16_pair(float x, float y) { // rounded half to even
    typedef float f2 __attribute__((ext_vector_type(2)));
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){x, y}, b2));
}
// (rows of a cache start at multiples of 4 bytes: a store of that alignment, still one instruction)
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2u __attribute__((ext_vector_type(2), aligned(4)));
template <int RT>
__device__ __forceinline__ void put4(uint8_t *p, float4 v) {
    if constexpr (RT == LLM_F32) *(f32x4u *)p = (f32x4u){v.x, v.y, v.z, v.w};
    else *(u32x2u *)p = (u32x2u){bf16_pair(v.x, v.y), bf16_pair(v.z, v.w)};
}

// x / s (s > 0, both scaled so that no step underflows) rounded to odd: the fp32 quotient that lies towards zero, its last
// bit set where the quotient is not exact.  Rounding that once more to at most 22 bits gives the correctly rounded exact
// quotient, so a value next to a border between two codes gets the right one.
__device__ __forceinline__ float div_to_odd(float x, float s) {
    const float v = x / s, r = fmaf(-v, s, x); // (the remainder of a correctly rounded quotient is exact)
    uint32_t b = __float_as_uint(v);
    if (r != 0.0f && v != 0.0f) {
        if ((__float_as_uint(r) ^ b) >> 31) b -= 1; // the quotient is nearer to zero than v
        b |= 1;
    }
    return __uint_as_float(b);
}
