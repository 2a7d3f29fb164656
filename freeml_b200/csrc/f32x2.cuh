// Two fp32 operations in one instruction (sm_100 packed arithmetic).
#pragma once

#include <stdint.h>

namespace fml {

__device__ __forceinline__ uint64_t f32x2_bits(float2 a) { return *reinterpret_cast<const uint64_t*>(&a); }

// a b + c
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c)
{
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(f32x2_bits(a)), "l"(f32x2_bits(b)), "l"(f32x2_bits(c)));
    return *reinterpret_cast<float2*>(&d);
}

__device__ __forceinline__ float2 mul2(float2 a, float2 b)
{
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(f32x2_bits(a)), "l"(f32x2_bits(b)));
    return *reinterpret_cast<float2*>(&d);
}

__device__ __forceinline__ float2 add2(float2 a, float2 b)
{
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(f32x2_bits(a)), "l"(f32x2_bits(b)));
    return *reinterpret_cast<float2*>(&d);
}

}  // namespace fml
