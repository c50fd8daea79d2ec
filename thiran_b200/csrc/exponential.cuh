// Exponentials of the softmax losses, two values at a time where the
// arithmetic allows (packed f32x2 instructions round each half as the scalar
// ones do).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace thb {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// 2^x with a relative error of about 2^-22; results under 2^-126 become 0.
__device__ __forceinline__ float pow2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
    return reinterpret_cast<float2&>(r);
}

__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
    return reinterpret_cast<float2&>(r);
}

// 2^((x - shift) c) of both halves. The difference is taken first: it is
// exact for near values, and stays finite for the type's lowest value.
__device__ __forceinline__ float2 pow2Shifted(float2 x, float minusShift, float c) {
    const float2 t = mul2(add2(x, make_float2(minusShift, minusShift)), make_float2(c, c));
    return make_float2(pow2(t.x), pow2(t.y));
}

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(r)
        : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)), "l"(reinterpret_cast<uint64_t&>(c)));
    return reinterpret_cast<float2&>(r);
}

} // namespace thb
