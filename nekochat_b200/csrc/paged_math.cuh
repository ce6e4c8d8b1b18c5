// Arithmetic that the paged attention kernels share (k_paged_attn.cu, k_paged_prompt.cu).
#pragma once
#include "neko_common.cuh"

namespace neko {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kNoRow = -(1 << 30);  // the position of a place without a row: it sees nothing

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// The smaller of two numbers, NaN where either is one.
__device__ __forceinline__ float min_nan(float x, float y) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
    return r;
}
// tanh(x) = 1 - 2 / (1 + e^2x): absolute error of a few 2^-23, which the cap multiplies; large |x| saturate, NaN stays.
__device__ __forceinline__ float tanh_abs(float x) {
    return 1.0f - __fdividef(2.0f, 1.0f + ex2(min_nan(x * (2.0f * kLog2e), 64.0f)));
}
// tanh of |x| <= 1/2 as an odd polynomial of degree 9 (largest error there: 6.3e-9): no special functions, and exact to the
// last places where tanh_abs is off by a few 2^-23, which a cap of 50 makes 1e-5 of a score.
__device__ __forceinline__ float tanh_small(float x) {
    const float y = x * x;
    float p = fmaf(y, 0.016737453639507294f, -0.05276207625865936f);
    p = fmaf(p, y, 0.13320569694042206f);
    p = fmaf(p, y, -0.3333277702331543f);
    p = fmaf(p, y, 0.9999999403953552f);
    return p * x;
}
__device__ __forceinline__ float finite_abs(float x) {
    const float m = fabsf(x);
    return m <= 3.402823466e38f ? m : 0.0f;
}
// The power of two that brings a row's largest magnitude to [1, 2), or to [2, 4) where that power would be subnormal.
__device__ __forceinline__ float row_up(float most) {
    const int ex = most > 0.0f ? max(int(__float_as_uint(most) >> 23) - 127, -126) : 0;
    return __uint_as_float(uint32_t(min(max(127 - ex, 1), 253)) << 23);
}

// Two f32 operations in one instruction.
__device__ __forceinline__ uint64_t pack2(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void unpack2(uint64_t r, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(r)); }
__device__ __forceinline__ uint64_t fma2(uint64_t x, uint64_t y, uint64_t z) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t x, uint64_t y) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t x, uint64_t y) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    return r;
}
// 1 / sqrt(x), relative error below 2^-22.
__device__ __forceinline__ float rsqrt_near(float x) {
    float y;
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

}  // namespace neko
