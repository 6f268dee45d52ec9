// Weights of a softmax as powers of two by the hardware's exponential, and score caps made of them (shared_attention.cu, paged_attention.cu).
#pragma once

namespace {

__device__ __forceinline__ float sa_ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// cap * tanh(s / cap), from the definition 1 - 2 / (e^2x + 1) and, where that cancels, the series to x^9 (the next term is below 2^-26 of the value there).  Sixteen
// tanhf of a thread took 3700 clocks a tile.
__device__ __forceinline__ float sa_capped(float s, float cap, float inv_cap) {
    const float x = fabsf(s * inv_cap), x2 = x * x;
    const float series = fmaf(x * x2, fmaf(x2, fmaf(x2, fmaf(x2, 62.0f / 2835.0f, -17.0f / 315.0f), 2.0f / 15.0f), -1.0f / 3.0f), x);
    const float far = 1.0f - __fdividef(2.0f, sa_ex2(x * (2.0f * kLog2e)) + 1.0f);
    return copysignf(cap * (x < 0.25f ? series : x > 10.0f ? 1.0f : far), s);
}

}  // namespace
