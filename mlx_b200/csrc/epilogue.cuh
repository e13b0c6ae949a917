// What a product's epilogue does to sums in fp32: the activations of qmatmul_epi and qmatmul_experts.
#pragma once
#include "internal.h"

namespace luxcuda {

// v / (1 + exp(-u)).  exp(-u) = 2^t, t = -u log2(e): the machine's exponential (2 units in the last place) of the rounded t, corrected by what the
// rounding left (beyond 2^126 there is nothing to correct: the quotient is v or 0), then the machine's reciprocal (1): 5 units or so, in ten
// instructions where exp and a division of CUDA's own take forty.
__device__ __forceinline__ float times_sigmoid(float v, float u) {
    constexpr float kLog2e = 1.44269504f, kLn2 = 0.693147181f;
    const float t = u * -kLog2e, lost = fmaf(u, -kLog2e, -t);
    float e, r;
    asm("ex2.approx.f32 %0, %1;" : "=f"(e) : "f"(t));
    if (fabsf(t) < 126.0f) e = fmaf(e, lost * kLn2, e);
    asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    return v * r;
}
// An activation of N sums.  One switch around the loops: the epilogue warps' code shares the instruction caches with all other roles of a GEMM (a
// switch per value, with CUDA's own exponential and hyperbolic tangent, made a 2048 x 4096 x 4096 product without any activation 84 us
// instead of 50).  gelu_tanh: (1 + tanh(z)) / 2 = 1 / (1 + exp(-2z)).
template <int N>
__device__ __forceinline__ void activate(int act, float (&v)[N]) {
    if (act == LUX_CUDA_ACT_NONE) return;
    if (act == LUX_CUDA_ACT_RELU) {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = v[i] < 0.0f ? 0.0f : v[i];
    } else if (act == LUX_CUDA_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = times_sigmoid(v[i], v[i]);
    } else if (act == LUX_CUDA_ACT_GELU_TANH) {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = times_sigmoid(v[i], v[i] * fmaf(0.0713548163f, v[i] * v[i], 1.59576912f));
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = 0.5f * v[i] * (1.0f + erff(v[i] * 0.70710678f));
    }
}
}  // namespace luxcuda
