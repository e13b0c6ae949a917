// What a product's epilogue does to sums in fp32: the activations of qmatmul_epi and qmatmul_experts.
#pragma once
#include "internal.h"

namespace luxcuda {

// v / (1 + exp(-u)).  exp(-u) = 2^t, t = -u log2(e): the machine's exponential (off by 4 U at most, U = 2^-24) of the rounded t, corrected by what the
// rounding left (beyond 2^126 there is nothing to correct: the quotient is v or 0), then the machine's reciprocal (2 U).  With the other roundings 9 U at
// most, and 0.23 U |u| where u < 0, since log2(e) has 24 bits (met: 5.9 U down to u = -13), in ten instructions where exp and a division of CUDA's own take forty.
__device__ __forceinline__ float times_sigmoid(float v, float u) {
    constexpr float kLog2e = 1.44269504f, kLn2 = 0.693147181f;
    const float t = u * -kLog2e, lost = fmaf(u, -kLog2e, -t);
    float e, r;
    asm("ex2.approx.f32 %0, %1;" : "=f"(e) : "f"(t));
    if (fabsf(t) < 126.0f) e = fmaf(e, lost * kLn2, e);
    asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    return v * r;
}
// The normal distribution, (1 + erf(v / sqrt 2)) / 2 = T(-v), T(a) = erfc(a / sqrt 2) / 2 = 1 - T(-a); 1 + erf would lose what the two have in common, at v = -5
// all but four bits.  For a >= 0, T(a) = exp(-a^2 / 2) k h(k) with k = 1 / (1 + 121/256 a): h is smooth down to k = 0, and a polynomial of degree 8
// has it to 1.2 U of itself (least squares, weighted towards the largest error, for a up to 13.5, where T is no normal number any more).  With all
// roundings 5.4 U + 1.1 U a^2 (the exponent's); the machine's exponential and reciprocal add 7.4 U at most (met, over 8 million values: 7.6 U above v = -2).  Fewer
// instructions than 1 + erff: 777 x 2880 x 5003 28.8 us against 31.1; with erfcf, which has two branches, 39.6.
__device__ __forceinline__ float normal_cdf(float v) {
    float k, e;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(k) : "f"(fmaf(fabsf(v), 0.47265625f, 1.0f)));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(v * v * -0.72134751f));
    float h = 0.0491005369f;
    h = fmaf(h, k, -0.264752924f);
    h = fmaf(h, k, 0.567046583f);
    h = fmaf(h, k, -0.554204941f);
    h = fmaf(h, k, 0.160714924f);
    h = fmaf(h, k, 0.0112647489f);
    h = fmaf(h, k, 0.154359177f);
    h = fmaf(h, k, 0.187884957f);
    h = fmaf(h, k, 0.18858692f);
    const float t = h * k * e;
    return v > 0.0f ? 1.0f - t : t;
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
        for (int i = 0; i < N; i++) v[i] = v[i] * normal_cdf(v[i]);
    }
}
}  // namespace luxcuda
