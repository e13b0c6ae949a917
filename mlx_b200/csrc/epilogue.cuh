// What a product's epilogue does to a sum in fp32: activation of qmatmul_epi and qmatmul_experts.
#pragma once
#include "internal.h"

namespace luxcuda {

// expf, erff and tanhf are CUDA's own, a few units in the last place of fp32: far below the one rounding to bf16, and of the order of
// the sum's own error where y is fp32.
__device__ __forceinline__ float activate(int act, float v) {
    switch (act) {
        case LUX_CUDA_ACT_RELU: return v > 0.0f || v != v ? v : 0.0f;
        case LUX_CUDA_ACT_SILU: return v / (1.0f + expf(-v));
        case LUX_CUDA_ACT_GELU: return 0.5f * v * (1.0f + erff(v * 0.70710678f));
        case LUX_CUDA_ACT_GELU_TANH: return 0.5f * v * (1.0f + tanhf(0.79788456f * (v + 0.044715f * v * v * v)));
        default: return v;
    }
}

}  // namespace luxcuda
