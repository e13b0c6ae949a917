// Microscaled 4-bit floating point (mx4.cuh): values into the format, and the values that it stands for.
#include <algorithm>

#include "internal.h"
#include "mx4.cuh"

namespace luxcuda {

namespace {

constexpr int kRows = 8;       // rows per block, a warp each
constexpr int kChunk = 512;    // values of a row per warp: 16 per lane
constexpr int kMaxGridY = 65535;

__device__ __forceinline__ void load16(const void* p, bool bf16, bool vec, int left, float (&u)[16]) {
#pragma unroll
    for (int i = 0; i < 16; i++) u[i] = 0.0f;
    if (left <= 0) return;
    if (vec) {
        if (bf16) {
            const uint4* q = static_cast<const uint4*>(p);
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint4 v = __ldcs(q + h);
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    u[8 * h + 2 * i] = __uint_as_float(w[i] << 16);
                    u[8 * h + 2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
                }
            }
        } else {
            const float4* q = static_cast<const float4*>(p);
#pragma unroll
            for (int h = 0; h < 4; h++) {
                const float4 v = __ldcs(q + h);
                u[4 * h] = v.x; u[4 * h + 1] = v.y; u[4 * h + 2] = v.z; u[4 * h + 3] = v.w;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; i++) u[i] = bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]) : static_cast<const float*>(p)[i];
    }
}

// HBM-bound: 4 or 2 bytes read and 0.53 or 0.56 written per value.  A lane takes 16 neighbouring values (a block of 16, or half a
// block of 32), a warp 512 of one row.
template <int FMT, bool BF16>
__global__ void __launch_bounds__(32 * kRows) mx4_quantize_kernel(const void* __restrict__ in, uint32_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                                int rows, int K, size_t ld, float pre, bool vec) {
    // (dependents first: a matmul behind this kernel fetches its weights while the kernel before it still runs; see note_early_chain_launch)
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    constexpr int LPW = 4 * mx4_block(FMT) / 16;  // lanes per scale word
    const int lane = threadIdx.x & 31, tiles_k = mx4_tiles_k(K, FMT);
    const int k = blockIdx.x * kChunk + lane * 16;
    for (size_t row = (size_t)blockIdx.y * kRows + (threadIdx.x >> 5); row < (size_t)rows; row += (size_t)gridDim.y * kRows) {
        float u[16];
        load16(static_cast<const char*>(in) + (row * ld + k) * (BF16 ? 2 : 4), BF16, vec, K - k, u);
#pragma unroll
        for (int i = 0; i < 16; i++) u[i] = __fmul_rn(u[i], pre);
        uint32_t c[2], byte;
        mx4_encode<FMT, 16>(u, c, byte);
        const uint32_t word = mx4_scale_word<FMT, 16>(byte, lane);
        if (k >= K) continue;
        reinterpret_cast<uint2*>(codes)[(row * K + k) >> 4] = make_uint2(c[0], c[1]);
        if (lane % LPW == 0) *reinterpret_cast<uint32_t*>(scales + mx4_scale_at(row, k / (4 * mx4_block(FMT)), tiles_k)) = word;
    }
}

template <int FMT, bool BF16>
__global__ void __launch_bounds__(32 * kRows) mx4_dequantize_kernel(const uint32_t* __restrict__ codes, const uint8_t* __restrict__ scales, void* __restrict__ out,
                                                                  int rows, int K, float post, bool vec) {
    const int lane = threadIdx.x & 31, tiles_k = mx4_tiles_k(K, FMT);
    const int k = blockIdx.x * kChunk + lane * 16;
    if (k >= K) return;
    const int b = k / mx4_block(FMT);
    for (size_t row = (size_t)blockIdx.y * kRows + (threadIdx.x >> 5); row < (size_t)rows; row += (size_t)gridDim.y * kRows) {
        const uint2 c = __ldcs(reinterpret_cast<const uint2*>(codes) + ((row * K + k) >> 4));
        const float s = mx4_scale_value<FMT>(__ldg(scales + mx4_scale_at(row, b >> 2, tiles_k) + (b & 3)));
        float v[16];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float2 p = e2m1x2_value((i < 4 ? c.x : c.y) >> (8 * (i & 3)) & 0xFFu);
            v[2 * i] = __fmul_rn(__fmul_rn(p.x, s), post);  // (code * scale is exact)
            v[2 * i + 1] = __fmul_rn(__fmul_rn(p.y, s), post);
        }
        const size_t at = row * K + k;
        if (BF16) {
            uint32_t w[8];
#pragma unroll
            for (int i = 0; i < 8; i++) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(v[2 * i + 1]), "f"(v[2 * i]));
            if (vec) {
                uint4* o = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(out) + at);
                __stcs(o, make_uint4(w[0], w[1], w[2], w[3]));
                __stcs(o + 1, make_uint4(w[4], w[5], w[6], w[7]));
            } else {
                uint16_t* o = static_cast<uint16_t*>(out) + at;
#pragma unroll
                for (int i = 0; i < 16; i++) o[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
            }
        } else {
            float* o = static_cast<float*>(out) + at;
            if (vec) {
#pragma unroll
                for (int i = 0; i < 4; i++) __stcs(reinterpret_cast<float4*>(o) + i, make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]));
            } else {
#pragma unroll
                for (int i = 0; i < 16; i++) o[i] = v[i];
            }
        }
    }
}

}  // namespace

cudaError_t launch_mx4_quantize(const void* in, uint32_t* codes, uint8_t* scales, int rows, int K, size_t ld, int format, int in_dtype, float pre,
                                cudaStream_t stream, bool overlap_prev) {
    if (!rows) return cudaSuccess;
    const bool bf16 = in_dtype == LUX_DTYPE_BFLOAT16, vec = ((uintptr_t)in & 15) == 0 && ld % (bf16 ? 8 : 4) == 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((K + kChunk - 1) / kChunk, std::min((rows + kRows - 1) / kRows, kMaxGridY));
    cfg.blockDim = dim3(32 * kRows);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = overlap_prev ? 1 : 0;
    auto kern = format == LUX_CUDA_MX4_E8M0 ? (bf16 ? mx4_quantize_kernel<LUX_CUDA_MX4_E8M0, true> : mx4_quantize_kernel<LUX_CUDA_MX4_E8M0, false>)
                                            : (bf16 ? mx4_quantize_kernel<LUX_CUDA_MX4_E4M3, true> : mx4_quantize_kernel<LUX_CUDA_MX4_E4M3, false>);
    return cudaLaunchKernelEx(&cfg, kern, in, codes, scales, rows, K, ld, pre, vec);
}

cudaError_t launch_mx4_dequantize(const uint32_t* codes, const uint8_t* scales, void* out, int rows, int K, int format, int out_dtype, float post,
                                  cudaStream_t stream) {
    if (!rows) return cudaSuccess;
    const bool bf16 = out_dtype == LUX_DTYPE_BFLOAT16, vec = ((uintptr_t)out & 15) == 0;
    const dim3 grid((K + kChunk - 1) / kChunk, std::min((rows + kRows - 1) / kRows, kMaxGridY));
    auto kern = format == LUX_CUDA_MX4_E8M0 ? (bf16 ? mx4_dequantize_kernel<LUX_CUDA_MX4_E8M0, true> : mx4_dequantize_kernel<LUX_CUDA_MX4_E8M0, false>)
                                            : (bf16 ? mx4_dequantize_kernel<LUX_CUDA_MX4_E4M3, true> : mx4_dequantize_kernel<LUX_CUDA_MX4_E4M3, false>);
    kern<<<grid, 32 * kRows, 0, stream>>>(codes, scales, out, rows, K, post, vec);
    return cudaGetLastError();
}

}  // namespace luxcuda
