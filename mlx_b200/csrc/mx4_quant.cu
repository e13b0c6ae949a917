// Microscaled 4-bit floating point (mx4.cuh): values into the format, and the values that it stands for.
#include <algorithm>

#include "internal.h"
#include "mx4.cuh"

namespace luxcuda {

namespace {

constexpr int kWarps = 8;      // per block, a row each at a time
constexpr int kChunk = 512;    // values of a row per warp: 16 per lane
constexpr int kMaxGridY = 65535;

// 16 neighbouring values as they lie; align: 32 or 16 bytes, or less
template <bool BF16>
struct Raw16 {
    Words8 w[BF16 ? 1 : 2];
    __device__ __forceinline__ void load(const void* p, int align) {
#pragma unroll
        for (int h = 0; h < (BF16 ? 1 : 2); h++) {
            const char* s = static_cast<const char*>(p) + 32 * h;
            if (align == 32) {
                w[h] = ld_once_32(s);
            } else if (align == 16) {
                const uint4 a = __ldcs(reinterpret_cast<const uint4*>(s)), b = __ldcs(reinterpret_cast<const uint4*>(s) + 1);
                w[h] = Words8{{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++)
                    w[h].v[i] = BF16 ? (uint32_t)reinterpret_cast<const uint16_t*>(s)[2 * i] | (uint32_t)reinterpret_cast<const uint16_t*>(s)[2 * i + 1] << 16
                                     : reinterpret_cast<const uint32_t*>(s)[i];
            }
        }
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int h = 0; h < (BF16 ? 1 : 2); h++)
#pragma unroll
            for (int i = 0; i < 8; i++) w[h].v[i] = 0;
    }
    __device__ __forceinline__ Pair get(int i) const {  // i = 0 .. 7
        if (BF16) return unpack2(w[0].v[i]);
        return pair_of(w[i >> 2 & (BF16 ? 0 : 1)].v[(2 * i) & 7], w[i >> 2 & (BF16 ? 0 : 1)].v[(2 * i + 1) & 7]);
    }
};

// HBM-bound (4 or 2 bytes read and 0.53 or 0.56 written per value) with the instructions around a value close behind: 11 at E4M3.
// A lane takes 16 neighbouring values (a block of 16, or half a block of 32), a warp 512 of a row.  What hides the memory is the number of
// warps: 32 registers and 64 warps on an SM, one row each, beat two rows each with 32 warps (4096 x 8192, bf16, E4M3: 16.7 us
// against 18.3; four rows: 22.9; one row with 44 registers: 22.3).  Now 16.9 us, 5.1 TB/s; 11008 x 4096 fp32 31.9 us, 6.4 TB/s.
// AHEAD: see mx4_quantize_is_short.
template <int FMT, bool BF16, bool AHEAD>
__global__ void __launch_bounds__(32 * kWarps, 8) mx4_quantize_kernel(const void* __restrict__ in, uint32_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                                    int rows, int K, size_t ld, float pre, int align) {
    // (dependents first: a matmul behind this kernel fetches its weights while the kernel before it still runs; see note_early_chain_launch)
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (!AHEAD) asm volatile("griddepcontrol.wait;" ::: "memory");
    constexpr int LPW = 4 * mx4_block(FMT) / 16;  // lanes per scale word
    const int lane = threadIdx.x & 31, tiles_k = mx4_tiles_k(K, FMT);
    const int k = blockIdx.x * kChunk + lane * 16;
    const Pair pre2 = pair_of(pre, pre);
    for (uint32_t row = blockIdx.y * kWarps + (threadIdx.x >> 5); row < (uint32_t)rows; row += gridDim.y * kWarps) {
        Raw16<BF16> raw;
        if (k < K) raw.load(static_cast<const char*>(in) + (row * ld + k) * (BF16 ? 2 : 4), align);
        else raw.zero();
        Pair v[8];
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = mul2(raw.get(i), pre2);
        uint32_t c[2], byte;
        mx4_encode<FMT, 16>(v, c, byte);
        const uint32_t word = mx4_scale_word<FMT, 16>(k < K ? byte : 0u, lane);  // (a factor that is infinite or NaN leaves one in lanes past the row)
        if (k >= K) continue;
        reinterpret_cast<uint2*>(codes)[((size_t)row * (uint32_t)K + k) >> 4] = make_uint2(c[0], c[1]);
        if (lane % LPW == 0) *reinterpret_cast<uint32_t*>(scales + mx4_scale_at(row, k / (4 * mx4_block(FMT)), tiles_k)) = word;
    }
    // (whoever waits for this kernel relies on all before it having ended, too)
    if (AHEAD) asm volatile("griddepcontrol.wait;" ::: "memory");
}

// HBM-bound, most of it the stores; the same division of the work, but U rows per warp, all of whose loads are under way before the
// first is used (11008 x 4096, bf16: 20.0 us, 5.7 TB/s, against 21.9 row by row; 5003 x 2880, fp32, with 32-byte instead of
// 16-byte stores, which fill a sector: 11.9 against 19.3).
template <int FMT, bool BF16, int U>
__global__ void __launch_bounds__(32 * kWarps) mx4_dequantize_kernel(const uint32_t* __restrict__ codes, const uint8_t* __restrict__ scales, void* __restrict__ out,
                                                                   int rows, int K, float post, bool aligned) {
    const int lane = threadIdx.x & 31, tiles_k = mx4_tiles_k(K, FMT);
    const int k = blockIdx.x * kChunk + lane * 16;
    if (k >= K) return;
    const int b = k / mx4_block(FMT);
    const Pair post2 = pair_of(post, post);
    for (size_t row0 = (size_t)blockIdx.y * (kWarps * U) + (threadIdx.x >> 5); row0 < (size_t)rows; row0 += (size_t)gridDim.y * (kWarps * U)) {
        uint2 c[U];
        uint32_t byte[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const size_t row = min(row0 + u * kWarps, (size_t)rows - 1);
            c[u] = __ldcs(reinterpret_cast<const uint2*>(codes) + ((row * K + k) >> 4));
            byte[u] = __ldg(scales + mx4_scale_at(row, b >> 2, tiles_k) + (b & 3));
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const size_t row = row0 + u * kWarps, at = row * K + k;
            if (row >= (size_t)rows) break;
            const float s = mx4_scale_value<FMT>(byte[u]);
            const Pair s2 = pair_of(s, s);
            Pair v[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float2 p = e2m1x2_value((i < 4 ? c[u].x : c[u].y) >> (8 * (i & 3)) & 0xFFu);
                v[i] = mul2(mul2(pair_of(p.x, p.y), s2), post2);  // (code * scale is exact)
            }
            Words8 w[BF16 ? 1 : 2];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                if (BF16) {
                    w[0].v[i] = pack2(v[i]);
                } else {
                    w[i >> 2 & (BF16 ? 0 : 1)].v[(2 * i) & 7] = (uint32_t)v[i];
                    w[i >> 2 & (BF16 ? 0 : 1)].v[(2 * i + 1) & 7] = (uint32_t)(v[i] >> 32);
                }
            }
            char* o = static_cast<char*>(out) + at * (BF16 ? 2 : 4);
#pragma unroll
            for (int h = 0; h < (BF16 ? 1 : 2); h++) {
                if (aligned) {
                    st_once_32(o + 32 * h, w[h]);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        if (BF16) {
                            reinterpret_cast<uint16_t*>(o)[2 * i] = (uint16_t)w[h].v[i];
                            reinterpret_cast<uint16_t*>(o)[2 * i + 1] = (uint16_t)(w[h].v[i] >> 16);
                        } else {
                            reinterpret_cast<uint32_t*>(o)[8 * h + i] = w[h].v[i];
                        }
                    }
                }
            }
        }
    }
}

dim3 grid_of(int rows, int K, int u) { return dim3((K + kChunk - 1) / kChunk, std::min((rows - 1) / (kWarps * u) + 1, kMaxGridY)); }
// a full wave of warps, a row each
bool many(int rows, int K) { return (long long)rows * K >= 148ll * 64 * kChunk; }

template <int FMT, bool BF16>
cudaError_t quantize(const void* in, uint32_t* codes, uint8_t* scales, int rows, int K, size_t ld, float pre, cudaStream_t stream, bool overlap_prev, bool ahead) {
    const size_t step = ld * (BF16 ? 2 : 4);
    const int align = ((uintptr_t)in | step) % 32 == 0 ? 32 : ((uintptr_t)in | step) % 16 == 0 ? 16 : 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid_of(rows, K, 1);
    cfg.blockDim = dim3(32 * kWarps);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = overlap_prev ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, overlap_prev && ahead ? mx4_quantize_kernel<FMT, BF16, true> : mx4_quantize_kernel<FMT, BF16, false>, in, codes, scales, rows, K, ld,
                              pre, align);
}

template <int FMT, bool BF16>
cudaError_t dequantize(const uint32_t* codes, const uint8_t* scales, void* out, int rows, int K, float post, cudaStream_t stream) {
    constexpr int U = 4;
    const bool aligned = (uintptr_t)out % 32 == 0;
    if (many(rows, K)) mx4_dequantize_kernel<FMT, BF16, U><<<grid_of(rows, K, U), 32 * kWarps, 0, stream>>>(codes, scales, out, rows, K, post, aligned);
    else mx4_dequantize_kernel<FMT, BF16, 1><<<grid_of(rows, K, 1), 32 * kWarps, 0, stream>>>(codes, scales, out, rows, K, post, aligned);
    return cudaGetLastError();
}

}  // namespace

// At work beside the kernel before it, the quantisation costs a run of independent layers hardly anything: 8 of 1 x 4096 x 11008 with their
// products 61.8 us against 71.  But its blocks stay until that kernel has ended: at most one per SM.
bool mx4_quantize_is_short(int rows, int K, int sm_count) {
    const dim3 g = grid_of(rows, K, 1);
    return (long long)g.x * g.y <= sm_count;
}

cudaError_t launch_mx4_quantize(const void* in, uint32_t* codes, uint8_t* scales, int rows, int K, size_t ld, int format, int in_dtype, float pre,
                                cudaStream_t stream, bool overlap_prev, bool ahead) {
    if (!rows) return cudaSuccess;
    auto f = format == LUX_CUDA_MX4_E8M0 ? (in_dtype == LUX_DTYPE_BFLOAT16 ? quantize<LUX_CUDA_MX4_E8M0, true> : quantize<LUX_CUDA_MX4_E8M0, false>)
                                         : (in_dtype == LUX_DTYPE_BFLOAT16 ? quantize<LUX_CUDA_MX4_E4M3, true> : quantize<LUX_CUDA_MX4_E4M3, false>);
    return f(in, codes, scales, rows, K, ld, pre, stream, overlap_prev, ahead);
}

cudaError_t launch_mx4_dequantize(const uint32_t* codes, const uint8_t* scales, void* out, int rows, int K, int format, int out_dtype, float post,
                                  cudaStream_t stream) {
    if (!rows) return cudaSuccess;
    auto f = format == LUX_CUDA_MX4_E8M0 ? (out_dtype == LUX_DTYPE_BFLOAT16 ? dequantize<LUX_CUDA_MX4_E8M0, true> : dequantize<LUX_CUDA_MX4_E8M0, false>)
                                         : (out_dtype == LUX_DTYPE_BFLOAT16 ? dequantize<LUX_CUDA_MX4_E4M3, true> : dequantize<LUX_CUDA_MX4_E4M3, false>);
    return f(codes, scales, out, rows, K, post, stream);
}

}  // namespace luxcuda
