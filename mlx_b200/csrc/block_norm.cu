// The row step between two blocks of a model: the norm after a block, its gate, the residual sum, and the norm before the next
// block, in one pass over the data:
//   b  = post(h)                                     none | rms: h / sqrt(mean h^2 + eps) * w | layer: (h - mean) / sqrt(var + eps) * w + c
//   r' = round(res_scale * r + branch_scale * act(gate) * b)
//   o  = pre(r')                                     of the rounded r', so that it is what a call on the stored stream would give
// o leaves as fp32, as bf16, or rounded to bf16 and from there in the microscaled format (mx4.cuh) that the product takes.
//
// HBM-bound: h, r, (gate) read and r', o written once.  A block keeps its row in registers between the statistics; sums of squares,
// means and everything between are fp32, the variance is the mean of squared differences.
#include <algorithm>

#include "internal.h"
#include "mx4.cuh"

namespace luxcuda {

namespace {

constexpr int kMaxThreads = 1024;

__device__ __forceinline__ float act_of(float g, int act) {
    if (act == LUX_CUDA_GATE_SIGMOID) return __fdiv_rn(1.0f, 1.0f + expf(-g));
    if (act == LUX_CUDA_GATE_TANH) return tanhf(g);
    return g;
}
// V neighbouring elements from element i on
template <int V>
__device__ __forceinline__ void load_v(const void* p, bool bf16, bool vec, size_t i, float (&v)[V]) {
    if (V == 8 && vec) {
        if (bf16) {
            const uint4 q = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p) + i);
            const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int j = 0; j < V / 2; j++) {
                v[2 * j] = __uint_as_float(w[j & 3] << 16);
                v[(2 * j + 1) % V] = __uint_as_float(w[j & 3] & 0xFFFF0000u);
            }
        } else {
            const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
#pragma unroll
            for (int j = 0; j < V / 4; j++) {
                const float4 f = q[j];
                v[(4 * j) % V] = f.x; v[(4 * j + 1) % V] = f.y; v[(4 * j + 2) % V] = f.z; v[(4 * j + 3) % V] = f.w;
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; j++) v[j] = bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i + j]) : static_cast<const float*>(p)[i + j];
    }
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t w;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
    return w;
}
template <int V>
__device__ __forceinline__ void store_v(void* p, bool bf16, bool vec, size_t i, const float (&v)[V]) {
    if (V == 8 && vec) {
        if (bf16) {
            uint4 q;
            q.x = pack_bf16(v[0], v[1 % V]); q.y = pack_bf16(v[2 % V], v[3 % V]); q.z = pack_bf16(v[4 % V], v[5 % V]); q.w = pack_bf16(v[6 % V], v[7 % V]);
            *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p) + i) = q;
        } else {
            float4* q = reinterpret_cast<float4*>(static_cast<float*>(p) + i);
#pragma unroll
            for (int j = 0; j < V / 4; j++) q[j] = make_float4(v[(4 * j) % V], v[(4 * j + 1) % V], v[(4 * j + 2) % V], v[(4 * j + 3) % V]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; j++) {
            if (bf16) static_cast<__nv_bfloat16*>(p)[i + j] = __float2bfloat16_rn(v[j]);
            else static_cast<float*>(p)[i + j] = v[j];
        }
    }
}
__device__ __forceinline__ float block_sum(float v, float* red) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();  // (the previous sum has been read)
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    const int warps = blockDim.x >> 5;
    v = (threadIdx.x & 31) < warps ? red[threadIdx.x & 31] : 0.0f;
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// CH chunks of V elements per thread, chunk j of thread t being the row's (j * threads + t)-th; CH = 0: rows longer than the
// registers hold, read again for every step.
template <int V, int CH, int MX>
__global__ void __launch_bounds__(kMaxThreads) block_norm_kernel(const __grid_constant__ BlockNormArgs a) {
    __shared__ float red[32];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int tid = threadIdx.x, T = blockDim.x;
    const size_t dim = a.dim;
    const bool xb = a.x_bf16, rb = a.r_bf16, ob = a.out_bf16;
    const float inv_dim = 1.0f / (float)dim;  // (the mean: one more rounding than a division, of the same size)
    for (size_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const char* h = a.h ? static_cast<const char*>(a.h) + row * a.h_ld * (xb ? 2 : 4) : nullptr;
        const char* gate = a.gate ? static_cast<const char*>(a.gate) + (a.gate_rows ? row / a.gate_rows : 0) * a.gate_ld * (xb ? 2 : 4) : nullptr;
        const char* r = a.r ? static_cast<const char*>(a.r) + row * dim * (rb ? 2 : 4) : nullptr;
        char* r_out = a.r_out ? static_cast<char*>(a.r_out) + row * dim * (rb ? 2 : 4) : nullptr;
        constexpr int NC = CH ? CH : 1;  // chunks that are kept
        const int loops = CH ? CH : (int)((dim / V + T - 1) / T);
        float v[NC][V];
        auto chunk = [&](int j) { return ((size_t)j * T + tid) * V; };
        float mean = 0.0f, inv = 1.0f;
        // the statistics of a norm over the row that values(j, t) gives chunk by chunk
        auto stats = [&](int kind, auto&& values) {
            mean = 0.0f;
            if (kind == LUX_CUDA_NORM_NONE) return;
            float s = 0.0f;
            if (kind == LUX_CUDA_NORM_LAYER) {
#pragma unroll (NC)
                for (int j = 0; j < loops; j++)
                    if (chunk(j) < dim) {
                        float t[V];
                        values(j, t);
#pragma unroll
                        for (int e = 0; e < V; e++) s += t[e];
                    }
                mean = block_sum(s, red) * inv_dim;
                s = 0.0f;
            }
#pragma unroll (NC)
            for (int j = 0; j < loops; j++)
                if (chunk(j) < dim) {
                    float t[V];
                    values(j, t);
#pragma unroll
                    for (int e = 0; e < V; e++) s = fmaf(t[e] - mean, t[e] - mean, s);
                }
            inv = __fdiv_rn(1.0f, sqrtf(fmaf(block_sum(s, red), inv_dim, a.eps)));
        };
        auto norm = [&](int kind, const float* w, const float* c, size_t i, float (&t)[V]) {
            if (kind == LUX_CUDA_NORM_NONE) return;
            float wv[V], cv[V];
            if (w) load_v<V>(w, false, a.w_vec, i, wv);
            if (c) load_v<V>(c, false, a.w_vec, i, cv);
#pragma unroll
            for (int e = 0; e < V; e++) {
                t[e] = (t[e] - mean) * inv;
                if (w) t[e] *= wv[e];
                if (c) t[e] += cv[e];
            }
        };
        // the new stream, rounded to its type
        auto residual = [&](size_t i, float (&t)[V]) {  // t: h of this chunk
            float g[V], rv[V];
            if (h) {
                norm(a.post_kind, a.post_w, a.post_b, i, t);
                if (gate) {
                    load_v<V>(gate, xb, a.gate_vec, i, g);
#pragma unroll
                    for (int e = 0; e < V; e++) t[e] *= act_of(g[e], a.gate_act);
                }
            }
            if (r) load_v<V>(r, rb, a.r_vec, i, rv);
#pragma unroll
            for (int e = 0; e < V; e++) {
                float s = h ? a.branch_scale * t[e] : 0.0f;
                if (r) s = fmaf(a.res_scale, rv[e], s);
                t[e] = rb ? __bfloat162float(__float2bfloat16_rn(s)) : s;
            }
        };
        auto emit = [&](size_t i, float (&t)[V]) {
            if (MX == 0) {
                if (i < dim && a.out) store_v<V>(static_cast<char*>(a.out) + row * dim * (ob ? 2 : 4), ob, a.out_vec, i, t);
            } else {
                // (every lane of the warp is here; lanes past the row carry zeros)
                float u[8];
                uint32_t c[1], byte;
#pragma unroll
                for (int e = 0; e < 8; e++) u[e] = i < dim ? __fmul_rn(__bfloat162float(__float2bfloat16_rn(t[e % V])), a.out_pre) : 0.0f;
                constexpr int F = MX ? MX : 1;
                mx4_encode<F, 8>(u, c, byte);
                const uint32_t word = mx4_scale_word<F, 8>(byte, tid & 31);
                if (i < dim) {
                    static_cast<uint32_t*>(a.out)[(row * dim + i) >> 3] = c[0];
                    if ((tid & 31) % (4 * mx4_block(F) / 8) == 0)
                        *reinterpret_cast<uint32_t*>(a.out_scales + mx4_scale_at(row, (int)(i / (4 * mx4_block(F))), mx4_tiles_k((int)dim, F))) = word;
                }
            }
        };
        auto kept = [&](int j, float (&t)[V]) {
#pragma unroll
            for (int e = 0; e < V; e++) t[e] = v[CH ? j : 0][e];
        };
        auto h_of = [&](int j, float (&t)[V]) { load_v<V>(h, xb, a.h_vec, chunk(j), t); };
        auto r_of = [&](int j, float (&t)[V]) { load_v<V>(r_out, rb, a.r_out_vec, chunk(j), t); };  // what this thread stored
        if (CH) {
            if (h) {
#pragma unroll
                for (int j = 0; j < NC; j++)
                    if (chunk(j) < dim) h_of(j, v[j]);
                stats(a.post_kind, kept);
            }
#pragma unroll
            for (int j = 0; j < NC; j++)
                if (chunk(j) < dim) {
                    residual(chunk(j), v[j]);
                    if (r_out) store_v<V>(r_out, rb, a.r_out_vec, chunk(j), v[j]);
                }
            if (!a.out) continue;
            stats(a.pre_kind, kept);
#pragma unroll
            for (int j = 0; j < NC; j++) {
                if (chunk(j) < dim) norm(a.pre_kind, a.pre_w, a.pre_b, chunk(j), v[j]);
                emit(chunk(j), v[j]);
            }
        } else {
            if (h) stats(a.post_kind, h_of);
            for (int j = 0; j < loops; j++)
                if (chunk(j) < dim) {
                    if (h) h_of(j, v[0]);
                    residual(chunk(j), v[0]);
                    store_v<V>(r_out, rb, a.r_out_vec, chunk(j), v[0]);
                }
            if (!a.out) continue;
            stats(a.pre_kind, r_of);
            for (int j = 0; j < loops; j++) {
                if (chunk(j) < dim) {
                    r_of(j, v[0]);
                    norm(a.pre_kind, a.pre_w, a.pre_b, chunk(j), v[0]);
                }
                emit(chunk(j), v[0]);
            }
        }
    }
}

template <int V, int CH>
const void* pick_mx(int format) {
    if constexpr (V == 8) {
        if (format == LUX_CUDA_MX4_E8M0) return (const void*)block_norm_kernel<V, CH, LUX_CUDA_MX4_E8M0>;
        if (format == LUX_CUDA_MX4_E4M3) return (const void*)block_norm_kernel<V, CH, LUX_CUDA_MX4_E4M3>;
    }
    return (const void*)block_norm_kernel<V, CH, 0>;
}

}  // namespace

// A row's chunks per thread: one or two with up to 1024 threads where rows are few (latency), four where they fill the machine.
bool block_norm_needs_stream(size_t dim) { return dim % 8 ? dim > 16384 : dim > 32768; }

cudaError_t launch_block_norm(const BlockNormArgs& a, int sm_count, cudaStream_t stream, bool overlap_prev) {
    if (!a.rows || !a.dim) return cudaSuccess;
    const bool wide = a.dim % 8 == 0;
    const size_t chunks = wide ? a.dim / 8 : a.dim;
    const void* kern;
    size_t per;
    if (!wide) {
        per = chunks <= 16 * kMaxThreads ? 16 : 0;
        kern = per ? pick_mx<1, 16>(0) : pick_mx<1, 0>(0);
    } else {
        const bool few = a.rows < (size_t)2 * sm_count;
        per = few && chunks <= kMaxThreads ? 1 : few && chunks <= 2 * kMaxThreads ? 2 : chunks <= 4 * kMaxThreads ? 4 : 0;
        kern = per == 1 ? pick_mx<8, 1>(a.out_format) : per == 2 ? pick_mx<8, 2>(a.out_format) : per == 4 ? pick_mx<8, 4>(a.out_format) : pick_mx<8, 0>(a.out_format);
    }
    const size_t threads = per ? std::min<size_t>(kMaxThreads, ((chunks + per - 1) / per + 31) / 32 * 32) : kMaxThreads;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)std::min<size_t>(a.rows, 0x7fffffff));
    cfg.blockDim = dim3((unsigned)threads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = overlap_prev ? 1 : 0;
    void* args[] = {(void*)&a};
    return cudaLaunchKernelExC(&cfg, kern, args);
}

}  // namespace luxcuda
