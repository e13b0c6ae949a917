// The row step between two blocks of a model: the norm after a block, its gate, the residual sum, and the norm before the next
// block, in one pass over the data:
//   b  = post(h)                                     none | rms: h / sqrt(mean h^2 + eps) * w | layer: (h - mean) / sqrt(var + eps) * w + c
//   r' = round(res_scale * r + branch_scale * act(gate) * b)
//   o  = pre(r')                                     of the rounded r', so that it is what a call on the stored stream would give
// o leaves as fp32, as bf16, or rounded to bf16 and from there in the microscaled format (mx4.cuh) that the product takes.
//
// HBM-bound: h, r, (gate) read and r', o written once.  A group of threads takes a row, asks for all of it at once and keeps it in
// registers between the statistics, which are fp32 sums over threads, lanes and warps; the variance is the mean of squared differences.
#include <algorithm>

#include "internal.h"
#include "mx4.cuh"
#include "pair.cuh"

namespace luxcuda {

namespace {

__device__ __forceinline__ float act_of(float g, int act) {
    if (act == LUX_CUDA_GATE_SIGMOID) {
        // 1 / (1 + 2^t), t = -g / ln 2 in two pieces, so that a large g costs no accuracy; at a third of what expf and an exact
        // reciprocal issue, which were a quarter of the kernel
        const float c_hi = -1.44269504f, c_lo = -1.92596299e-8f;  // -1 / ln 2
        const float t = g * c_hi, lo = fmaf(g, c_lo, fmaf(g, c_hi, -t));
        float e, d;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
        e = fmaf(e, lo * 0.693147181f, e);
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(d) : "f"(1.0f + e));
        return d;
    }
    if (act == LUX_CUDA_GATE_TANH) return tanhf(g);
    return g;
}
__device__ __forceinline__ float round_bf16(float v) { return __bfloat162float(__float2bfloat16_rn(v)); }
// rows are read once and their results not again here: neither stays in L1, where the weights are
__device__ __forceinline__ uint4 ld_row(const void* p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ void st_row(void* p, const uint4& v) {
    asm volatile("st.global.L1::no_allocate.v4.u32 [%0], {%1,%2,%3,%4};" ::"l"(p), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
// A thread's eight elements of a chunk: neighbours, on a 16-byte boundary (kWide: kFull where no chunk is cut off by the row's end),
// or, on any boundary, `step` apart, those at `end` and behind it zero (kApart).
enum Mode { kWide, kFull, kApart };
struct Place {
    uint32_t first, step, end;
};
template <bool BF16, int MODE>
struct Raw {
    uint4 q[BF16 ? 1 : 2];
    __device__ __forceinline__ void load(const char* row, const Place& p) {
        if constexpr (MODE != kApart) {
            const char* s = row + (size_t)p.first * (BF16 ? 2 : 4);
            q[0] = ld_row(s);
            if (!BF16) q[BF16 ? 0 : 1] = ld_row(s + 16);
        } else {
            uint32_t w[8];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const uint32_t i = p.first + e * p.step;
                w[e] = i >= p.end ? 0u : BF16 ? (uint32_t)reinterpret_cast<const uint16_t*>(row)[i] : reinterpret_cast<const uint32_t*>(row)[i];
            }
            if (BF16) {
                q[0] = make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
            } else {
                q[0] = make_uint4(w[0], w[1], w[2], w[3]);
                q[BF16 ? 0 : 1] = make_uint4(w[4], w[5], w[6], w[7]);
            }
        }
    }
    __device__ __forceinline__ Pair get(int i) const {  // i = 0 .. 3
        if (BF16) return unpack2(i == 0 ? q[0].x : i == 1 ? q[0].y : i == 2 ? q[0].z : q[0].w);
        const uint4 t = q[BF16 ? 0 : i >> 1];
        return i & 1 ? pair_of(t.z, t.w) : pair_of(t.x, t.y);
    }
};
template <bool BF16, int MODE>
__device__ __forceinline__ void store8(char* row, const Place& p, const Pair (&v)[4]) {
    if (MODE == kApart) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const uint32_t i = p.first + e * p.step;
            const float x = e & 1 ? hi_of(v[e >> 1]) : lo_of(v[e >> 1]);
            if (i < p.end) {
                if (BF16) reinterpret_cast<__nv_bfloat16*>(row)[i] = __float2bfloat16_rn(x);
                else reinterpret_cast<float*>(row)[i] = x;
            }
        }
    } else if (BF16) {
        st_row(row + (size_t)p.first * 2, make_uint4(pack2(v[0]), pack2(v[1]), pack2(v[2]), pack2(v[3])));
    } else {
#pragma unroll
        for (int h = 0; h < 2; h++)
            st_row(row + (size_t)p.first * 4 + 16 * h, make_uint4((uint32_t)v[2 * h], (uint32_t)(v[2 * h] >> 32), (uint32_t)v[2 * h + 1], (uint32_t)(v[2 * h + 1] >> 32)));
    }
}
template <int MODE>
__device__ __forceinline__ void weights8(const float* w, const Place& p, Pair (&v)[4]) {
    if (MODE == kApart) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const uint32_t i = p.first + 2 * e * p.step, k = i + p.step;
            v[e] = pair_of(i < p.end ? __ldg(w + i) : 0.0f, k < p.end ? __ldg(w + k) : 0.0f);
        }
    } else {
        const ulonglong2 a = __ldg(reinterpret_cast<const ulonglong2*>(w + p.first)), b = __ldg(reinterpret_cast<const ulonglong2*>(w + p.first) + 1);
        v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
    }
}
// What the threads of a row, a warp of its own or the whole block, exchange: two places, used in turn, so that a warp may be a step
// ahead of those that still read.
struct Shared {
    float2 part[2][32];
};
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// every lane gets the contribution of the warp of its number (zeros past the last).  All warps go on with all of them: one warp that
// does, and tells the others, makes two waits of one (2048 x 4096, layer | layer: 51 us against 40).
__device__ __forceinline__ float2 exchange(float2 v, Shared& sh, int& turn) {
    const int lane = threadIdx.x & 31;
    if (lane == 0) sh.part[turn][threadIdx.x >> 5] = v;
    __syncthreads();
    v = lane < (int)(blockDim.x >> 5) ? sh.part[turn][lane] : make_float2(0.0f, 0.0f);
    turn ^= 1;
    return v;
}
__device__ __forceinline__ float row_sum(float v, Shared& sh, int& turn) {
    v = warp_sum(v);
    return blockDim.x == 32 ? v : warp_sum(exchange(make_float2(v, 0.0f), sh, turn).x);
}
struct Stats {
    float mean, squares;
};
// The row's mean and the squared differences from it, in one exchange, from every thread's own mean and squared differences over n
// elements, the same number in all threads: two halves of 2n elements have their means' mean and, besides their own, n/2 times the
// squared difference of the means (Chan, Golub, LeVeque 1979).
__device__ __forceinline__ Stats row_moments(float mean, float squares, int n, float inv_dim, Shared& sh, int& turn) {
    float half = 0.5f * n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1, half *= 2.0f) {
        const float d = __shfl_xor_sync(0xffffffffu, mean, o) - mean;
        squares += __shfl_xor_sync(0xffffffffu, squares, o);
        squares = fmaf(d * d, half, squares);
        mean = fmaf(0.5f, d, mean);
    }
    if (blockDim.x == 32) return Stats{mean, squares};
    const float2 p = exchange(make_float2(mean, squares), sh, turn);
    mean = warp_sum(p.x) * (32 * n * inv_dim);
    const float d = (threadIdx.x & 31) < blockDim.x >> 5 ? p.x - mean : 0.0f;
    return Stats{mean, warp_sum(fmaf(d * d, 32.0f * n, p.y))};
}
__device__ __forceinline__ float inv_root(float squares, float inv_dim, float eps) { return __frsqrt_rn(fmaf(squares, inv_dim, eps)); }

// Rows of up to 8 * CH elements per thread, a multiple of 8, every row on a 16-byte boundary; FULL: exactly so many.  blockDim =
// (threads of a row, rows): several rows only where a row is a warp's.  OUT: 0: fp32 or bf16, else a microscaled format.
// What bounds a row in registers is not the memory but the instructions around its elements.  A choice is therefore made once
// for all of a thread's chunks, not chunk by chunk, and rows that fill their threads (FULL) check no element: see
// launch_block_norm for what that is worth.
template <int CH, bool XB, bool RB, int OUT, int MODE>
__global__ void __launch_bounds__(512, CH == 2 && XB ? 2 : 1) block_norm_kernel(const __grid_constant__ BlockNormArgs a) {
    __shared__ Shared sh;
    int turn = 0;
    // (dependents first: a matmul behind this kernel fetches its weights while the kernel before it still runs; see note_early_chain_launch)
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint32_t dim = (uint32_t)a.dim;
    const uint32_t row = blockIdx.x * blockDim.y + threadIdx.y;
    if (row >= a.rows) return;  // (several rows in a block: each is a warp's, and warps share nothing)
    constexpr bool FULL = MODE == kFull;
    static_assert(OUT == 0 || MODE != kApart, "blocks of codes are neighbours");
    auto at = [&](int j) {
        if (MODE == kApart) return Place{j * 8 * blockDim.x + threadIdx.x, blockDim.x, dim};
        return Place{(j * blockDim.x + threadIdx.x) * 8, 1, dim};
    };
    // f(chunk, its place) for the thread's chunks that lie within the row
    auto chunks = [&](auto&& f) {
#pragma unroll
        for (int j = 0; j < CH; j++) {
            const Place p = at(j);
            if (FULL || p.first < dim) f(j, p);
        }
    };
    const size_t r0 = (size_t)row * dim;
    Raw<XB, MODE> rh[CH], rg[CH];
    Raw<RB, MODE> rr[CH];
    if (a.h) {
        const char* h = static_cast<const char*>(a.h) + row * a.h_ld * (XB ? 2 : 4);
        chunks([&](int j, const Place& p) { rh[j].load(h, p); });
    }
    if (a.r) {
        const char* r = static_cast<const char*>(a.r) + r0 * (RB ? 2 : 4);
        chunks([&](int j, const Place& p) { rr[j].load(r, p); });
    }
    if (a.gate) {
        const char* gate = static_cast<const char*>(a.gate) + (a.gate_rows ? row / (uint32_t)a.gate_rows : 0) * a.gate_ld * (XB ? 2 : 4);
        chunks([&](int j, const Place& p) { rg[j].load(gate, p); });
    }
    Pair v[CH][4];
    auto total = [&]() {
        Pair s = 0;
        chunks([&](int j, const Place&) {
#pragma unroll
            for (int e = 0; e < 4; e++) s = add2(s, v[j][e]);
        });
        return lo_of(s) + hi_of(s);
    };
    auto squares = [&](float mean) {  // of the differences from mean
        Pair s = 0;
        const Pair neg = pair_of(-mean, -mean);
        chunks([&](int j, const Place&) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const Pair d = mean == 0.0f ? v[j][e] : add2(v[j][e], neg);
                s = fma2(d, d, s);
            }
        });
        return lo_of(s) + hi_of(s);
    };
    auto shift = [&](float mean) {
        const Pair neg = pair_of(-mean, -mean);
        chunks([&](int j, const Place& p) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                v[j][e] = add2(v[j][e], neg);
                if (MODE == kApart) {  // (what is not there stays zero)
                    const uint32_t i = p.first + 2 * e * p.step;
                    v[j][e] = i + p.step < dim ? v[j][e] : i < dim ? v[j][e] & 0xFFFFFFFFull : 0;
                }
            }
        });
    };
    // 1 / sqrt(...) of a norm; its mean is taken off
    auto scale_of = [&](int kind) {
        if (kind == LUX_CUDA_NORM_LAYER) {
            if (FULL) {
                const float own = total() * (1.0f / (8 * CH));
                const Stats st = row_moments(own, squares(own), 8 * CH, a.inv_dim, sh, turn);
                shift(st.mean);
                return inv_root(st.squares, a.inv_dim, a.eps);
            }
            shift(row_sum(total(), sh, turn) * a.inv_dim);
        }
        return inv_root(row_sum(squares(0.0f), sh, turn), a.inv_dim, a.eps);
    };
    auto norm = [&](int kind, const float* w, const float* c) {
        if (kind == LUX_CUDA_NORM_NONE) return;
        const float scale = scale_of(kind);
        const Pair inv = pair_of(scale, scale);
        if (w) {
            chunks([&](int j, const Place& p) {
                Pair wv[4];
                weights8<MODE>(w, p, wv);
#pragma unroll
                for (int e = 0; e < 4; e++) v[j][e] = mul2(mul2(v[j][e], inv), wv[e]);
            });
        } else {
            chunks([&](int j, const Place&) {
#pragma unroll
                for (int e = 0; e < 4; e++) v[j][e] = mul2(v[j][e], inv);
            });
        }
        if (c)
            chunks([&](int j, const Place& p) {
                Pair cv[4];
                weights8<MODE>(c, p, cv);
#pragma unroll
                for (int e = 0; e < 4; e++) v[j][e] = add2(v[j][e], cv[e]);
            });
    };
    if (a.h) {
        chunks([&](int j, const Place&) {
#pragma unroll
            for (int e = 0; e < 4; e++) v[j][e] = rh[j].get(e);
        });
        norm(a.post_kind, a.post_w, a.post_b);
        auto gated = [&](auto&& act) {
            chunks([&](int j, const Place&) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const Pair g = rg[j].get(e);
                    v[j][e] = mul2(v[j][e], pair_of(act(lo_of(g)), act(hi_of(g))));
                }
            });
        };
        if (a.gate) {
            if (a.gate_act == LUX_CUDA_GATE_SIGMOID) gated([](float g) { return act_of(g, LUX_CUDA_GATE_SIGMOID); });
            else if (a.gate_act == LUX_CUDA_GATE_TANH) gated([](float g) { return act_of(g, LUX_CUDA_GATE_TANH); });
            else gated([](float g) { return g; });
        }
        const Pair branch = pair_of(a.branch_scale, a.branch_scale);
        chunks([&](int j, const Place&) {
#pragma unroll
            for (int e = 0; e < 4; e++) v[j][e] = mul2(branch, v[j][e]);
        });
    } else {
        chunks([&](int j, const Place&) {
#pragma unroll
            for (int e = 0; e < 4; e++) v[j][e] = 0;
        });
    }
    if (a.r) {
        const Pair res = pair_of(a.res_scale, a.res_scale);
        chunks([&](int j, const Place&) {
#pragma unroll
            for (int e = 0; e < 4; e++) v[j][e] = fma2(res, rr[j].get(e), v[j][e]);
        });
    }
    char* r_out = static_cast<char*>(a.r_out) + r0 * (RB ? 2 : 4);
    if (a.r_out) chunks([&](int j, const Place& p) { store8<RB, MODE>(r_out, p, v[j]); });
    if (RB)  // what is stored is what the second norm sees
        chunks([&](int j, const Place&) {
#pragma unroll
            for (int e = 0; e < 4; e++) v[j][e] = unpack2(pack2(v[j][e]));
        });
    if (!a.out) return;
    norm(a.pre_kind, a.pre_w, a.pre_b);
    if (OUT == 0) {
        char* out = static_cast<char*>(a.out) + r0 * (a.out_bf16 ? 2 : 4);
        if (a.out_bf16) chunks([&](int j, const Place& p) { store8<true, MODE>(out, p, v[j]); });
        else chunks([&](int j, const Place& p) { store8<false, MODE>(out, p, v[j]); });
    } else {
        constexpr int F = OUT ? OUT : 1;
        const Pair pre = pair_of(a.out_pre, a.out_pre);
        const int tiles_k = mx4_tiles_k(dim, F);
#pragma unroll
        for (int j = 0; j < CH; j++) {  // (the whole warp: lanes past the row carry zeros)
            const uint32_t i = at(j).first;
            Pair u[4];
            uint32_t c[1], byte;
#pragma unroll
            for (int e = 0; e < 4; e++) u[e] = FULL || i < dim ? mul2(unpack2(pack2(v[j][e])), pre) : 0;
            mx4_encode<F, 8>(u, c, byte);
            const uint32_t word = mx4_scale_word<F, 8>(byte, threadIdx.x & 31);
            if (FULL || i < dim) {
                static_cast<uint32_t*>(a.out)[(r0 + i) >> 3] = c[0];
                if ((threadIdx.x & 31) % (mx4_block(F) / 2) == 0)
                    *reinterpret_cast<uint32_t*>(a.out_scales + mx4_scale_at(row, i / (4 * mx4_block(F)), tiles_k)) = word;
            }
        }
    }
}

// Longer rows, and rows of a multiple of 8 on odd boundaries: nothing is kept, what is needed is read (or, without r_out, computed) again
// for every step.  V neighbours to a thread.  (V = 8 with and without OUT: the same sums, so the same stream whatever becomes of the
// output.)
template <int OUT, int V>
__global__ void __launch_bounds__(1024) block_norm_any_kernel(const __grid_constant__ BlockNormArgs a) {
    static_assert(OUT == 0 || V == 8, "blocks of codes: eight neighbours");
    __shared__ Shared sh;
    int turn = 0;
    // (dependents first: a matmul behind this kernel fetches its weights while the kernel before it still runs; see note_early_chain_launch)
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const size_t dim = a.dim, row = (size_t)blockIdx.x * blockDim.y + threadIdx.y;
    if (row >= a.rows) return;
    const bool xb = a.x_bf16, rb = a.r_bf16;
    const size_t h0 = row * a.h_ld, g0 = (a.gate_rows ? row / a.gate_rows : 0) * a.gate_ld, r0 = row * dim;
    auto ld = [](const void* p, bool bf16, size_t i) { return bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]) : static_cast<const float*>(p)[i]; };
    auto st = [](void* p, bool bf16, size_t i, float x) {
        if (bf16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
        else static_cast<float*>(p)[i] = x;
    };
    struct Norm {
        float mean, inv;
    };
    auto norm = [&](const Norm& s, int kind, const float* w, const float* c, size_t i, float x) {
        if (kind == LUX_CUDA_NORM_NONE) return x;
        x = (x - s.mean) * s.inv;
        if (w) x *= w[i];
        return c ? x + c[i] : x;
    };
    Norm post{0.0f, 1.0f};
    auto h_at = [&](size_t i) { return ld(a.h, xb, h0 + i); };
    auto stream = [&](size_t i) {  // r' of element i
        float s = 0.0f;
        if (a.h) {
            float x = norm(post, a.post_kind, a.post_w, a.post_b, i, h_at(i));
            if (a.gate) x *= act_of(ld(a.gate, xb, g0 + i), a.gate_act);
            s = a.branch_scale * x;
        }
        if (a.r) s = fmaf(a.res_scale, ld(a.r, rb, r0 + i), s);
        return rb ? round_bf16(s) : s;
    };
    // (what this thread has stored; without a place to store it, computed again)
    auto r_at = [&](size_t i) { return a.r_out ? ld(a.r_out, rb, r0 + i) : stream(i); };
    const size_t step = (size_t)blockDim.x * V;
    auto elements = [&](auto&& f) {
        for (size_t i0 = (size_t)threadIdx.x * V; i0 < dim; i0 += step)
            for (int e = 0; e < V; e++)
                if (i0 + e < dim) f(i0 + e);
    };
    auto stats = [&](int kind, auto&& value) {
        Norm st{0.0f, 1.0f};
        if (kind == LUX_CUDA_NORM_NONE) return st;
        float s = 0.0f;
        if (kind == LUX_CUDA_NORM_LAYER) {
            elements([&](size_t i) { s += value(i); });
            st.mean = row_sum(s, sh, turn) * a.inv_dim;
            s = 0.0f;
        }
        elements([&](size_t i) {
            const float d = value(i) - st.mean;
            s = fmaf(d, d, s);
        });
        st.inv = inv_root(row_sum(s, sh, turn), a.inv_dim, a.eps);
        return st;
    };
    if (a.h) post = stats(a.post_kind, h_at);
    if (a.r_out) elements([&](size_t i) { st(a.r_out, rb, r0 + i, stream(i)); });
    if (!a.out) return;
    const Norm pre = stats(a.pre_kind, r_at);
    if (OUT == 0) {
        elements([&](size_t i) { st(a.out, a.out_bf16, r0 + i, norm(pre, a.pre_kind, a.pre_w, a.pre_b, i, r_at(i))); });
    } else {
        constexpr int F = OUT ? OUT : 1;
        for (size_t base = 0; base < dim; base += step) {  // (the whole warp: lanes past the row carry zeros)
            const size_t at = base + (size_t)threadIdx.x * V;
            Pair u[4];
            uint32_t c[1], byte;
            auto value = [&](size_t i) { return i < dim ? __fmul_rn(round_bf16(norm(pre, a.pre_kind, a.pre_w, a.pre_b, i, r_at(i))), a.out_pre) : 0.0f; };
#pragma unroll
            for (int e = 0; e < 4; e++) u[e] = pair_of(value(at + 2 * e), value(at + 2 * e + 1));
            mx4_encode<F, 8>(u, c, byte);
            const uint32_t word = mx4_scale_word<F, 8>(byte, threadIdx.x & 31);
            if (at < dim) {
                static_cast<uint32_t*>(a.out)[(r0 + at) >> 3] = c[0];
                if ((threadIdx.x & 31) % (mx4_block(F) / 2) == 0)
                    *reinterpret_cast<uint32_t*>(a.out_scales + mx4_scale_at(row, (int)(at / (4 * mx4_block(F))), mx4_tiles_k((int)dim, F))) = word;
            }
        }
    }
}

using NormKernel = void (*)(BlockNormArgs);
template <int CH, bool XB, bool RB, int MODE>
NormKernel pick_out(int format) {
    if constexpr (MODE != kApart) {
        if (format == LUX_CUDA_MX4_E8M0) return block_norm_kernel<CH, XB, RB, LUX_CUDA_MX4_E8M0, MODE>;
        if (format == LUX_CUDA_MX4_E4M3) return block_norm_kernel<CH, XB, RB, LUX_CUDA_MX4_E4M3, MODE>;
    }
    return block_norm_kernel<CH, XB, RB, 0, MODE>;
}
template <int CH, int MODE>
NormKernel pick(const BlockNormArgs& a) {
    return a.x_bf16 ? (a.r_bf16 ? pick_out<CH, true, true, MODE>(a.out_format) : pick_out<CH, true, false, MODE>(a.out_format))
                    : (a.r_bf16 ? pick_out<CH, false, true, MODE>(a.out_format) : pick_out<CH, false, false, MODE>(a.out_format));
}

}  // namespace

cudaError_t launch_block_norm(const BlockNormArgs& a, int sm_count, cudaStream_t stream, bool overlap_prev) {
    if (!a.rows || !a.dim) return cudaSuccess;
    NormKernel kern;
    size_t threads;
    auto warps = [](size_t n) { return (n + 31) / 32 * 32; };
    const bool wide = a.vec && a.dim % 8 == 0;
    if ((wide || a.dim % 8) && a.dim <= 16384) {
        // two chunks per thread as far as 512 threads hold the row (2048 x 4096, rms | rms, bf16: 17.5 us against 19.2 with four)
        const int ch = a.dim <= 8192 ? 2 : 4;
        threads = warps((a.dim + 8 * ch - 1) / (8 * ch));
        const bool full = a.dim == threads * 8 * ch;
        kern = ch == 2 ? (!wide ? pick<2, kApart>(a) : full ? pick<2, kFull>(a) : pick<2, kWide>(a))
                       : (!wide ? pick<4, kApart>(a) : full ? pick<4, kFull>(a) : pick<4, kWide>(a));
    } else if (a.dim % 8 == 0) {
        kern = a.out_format == LUX_CUDA_MX4_E8M0   ? block_norm_any_kernel<LUX_CUDA_MX4_E8M0, 8>
               : a.out_format == LUX_CUDA_MX4_E4M3 ? block_norm_any_kernel<LUX_CUDA_MX4_E4M3, 8>
                                                   : block_norm_any_kernel<0, 8>;
        threads = std::min<size_t>(1024, warps(a.dim / 8));
    } else {
        kern = block_norm_any_kernel<0, 1>;
        threads = 1024;
    }
    const unsigned rows_per_block = threads == 32 ? 4 : 1;
    const size_t blocks = (a.rows + rows_per_block - 1) / rows_per_block;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3((unsigned)threads, rows_per_block);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = overlap_prev ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kern, a);
}

}  // namespace luxcuda
