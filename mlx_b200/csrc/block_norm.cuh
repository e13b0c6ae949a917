// What the kernels of the row step between two blocks (block_norm.cu, block_norm_stream.cu) share.
#pragma once
#include "internal.h"
#include "mx4.cuh"
#include "pair.cuh"

namespace luxcuda {

__device__ __forceinline__ float act_of(float g, int act) {
    if (act == LUX_CUDA_GATE_SIGMOID) {
        // 1 / (1 + 2^t), t = -g / ln 2 in two pieces, so that a large g costs no accuracy; at half of what expf and an exact
        // reciprocal issue, which were a quarter of the kernel.  From |t| = 127 on the result is 0 (below the normal numbers) or 1
        // whatever the second piece says, which is then no small number or none at all (infinity - infinity); a NaN passes through
        // ex2.
        const float c_hi = -1.44269504f, c_lo = -1.92596299e-8f;  // -1 / ln 2
        const float t = g * c_hi, lo = fmaf(g, c_lo, fmaf(g, c_hi, -t));
        float e, d;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
        if (fabsf(t) < 127.0f) e = fmaf(e, lo * 0.693147181f, e);
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
// or, on any boundary, 32 apart (kApart: a warp's chunk is 256 neighbours, of which each access takes 32; those at `end` and behind
// it are zero, and nobody asks where the whole chunk lies ahead of it).
enum Mode { kWide, kFull, kApart };
struct Place {
    uint32_t first, end;
    bool whole;  // (the same in all lanes)
};
// f(element 0 .. 7 of the thread's, whether it lies within the row)
template <class F>
__device__ __forceinline__ void apart8(const Place& p, F&& f) {
    if (p.whole) {
#pragma unroll
        for (int e = 0; e < 8; e++) f(e, true);
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) f(e, p.first + 32 * e < p.end);
    }
}
template <bool BF16, int MODE>
struct Raw {
    uint4 q[BF16 ? 1 : 2];
    __device__ __forceinline__ void load(const char* row, const Place& p) {
        const char* s = row + (size_t)p.first * (BF16 ? 2 : 4);
        if constexpr (MODE != kApart) {
            q[0] = ld_row(s);
            if (!BF16) q[BF16 ? 0 : 1] = ld_row(s + 16);
        } else {
            uint32_t w[8];
            apart8(p, [&](int e, bool in) {
                w[e] = !in ? 0u : BF16 ? (uint32_t)reinterpret_cast<const uint16_t*>(s)[32 * e] : reinterpret_cast<const uint32_t*>(s)[32 * e];
            });
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
        char* const d = row + (size_t)p.first * (BF16 ? 2 : 4);
        apart8(p, [&](int e, bool in) {
            const float x = e & 1 ? hi_of(v[e >> 1]) : lo_of(v[e >> 1]);
            if (!in) return;
            if (BF16) reinterpret_cast<__nv_bfloat16*>(d)[32 * e] = __float2bfloat16_rn(x);
            else reinterpret_cast<float*>(d)[32 * e] = x;
        });
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
        uint32_t u[8];
        apart8(p, [&](int e, bool in) { u[e] = in ? __float_as_uint(__ldg(w + p.first + 32 * e)) : 0u; });
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = pair_of(u[2 * e], u[2 * e + 1]);
    } else {
        const ulonglong2 a = __ldg(reinterpret_cast<const ulonglong2*>(w + p.first)), b = __ldg(reinterpret_cast<const ulonglong2*>(w + p.first) + 1);
        v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
    }
}
// What the warps of a row exchange: two places, used in turn, so that a warp may be a step ahead of those that still read.
struct Shared {
    float2 part[2][32];
};
// The threads of a row: `warps` warps, of which this is the `warp`-th, with a barrier of their own (none where it is one warp); or the 16
// `lanes` of a half of a warp.
struct Group {
    Shared* sh;
    int warps, warp, barrier, turn;
    int lanes = 32;
};
__device__ __forceinline__ float warp_sum(float v, int lanes = 32) {
    if (lanes == 32) v += __shfl_xor_sync(0xffffffffu, v, 16);
#pragma unroll
    for (int o = 8; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// every lane gets the contribution of the warp of its number (zeros past the last).  All warps go on with all of them: one warp that
// does, and tells the others, makes two waits of one (2048 x 4096, layer | layer: 51 us against 40).
__device__ __forceinline__ float2 exchange(float2 v, Group& g) {
    const int lane = threadIdx.x & 31;
    if (lane == 0) g.sh->part[g.turn][g.warp] = v;
    asm volatile("bar.sync %0, %1;" ::"r"(g.barrier), "r"(g.warps * 32) : "memory");
    v = lane < g.warps ? g.sh->part[g.turn][lane] : make_float2(0.0f, 0.0f);
    g.turn ^= 1;
    return v;
}
__device__ __forceinline__ float row_sum(float v, Group& g) {
    v = warp_sum(v, g.lanes);
    return g.warps == 1 ? v : warp_sum(exchange(make_float2(v, 0.0f), g).x);
}
struct Stats {
    float mean, squares;
};
// The row's mean and the squared differences from it, in one exchange, from every thread's own mean and squared differences over n
// elements, the same number in all threads: two halves of 2n elements have their means' mean and, besides their own, n/2 times the
// squared difference of the means (Chan, Golub, LeVeque 1979).
__device__ __forceinline__ Stats row_moments(float mean, float squares, int n, float inv_dim, Group& g) {
    float half = 0.5f * n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1, half *= 2.0f) {
        const float d = __shfl_xor_sync(0xffffffffu, mean, o) - mean;
        squares += __shfl_xor_sync(0xffffffffu, squares, o);
        squares = fmaf(d * d, half, squares);
        mean = fmaf(0.5f, d, mean);
    }
    if (g.warps == 1) return Stats{mean, squares};
    const float2 p = exchange(make_float2(mean, squares), g);
    mean = warp_sum(p.x) * (32 * n * inv_dim);
    const float d = (int)(threadIdx.x & 31) < g.warps ? p.x - mean : 0.0f;
    return Stats{mean, warp_sum(fmaf(d * d, 32.0f * n, p.y))};
}
__device__ __forceinline__ float inv_root(float squares, float inv_dim, float eps) { return __frsqrt_rn(fmaf(squares, inv_dim, eps)); }

// A row's elements in a thread's registers, CH chunks of four pairs, and the steps of the row on them.  In(j): chunk j lies within the
// row; FULL: all chunks do.
template <int CH, bool FULL, class In>
struct RowValues {
    Pair (&v)[CH][4];
    const In in;
    Group& g;
    const BlockNormArgs& a;
    template <class F>
    __device__ __forceinline__ void each(F&& f) {  // f(chunk)
#pragma unroll
        for (int j = 0; j < CH; j++)
            if (FULL || in(j)) f(j);
    }
    __device__ __forceinline__ float total() {
        Pair s = 0;
        each([&](int j) {
#pragma unroll
            for (int e = 0; e < 4; e++) s = add2(s, v[j][e]);
        });
        return lo_of(s) + hi_of(s);
    }
    __device__ __forceinline__ float squares(float mean) {  // of the differences from mean
        Pair s = 0;
        const Pair neg = pair_of(-mean, -mean);
        each([&](int j) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const Pair d = mean == 0.0f ? v[j][e] : add2(v[j][e], neg);
                s = fma2(d, d, s);
            }
        });
        return lo_of(s) + hi_of(s);
    }
    // 1 / sqrt(...) of a norm; shift(mean) takes its mean off
    template <class Shift>
    __device__ __forceinline__ float scale(int kind, Shift&& shift) {
        if (kind == LUX_CUDA_NORM_LAYER) {
            if (FULL) {
                const float own = total() * (1.0f / (8 * CH));
                const Stats st = row_moments(own, squares(own), 8 * CH, a.inv_dim, g);
                shift(st.mean);
                return inv_root(st.squares, a.inv_dim, a.eps);
            }
            shift(row_sum(total(), g) * a.inv_dim);
        }
        return inv_root(row_sum(squares(0.0f), g), a.inv_dim, a.eps);
    }
    // load(w, j, out): chunk j of a weight, which is whatever load takes (and false: none)
    template <class Weight, class Shift, class Load>
    __device__ __forceinline__ void norm(int kind, Weight w, Weight c, Shift&& shift, Load&& load) {
        if (kind == LUX_CUDA_NORM_NONE) return;
        const float s = scale(kind, shift);
        const Pair inv = pair_of(s, s);
        if (w) {
            each([&](int j) {
                Pair wv[4];
                load(w, j, wv);
#pragma unroll
                for (int e = 0; e < 4; e++) v[j][e] = mul2(mul2(v[j][e], inv), wv[e]);
            });
        } else {
            each([&](int j) {
#pragma unroll
                for (int e = 0; e < 4; e++) v[j][e] = mul2(v[j][e], inv);
            });
        }
        if (c)
            each([&](int j) {
                Pair cv[4];
                load(c, j, cv);
#pragma unroll
                for (int e = 0; e < 4; e++) v[j][e] = add2(v[j][e], cv[e]);
            });
    }
    __device__ __forceinline__ void scale_by(float s) {
        const Pair p = pair_of(s, s);
        each([&](int j) {
#pragma unroll
            for (int e = 0; e < 4; e++) v[j][e] = mul2(p, v[j][e]);
        });
    }
};
// Eight neighbouring values of a lane, rounded to bf16, into the microscaled format; the whole warp, zeros in lanes past the row (there: false)
template <int F>
__device__ __forceinline__ void put_codes(const BlockNormArgs& a, const Pair (&v)[4], size_t row, uint32_t i, bool there) {
    const Pair pre = pair_of(a.out_pre, a.out_pre);
    Pair u[4];
    uint32_t c[1], byte;
#pragma unroll
    for (int e = 0; e < 4; e++) u[e] = there ? mul2(unpack2(pack2(v[e])), pre) : 0;
    mx4_encode<F, 8>(u, c, byte);
    const uint32_t word = mx4_scale_word<F, 8>(byte, threadIdx.x & 31);
    if (there) {
        static_cast<uint32_t*>(a.out)[(row * a.dim + i) >> 3] = c[0];
        if ((threadIdx.x & 31) % (mx4_block(F) / 2) == 0)
            *reinterpret_cast<uint32_t*>(a.out_scales + mx4_scale_at(row, i / (4 * mx4_block(F)), mx4_tiles_k((int)a.dim, F))) = word;
    }
}

}  // namespace luxcuda
