// The row step between two blocks of a model: the norm after a block, its gate, the residual sum, and the norm before the next
// block, in one pass over the data:
//   b  = post(h)                                     none | rms: h / sqrt(mean h^2 + eps) * w | layer: (h - mean) / sqrt(var + eps) * w + c
//   r' = round(res_scale * r + branch_scale * act(gate) * b)
//   o  = pre(r')                                     of the rounded r', so that it is what a call on the stored stream would give
// o leaves as fp32, as bf16, or rounded to bf16 and from there in the microscaled format (mx4.cuh) that the product takes.
//
// HBM-bound: h, r, (gate) read and r', o written once.  A group of threads takes a row, asks for all of it at once and keeps it in
// registers (rows of 8193 to 16384 elements, in part, in local memory: see launch_block_norm) between the statistics, which are fp32 sums
// over threads, lanes and warps; the variance is the mean of squared differences.
#include <algorithm>

#include "block_norm.cuh"

namespace luxcuda {

namespace {

// Rows of up to 8 * CH elements per thread, a multiple of 8, every row on a 16-byte boundary; FULL: exactly so many.  blockDim =
// (threads of a row, rows): several rows only where a row is a warp's.  OUT: 0: fp32 or bf16, else a microscaled format.
// What bounds a row in registers is not the memory but the instructions around its elements.  A choice is therefore made once
// for all of a thread's chunks, not chunk by chunk, and rows that fill their threads (FULL) check no element: see
// launch_block_norm for what that is worth.
template <int CH, bool XB, bool RB, int OUT, int MODE>
__global__ void __launch_bounds__(512, CH == 1 ? 2 + XB + RB : CH == 2 && XB ? 2 : 1) block_norm_kernel(const __grid_constant__ BlockNormArgs a) {
    __shared__ Shared sh;
    // (dependents first: a matmul behind this kernel fetches its weights while the kernel before it still runs; see note_early_chain_launch)
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    constexpr bool FULL = MODE == kFull;
    const int lanes = MODE == kWide && blockDim.x < 32 ? 16 : 32;  // of a warp, for a row
    const uint32_t row = blockIdx.x * blockDim.y + threadIdx.y;
    if (lanes == 32 && row >= a.rows) return;  // (several rows in a block: each is a warp's, and warps share nothing)
    const uint32_t dim = MODE == kWide && row >= a.rows ? 0 : (uint32_t)a.dim;  // (a warp's second row that is not there has no elements)
    const uint32_t warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
    auto at = [&](int j) {
        if (MODE != kApart) return Place{(j * blockDim.x + threadIdx.x) * 8};
        const uint32_t chunk = (j * (blockDim.x / 32) + warp) * 256;
        return Place{chunk + (threadIdx.x & 31), dim, chunk + 256 <= dim};
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
    Group g{&sh, lanes == 32 ? (int)(blockDim.x >> 5) : 1, (int)(threadIdx.x >> 5), 0, 0, lanes};
    auto within = [&](int j) { return at(j).first < dim; };
    RowValues<CH, FULL, decltype(within)> values{v, within, g, a};
    auto shift = [&](float mean) {
        const Pair neg = pair_of(-mean, -mean);
        chunks([&](int j, const Place& p) {
#pragma unroll
            for (int e = 0; e < 4; e++) v[j][e] = add2(v[j][e], neg);
            if (MODE == kApart && !p.whole) {  // (what is not there stays zero)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const uint32_t i = p.first + 64 * e;
                    v[j][e] = i + 32 < dim ? v[j][e] : i < dim ? v[j][e] & 0xFFFFFFFFull : 0;
                }
            }
        });
    };
    auto weights = [&](const float* w, int j, Pair (&out)[4]) { weights8<MODE>(w, at(j), out); };
    if (a.h) {
        chunks([&](int j, const Place&) {
#pragma unroll
            for (int e = 0; e < 4; e++) v[j][e] = rh[j].get(e);
        });
        values.norm(a.post_kind, a.post_w, a.post_b, shift, weights);
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
        values.scale_by(a.branch_scale);
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
    values.norm(a.pre_kind, a.pre_w, a.pre_b, shift, weights);
    if (OUT == 0) {
        char* out = static_cast<char*>(a.out) + r0 * (a.out_bf16 ? 2 : 4);
        if (a.out_bf16) chunks([&](int j, const Place& p) { store8<true, MODE>(out, p, v[j]); });
        else chunks([&](int j, const Place& p) { store8<false, MODE>(out, p, v[j]); });
    } else {
        // (blocks of codes are neighbours: elements that lie 32 apart change places within the warp first)
        __shared__ uint4 turn[MODE == kApart && OUT ? 512 : 1];
        const uint32_t lane = threadIdx.x & 31;
        uint4* const mine = turn + (threadIdx.y * (blockDim.x >> 5) + warp) * 32;
#pragma unroll
        for (int j = 0; j < CH; j++) {
            uint32_t i = at(j).first;
            if (MODE == kApart) {
                __syncwarp();
#pragma unroll
                for (int e = 0; e < 8; e++)
                    reinterpret_cast<__nv_bfloat16*>(mine)[32 * e + lane] = __float2bfloat16_rn(e & 1 ? hi_of(v[j][e >> 1]) : lo_of(v[j][e >> 1]));
                __syncwarp();
                const uint4 q = mine[lane];
                v[j][0] = unpack2(q.x); v[j][1] = unpack2(q.y); v[j][2] = unpack2(q.z); v[j][3] = unpack2(q.w);
                i += 7 * lane;
            }
            put_codes<OUT ? OUT : 1>(a, v[j], row, i, FULL || i < dim);
        }
    }
}

// Longer rows: nothing is kept, what is needed is read (or, without r_out, computed) again for every step.  V neighbours to a thread.  (V = 8 with and without OUT: the same sums, so the same stream whatever becomes of the
// output.)
template <int OUT, int V>
__global__ void __launch_bounds__(1024) block_norm_any_kernel(const __grid_constant__ BlockNormArgs a) {
    static_assert(OUT == 0 || V == 8, "blocks of codes: eight neighbours");
    __shared__ Shared sh;
    Group g{&sh, (int)(blockDim.x >> 5), (int)(threadIdx.x >> 5), 0, 0};
    // (as above)
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
            st.mean = row_sum(s, g) * a.inv_dim;
            s = 0.0f;
        }
        elements([&](size_t i) {
            const float d = value(i) - st.mean;
            s = fmaf(d, d, s);
        });
        st.inv = inv_root(row_sum(s, g), a.inv_dim, a.eps);
        return st;
    };
    if (a.h) post = stats(a.post_kind, h_at);
    if (a.r_out) elements([&](size_t i) { st(a.r_out, rb, r0 + i, stream(i)); });
    if (!a.out) return;
    const Norm pre = stats(a.pre_kind, r_at);
    if (OUT == 0) {
        elements([&](size_t i) { st(a.out, a.out_bf16, r0 + i, norm(pre, a.pre_kind, a.pre_w, a.pre_b, i, r_at(i))); });
    } else {
        for (size_t base = 0; base < dim; base += step) {  // (the whole warp: lanes past the row carry zeros)
            const size_t at = base + (size_t)threadIdx.x * V;
            Pair u[4];
            auto value = [&](size_t i) { return i < dim ? norm(pre, a.pre_kind, a.pre_w, a.pre_b, i, r_at(i)) : 0.0f; };
#pragma unroll
            for (int e = 0; e < 4; e++) u[e] = pair_of(value(at + 2 * e), value(at + 2 * e + 1));
            put_codes<OUT ? OUT : 1>(a, u, row, (uint32_t)at, at < dim);
        }
    }
}

using NormKernel = void (*)(BlockNormArgs);
template <int CH, bool XB, bool RB, int MODE>
NormKernel pick_out(int format) {
    if (format == LUX_CUDA_MX4_E8M0) return block_norm_kernel<CH, XB, RB, LUX_CUDA_MX4_E8M0, MODE>;
    if (format == LUX_CUDA_MX4_E4M3) return block_norm_kernel<CH, XB, RB, LUX_CUDA_MX4_E4M3, MODE>;
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
    if (block_norm_streams(a, sm_count)) return launch_block_norm_stream(a, sm_count, stream, overlap_prev);
    NormKernel kern;
    size_t threads;
    auto warps = [](size_t n) { return (n + 31) / 32 * 32; };
    const bool wide = a.vec && a.dim % 8 == 0;
    if (a.dim <= 16384) {
        // Two chunks per thread as far as 512 threads hold the row (2048 x 4096, rms | rms, bf16: 17.5 us against 19.2 with four; one: 8192 x
        // 1024 18.5 against 15.4).  Single elements wait for memory one chunk at a time, and want twice as many warps for it:
        // one chunk (4000 x 1031 15.2 us, two 19.0; 8 x 4095 4.0 against 4.8).
        // Four chunks of fp32 h and r do not fit 128 registers: up to 800 bytes a thread spill (512 x 12288 50 us, bf16 18.5).
        const int ch = !wide && a.dim <= 4096 ? 1 : a.dim <= 8192 ? 2 : 4;
        threads = warps((a.dim + 8 * ch - 1) / (8 * ch));
        const bool full = a.dim == threads * 8 * ch;
        kern = ch == 1 ? pick<1, kApart>(a) : ch == 2 ? (!wide ? pick<2, kApart>(a) : full ? pick<2, kFull>(a) : pick<2, kWide>(a))
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
    // Many short rows on 16-byte boundaries: two to a warp (the 16 lanes that a scale word's blocks have at most).  65536 x 128, h,
    // the stream and one norm, 16.6 us against 28.9, 8192 x 256 rms | rms 5.9 against 7.2; but 8 x 256 2.65 against 2.4.
    if (wide && a.dim <= 256 && a.rows >= (size_t)8 * sm_count) threads = 16;
    const unsigned rows_per_block = threads <= 32 ? 128 / threads : 1;
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
