// The row step between two blocks (block_norm.cu) for many rows: one block per SM, weights in shared memory, rows on their way there
// by the copy engine while others are worked on.
//
// With a row per block and its data in registers (block_norm.cu) an SM has four rows under way, each in a chain of load, statistics,
// arithmetic, statistics, store; neither memory nor arithmetic is busy half of the time.  Here one warp keeps a ring of rows filled
// (h, r and a gate of the row's own, each one bulk copy), and groups of threads, 32 elements to a thread, take the rows in turn.
// Twice the elements of a thread halve what a row costs besides them; weights, biases and a gate that all rows share (as its
// function's value) are read once per block.  Figures: block_norm_streams.
#include <algorithm>
#include <atomic>

#include "block_norm.cuh"

namespace luxcuda {

namespace {

constexpr int kChunks = 4;          // of eight elements per thread
constexpr int kMaxGroups = 14;      // with a barrier of their own each, 1 .. 14 (0: the block's, 15: the workers')
constexpr int kMaxThreads = 768;    // 72 registers; more threads with 64 are no faster
constexpr int kMaxSlots = 32;
constexpr int kSmemLimit = 227 * 1024 - 1024;
constexpr uint32_t kWaitClocks = 4000000000u;

struct StreamPlan {
    int group_threads, groups, slots;
    int r_off, gate_off, slot_bytes;  // of a row's parts in its slot
    int w_off[5];                     // post_w, post_b, pre_w, pre_b, shared gate: -1 where there is none
    int ring_off, bar_off, smem;
    int* error;
};

__device__ __forceinline__ uint32_t s32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ bool bar_try(uint32_t b, uint32_t parity) {
    uint32_t ok;
    asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3; selp.u32 %0, 1, 0, p; }"
                 : "=r"(ok) : "r"(b), "r"(parity), "r"(20000u) : "memory");
    return ok != 0;
}
// Bounded wait (about two seconds of SM clock); after one that ran out nobody waits any more, the results are worthless and the host is told.
__device__ __forceinline__ void bar_wait(uint32_t b, uint32_t parity, volatile int* abort) {
    if (bar_try(b, parity)) return;
    const uint32_t t0 = clock();
    do {
#pragma unroll 1
        for (int i = 0; i < 64; i++)
            if (bar_try(b, parity)) return;
    } while (!*abort && (uint32_t)clock() - t0 < kWaitClocks);
    *abort = 1;
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ uint4 lds_v4(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}
// eight neighbours of a row
template <bool BF16>
__device__ __forceinline__ void row8(uint32_t base, uint32_t i, Pair (&v)[4]) {
    const uint4 a = lds_v4(base + i * (BF16 ? 2 : 4));
    if (BF16) {
        v[0] = unpack2(a.x); v[1] = unpack2(a.y); v[2] = unpack2(a.z); v[3] = unpack2(a.w);
    } else {
        const uint4 b = lds_v4(base + i * 4 + 16);
        v[0] = pair_of(a.x, a.y); v[1] = pair_of(a.z, a.w); v[2] = pair_of(b.x, b.y); v[3] = pair_of(b.z, b.w);
    }
}
// eight neighbours of a weight, which lies as the first four of every eight, then the other four: no bank conflicts
__device__ __forceinline__ void weight8(uint32_t base, uint32_t dim, uint32_t i, Pair (&v)[4]) {
    const uint4 a = lds_v4(base + i * 2), b = lds_v4(base + dim * 2 + i * 2);
    v[0] = pair_of(a.x, a.y); v[1] = pair_of(a.z, a.w); v[2] = pair_of(b.x, b.y); v[3] = pair_of(b.z, b.w);
}

template <bool XB, bool RB, int OUT, bool FULL>
__global__ void __launch_bounds__(kMaxThreads + 32) block_norm_stream_kernel(const __grid_constant__ BlockNormArgs a, const __grid_constant__ StreamPlan p) {
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ Shared sh[kMaxGroups];
    __shared__ int s_abort;
    volatile int* abort = &s_abort;
    const int tid = threadIdx.x, workers = p.groups * p.group_threads;
    const uint32_t dim = (uint32_t)a.dim, base = s32(smem), full = base + p.bar_off, empty = full + 8 * kMaxSlots;
    const bool own_gate = p.gate_off >= 0;  // the gate of a row comes with it
    if (tid == 0) {
        for (int i = 0; i < p.slots; i++) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(full + 8 * i), "r"(1));
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(empty + 8 * i), "r"(p.group_threads / 32));
        }
        s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // (dependents first: a matmul behind this kernel fetches its weights while the kernel before it still runs; see note_early_chain_launch)
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    __syncthreads();
    if (tid >= workers) {
        if (tid == workers) {
            const uint32_t hb = a.h ? dim * (XB ? 2 : 4) : 0, rb = a.r ? dim * (RB ? 2 : 4) : 0, gb = own_gate ? dim * (XB ? 2 : 4) : 0;
            int slot = 0;
            uint32_t ph = 1;
            for (uint32_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
                bar_wait(empty + 8 * slot, ph, abort);
                if (*abort) break;
                const uint32_t bar = full + 8 * slot, dst = base + p.ring_off + slot * p.slot_bytes;
                asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(hb + rb + gb) : "memory");
                if (hb) bulk_load(dst, static_cast<const char*>(a.h) + row * a.h_ld * (XB ? 2 : 4), hb, bar);
                if (rb) bulk_load(dst + p.r_off, static_cast<const char*>(a.r) + (size_t)row * dim * (RB ? 2 : 4), rb, bar);
                if (gb) bulk_load(dst + p.gate_off, static_cast<const char*>(a.gate) + (row / (uint32_t)a.gate_rows) * a.gate_ld * (XB ? 2 : 4), gb, bar);
                if (++slot == p.slots) { slot = 0; ph ^= 1; }
            }
        }
    } else {
        // Weights, biases and the shared gate's values, as weight8 reads them, for all workers.  All of a thread's loads are under way
        // before its first store: one by one, as many round trips, they take 6 us of the 26 at 2048 x 4096 with four weights.
        const float* ws[4] = {a.post_w, a.post_b, a.pre_w, a.pre_b};
        constexpr int kAhead = 2;
        for (uint32_t i0 = tid * 4; i0 < dim; i0 += kAhead * workers * 4) {
            float4 w[kAhead][4];
            float gv[kAhead][4];
#pragma unroll
            for (int n = 0; n < kAhead; n++) {
                const uint32_t i = i0 + n * workers * 4;
                if (i >= dim) continue;
#pragma unroll
                for (int k = 0; k < 4; k++)
                    if (p.w_off[k] >= 0) w[n][k] = __ldg(reinterpret_cast<const float4*>(ws[k] + i));
                if (p.w_off[4] >= 0) {
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        gv[n][e] = XB ? __bfloat162float(static_cast<const __nv_bfloat16*>(a.gate)[i + e]) : static_cast<const float*>(a.gate)[i + e];
                }
            }
#pragma unroll
            for (int n = 0; n < kAhead; n++) {
                const uint32_t i = i0 + n * workers * 4, at = (i & 4) * (dim / 2) + (i >> 3) * 16;
                if (i >= dim) continue;
#pragma unroll
                for (int k = 0; k < 4; k++)
                    if (p.w_off[k] >= 0) *reinterpret_cast<float4*>(smem + p.w_off[k] + at) = w[n][k];
                if (p.w_off[4] >= 0)
                    *reinterpret_cast<float4*>(smem + p.w_off[4] + at) =
                        make_float4(act_of(gv[n][0], a.gate_act), act_of(gv[n][1], a.gate_act), act_of(gv[n][2], a.gate_act), act_of(gv[n][3], a.gate_act));
            }
        }
        asm volatile("bar.sync 15, %0;" ::"r"(workers) : "memory");
        const int group = tid / p.group_threads, t = tid - group * p.group_threads, lane = tid & 31;
        Group g{&sh[group], p.group_threads / 32, t >> 5, 1 + group, 0};
        auto at = [&](int j) { return (uint32_t)(j * p.group_threads + t) * 8; };
        auto within = [&](int j) { return at(j) < dim; };
        Pair v[kChunks][4];
        RowValues<kChunks, FULL, decltype(within)> values{v, within, g, a};
        auto shift = [&](float mean) {
            const Pair neg = pair_of(-mean, -mean);
            values.each([&](int j) {
#pragma unroll
                for (int e = 0; e < 4; e++) v[j][e] = add2(v[j][e], neg);
            });
        };
        // a weight stands for its address in shared memory (0: none; other things lie there)
        auto weights = [&](uint32_t w, int j, Pair (&out)[4]) { weight8(w, dim, at(j), out); };
        auto placed = [&](int k) { return p.w_off[k] < 0 ? 0u : base + p.w_off[k]; };
        int slot = group % p.slots;
        uint32_t ph = (group / p.slots) & 1;
        for (uint32_t row = blockIdx.x + group * gridDim.x; row < a.rows; row += p.groups * gridDim.x) {
            bar_wait(full + 8 * slot, ph, abort);
            const uint32_t src = base + p.ring_off + slot * p.slot_bytes;
            if (a.h) {
                values.each([&](int j) { row8<XB>(src, at(j), v[j]); });
                values.norm(a.post_kind, placed(0), placed(1), shift, weights);
                if (own_gate) {
                    auto gated = [&](auto&& act) {
                        values.each([&](int j) {
                            Pair q[4];
                            row8<XB>(src + p.gate_off, at(j), q);
#pragma unroll
                            for (int e = 0; e < 4; e++) v[j][e] = mul2(v[j][e], pair_of(act(lo_of(q[e])), act(hi_of(q[e]))));
                        });
                    };
                    if (a.gate_act == LUX_CUDA_GATE_SIGMOID) gated([](float x) { return act_of(x, LUX_CUDA_GATE_SIGMOID); });
                    else if (a.gate_act == LUX_CUDA_GATE_TANH) gated([](float x) { return act_of(x, LUX_CUDA_GATE_TANH); });
                    else gated([](float x) { return x; });
                } else if (a.gate) {
                    values.each([&](int j) {
                        Pair q[4];
                        weight8(base + p.w_off[4], dim, at(j), q);
#pragma unroll
                        for (int e = 0; e < 4; e++) v[j][e] = mul2(v[j][e], q[e]);
                    });
                }
                values.scale_by(a.branch_scale);
            } else {
                values.each([&](int j) {
#pragma unroll
                    for (int e = 0; e < 4; e++) v[j][e] = 0;
                });
            }
            if (a.r) {
                const Pair res = pair_of(a.res_scale, a.res_scale);
                values.each([&](int j) {
                    Pair q[4];
                    row8<RB>(src + p.r_off, at(j), q);
#pragma unroll
                    for (int e = 0; e < 4; e++) v[j][e] = fma2(res, q[e], v[j][e]);
                });
            }
            // the slot has been read: these reads, then the copy engine's writes
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(empty + 8 * slot) : "memory");
            for (slot += p.groups; slot >= p.slots; slot -= p.slots) ph ^= 1;
            const size_t r0 = (size_t)row * dim;
            values.each([&](int j) {
                if (RB) {
                    uint4 q;
                    q.x = pack2(v[j][0]); q.y = pack2(v[j][1]); q.z = pack2(v[j][2]); q.w = pack2(v[j][3]);
                    if (a.r_out) st_row(static_cast<char*>(a.r_out) + (r0 + at(j)) * 2, q);
                    v[j][0] = unpack2(q.x); v[j][1] = unpack2(q.y); v[j][2] = unpack2(q.z); v[j][3] = unpack2(q.w);
                } else if (a.r_out) {
                    store8<false, kWide>(static_cast<char*>(a.r_out) + r0 * 4, Place{at(j)}, v[j]);
                }
            });
            if (!a.out) continue;
            values.norm(a.pre_kind, placed(2), placed(3), shift, weights);
            if (OUT == 0) {
                if (a.out_bf16) values.each([&](int j) { store8<true, kWide>(static_cast<char*>(a.out) + r0 * 2, Place{at(j)}, v[j]); });
                else values.each([&](int j) { store8<false, kWide>(static_cast<char*>(a.out) + r0 * 4, Place{at(j)}, v[j]); });
            } else {
#pragma unroll
                for (int j = 0; j < kChunks; j++) put_codes<OUT ? OUT : 1>(a, v[j], row, at(j), FULL || at(j) < dim);
            }
        }
    }
    __syncthreads();
    if (s_abort) {  // copies in flight get two milliseconds to land
        const uint32_t t0 = clock();
        while ((uint32_t)clock() - t0 < 4000000u) __nanosleep(1000);
        if (tid == 0 && p.error) *p.error = 1;
    }
}

bool make_plan(const BlockNormArgs& a, StreamPlan* p) {
    auto round = [](size_t n, size_t to) { return (int)((n + to - 1) / to * to); };
    const size_t xs = a.x_bf16 ? 2 : 4, rs = a.r_bf16 ? 2 : 4;
    p->group_threads = round((a.dim + 8 * kChunks - 1) / (8 * kChunks), 32);
    if (p->group_threads > kMaxThreads) return false;
    int off = 0;
    const void* const w[5] = {a.post_w, a.post_b, a.pre_w, a.pre_b, a.gate_rows ? nullptr : a.gate};
    for (int k = 0; k < 5; k++) {
        p->w_off[k] = w[k] ? off : -1;
        if (w[k]) off += round(a.dim * 4, 128);
    }
    p->ring_off = off;
    int slot = a.h ? round(a.dim * xs, 128) : 0;
    p->r_off = slot;
    if (a.r) slot += round(a.dim * rs, 128);
    p->gate_off = a.gate && a.gate_rows ? slot : -1;
    if (p->gate_off >= 0) slot += round(a.dim * xs, 128);
    p->slot_bytes = slot;
    p->slots = std::min(kMaxSlots, (kSmemLimit - (int)sizeof(Shared) * kMaxGroups - 1024 - 16 * kMaxSlots - off) / slot);
    if (p->slots < 3) return false;
    p->groups = std::min({kMaxGroups, kMaxThreads / p->group_threads, p->slots});
    p->bar_off = p->ring_off + p->slots * slot;
    p->smem = p->bar_off + 16 * kMaxSlots;
    return true;
}

using StreamKernel = void (*)(BlockNormArgs, StreamPlan);
template <bool XB, bool RB, bool FULL>
StreamKernel pick_out(int format) {
    return format == LUX_CUDA_MX4_E8M0   ? block_norm_stream_kernel<XB, RB, LUX_CUDA_MX4_E8M0, FULL>
           : format == LUX_CUDA_MX4_E4M3 ? block_norm_stream_kernel<XB, RB, LUX_CUDA_MX4_E4M3, FULL>
                                         : block_norm_stream_kernel<XB, RB, 0, FULL>;
}
template <bool FULL>
StreamKernel pick(const BlockNormArgs& a) {
    return a.x_bf16 ? (a.r_bf16 ? pick_out<true, true, FULL>(a.out_format) : pick_out<true, false, FULL>(a.out_format))
                    : (a.r_bf16 ? pick_out<false, true, FULL>(a.out_format) : pick_out<false, false, FULL>(a.out_format));
}

}  // namespace

// It pays by what a row brings with it: the one warp that asks for the rows takes 0.4 us for each, and the weights are on their way for
// a microsecond before the first.  Measured, us, here | a row per block (A: rms | rms, bf16; B: layer | layer, fp32 stream, a sigmoid gate
// per row; KB a row):
//   2048 x 4096 A (16) 14.0 | 17.5    B (32) 24.5 | 35.2     600 x 4096 A 7.0 | 7.6     B 10.8 | 14.8     300 x 4096 A 5.8 | 5.5
//   2048 x 2880 A (11.3) 12.1 | 15.1  B (22.5) 19.4 | 26.8   600 x 2880 A 6.7 | 6.2     B 9.8 | 10.6      8192 x 4096 A 51 | 56
//   2048 x 2048 A (8) 9.7 | 9.9       B (16) 13.6 | 19.1     1184 x 2048 A 7.0 | 6.3    B 9.6 | 11.4      4096 x 1024 A (4) 13.0 | 9.6
bool block_norm_streams(const BlockNormArgs& a, int sm_count) {
    StreamPlan p;
    if (!a.vec || a.dim % 8 || a.rows < (size_t)4 * sm_count || !make_plan(a, &p)) return false;
    return p.slot_bytes >= 11 * 1024 || (p.slot_bytes >= 8 * 1024 && a.rows >= (size_t)12 * sm_count);
}

cudaError_t launch_block_norm_stream(const BlockNormArgs& a, int sm_count, cudaStream_t stream, bool overlap_prev) {
    StreamPlan p;
    if (!make_plan(a, &p)) return cudaErrorInvalidValue;
    p.error = a.error ? a.error : device_error_word();
    const bool full = a.dim == (size_t)p.group_threads * 8 * kChunks;
    StreamKernel kern = full ? pick<true>(a) : pick<false>(a);
    static std::atomic<bool> attr_set[32][64];  // [kernel][device]
    const int which = (full ? 16 : 0) | (a.x_bf16 ? 8 : 0) | (a.r_bf16 ? 4 : 0) | a.out_format;
    if (cudaError_t e = allow_smem(kern, kSmemLimit - (int)sizeof(Shared) * kMaxGroups, attr_set[which])) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)std::min<size_t>(a.rows, sm_count));
    cfg.blockDim = dim3((unsigned)(p.groups * p.group_threads + 32));
    cfg.dynamicSmemBytes = p.smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = overlap_prev ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kern, a, p);
}

}  // namespace luxcuda
