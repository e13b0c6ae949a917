// Around the products of a layer of experts: the router with the sorting of its answers (moe_route), and the weighted sum of a
// token's expert outputs (moe_combine).
//
// moe_route.  One warp takes a token: lane l holds the logits of experts l, l + 32, ... as unsigned keys in the order of the numbers (0: not to
// be chosen), and top_k times the warp's largest key goes, of equal ones the lowest expert's.  Then a counting sort that keeps
// the order of the pairs: a block ranks its own pairs (ballots of equal experts within 32 pairs, counts per warp and expert in shared memory),
// and adds where its share of each expert begins.
//   * Few tokens: one block does it all, one launch.
//   * More: up to one block per SM, each with a run of neighbouring tokens; it leaves its counts per expert in a workspace, and a second
//     launch, every block for itself, adds up the counts of the blocks before it.  (No atomics: their order would change nothing here, but
//     a pair's rank must not depend on it.)
// Bytes: tokens * experts logits once, 16 bytes a pair out.  Few tokens are bound by the latency of a launch and of top_k dependent
// reductions.
//
// moe_combine.  HBM-bound: a thread takes 8 neighbouring columns of a token, with the loads of up to 8 slots under way.
#include <algorithm>
#include <type_traits>

#include <cuda_bf16.h>

#include "internal.h"

namespace luxcuda {

namespace {

constexpr int kRoundPairs = 2048;  // pairs that a block ranks at a time
constexpr unsigned kFull = 0xffffffffu;

__device__ __forceinline__ void wait_previous() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

template <bool BF16>
__device__ __forceinline__ float load_logit(const void* p, size_t i) {
    if (BF16) return __uint_as_float((uint32_t) reinterpret_cast<const uint16_t*>(p)[i] << 16);
    return reinterpret_cast<const float*>(p)[i];
}

// Unsigned integers in the order of the numbers; 0 for minus infinity and for what is no number.  (+ 0: both zeros are one number.)
__device__ __forceinline__ uint32_t order_key(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f), k = b & 0x80000000u ? ~b : b | 0x80000000u;
    return v > -INFINITY ? k : 0u;
}
__device__ __forceinline__ unsigned long long order_key(double v) {
    const unsigned long long b = (unsigned long long)__double_as_longlong(v + 0.0), top = 1ull << 63;
    return v > -(double)INFINITY ? (b & top ? ~b : b | top) : 0ull;
}
// the warp's largest key
__device__ __forceinline__ uint32_t warp_max(uint32_t k) { return __reduce_max_sync(kFull, k); }
__device__ __forceinline__ unsigned long long warp_max(unsigned long long k) {
    const uint32_t hi = __reduce_max_sync(kFull, (uint32_t)(k >> 32));
    const uint32_t lo = __reduce_max_sync(kFull, (uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
    return (unsigned long long)hi << 32 | lo;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(kFull, v, d);
    return v;
}

// The experts of one token (whole warp): lane j < top_k gets slot j's expert (-1: none) and weight.  VPT: logits per lane.  WIDE: keys are the
// fp64 sums of sigmoid and bias; in fp32 two experts next to a border could change places with the rounding of the exponential.
template <int VPT, bool BF16, bool WIDE>
__device__ __forceinline__ void choose(const MoeRouteArgs& a, size_t token, int lane, int* id, float* weight) {
    using Key = std::conditional_t<WIDE, unsigned long long, uint32_t>;
    const size_t row = token * a.ld;
    Key key[VPT];
    float mine[WIDE ? 1 : VPT];
#pragma unroll
    for (int i = 0; i < VPT; i++) {
        const int e = lane + 32 * i;
        float v = e < a.experts ? load_logit<BF16>(a.logits, row + e) : -INFINITY;
        if constexpr (WIDE) {
            key[i] = 0;
            if (v > -INFINITY) key[i] = order_key(1.0 / (1.0 + exp(-(double)v)) + (double)a.bias[e]);
        } else {
            mine[i] = v;
            key[i] = order_key(v);
        }
    }
    *id = -1;
    for (int j = 0; j < a.top_k; j++) {
        Key best = 0;
        int at = 0;
#pragma unroll
        for (int i = 0; i < VPT; i++)
            if (key[i] > best) { best = key[i]; at = lane + 32 * i; }
        const Key top = warp_max(best);
        if (!top) break;  // (the same for the whole warp)
        const int e = (int)__reduce_min_sync(kFull, best == top ? (uint32_t)at : 0x7fffffffu);
        if (lane == j) *id = e;
#pragma unroll
        for (int i = 0; i < VPT; i++)
            if (lane + 32 * i == e) key[i] = 0;
    }
    const bool got = *id >= 0;
    const float v = got ? load_logit<BF16>(a.logits, row + *id) : 0.0f;
    float w = 0.0f, total = 1.0f;
    if (a.score == LUX_CUDA_SCORE_SIGMOID) {
        w = got ? 1.0f / (1.0f + expf(-v)) : 0.0f;
        if (a.renorm) total = warp_sum(w);
    } else {
        const float top = __shfl_sync(kFull, v, 0);  // slot 0 has the largest (or there is none at all)
        w = got ? (v == top ? 1.0f : expf(v - top)) : 0.0f;
        if (a.renorm) {
            total = warp_sum(w);
        } else if constexpr (!WIDE) {
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < VPT; i++) s += !(mine[i] > -INFINITY) ? 0.0f : mine[i] == top ? 1.0f : expf(mine[i] - top);
            total = warp_sum(s);
        }
    }
    *weight = total > 0.0f ? a.scale * (w / total) : 0.0f;
}

// Whole block: base[e] = sum of n[0 .. e), base[experts] = the whole; both in shared memory (they may be the same array).
__device__ __forceinline__ void scan_experts(const int* n, int* base, int experts) {
    __syncthreads();
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x, per = (experts + 31) / 32, lo = min(lane * per, experts), hi = min(lo + per, experts);
        int s = 0;
        for (int e = lo; e < hi; e++) s += n[e];
        int before = s;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int v = __shfl_up_sync(kFull, before, d);
            if (lane >= d) before += v;
        }
        before -= s;
        for (int e = lo; e < hi; e++) {
            const int c = n[e];
            base[e] = before;
            before += c;
        }
        if (lane == 31) base[experts] = before;
    }
    __syncthreads();
}

// VPT 0: the experts are given.  one: the only block, which finishes the sort, too.
// A round: as many tokens as s_id has room for.  A pair's rank among the block's pairs of its expert is start[e] (the rounds before) +
// cnt[warp][e] (the warps before, 16 bits: a round has fewer pairs) + its rank within the warp's run of pairs.
template <int VPT, bool BF16, bool WIDE, int THREADS>
__global__ void __launch_bounds__(THREADS) moe_route_kernel(const MoeRouteArgs a, int chunk, bool one) {
    constexpr int W = THREADS / 32;
    extern __shared__ int smem[];
    const int E = a.experts, k = a.top_k, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int* start = smem;              // [E + 1]
    int* s_id = start + E + 1;      // [kRoundPairs]
    int* s_rank = s_id + kRoundPairs;
    uint16_t* cnt = reinterpret_cast<uint16_t*>(s_rank + kRoundPairs);  // [W + 1][E]; the last row: the round's counts
    for (int e = threadIdx.x; e <= E; e += THREADS) start[e] = 0;
    wait_previous();
    const size_t t_lo = (size_t)blockIdx.x * chunk, t_hi = min(t_lo + (size_t)chunk, a.tokens);
    const int per_round = min(chunk, kRoundPairs / k);
    for (size_t t0 = t_lo; t0 < t_hi; t0 += per_round) {
        const int tokens = (int)min((size_t)per_round, t_hi - t0), pairs = tokens * k;
        for (int i = threadIdx.x; i < W * E; i += THREADS) cnt[i] = 0;
        if constexpr (VPT == 0) {
            for (int i = threadIdx.x; i < pairs; i += THREADS) {
                const int e = a.ids[t0 * k + i];
                s_id[i] = e >= 0 && e < E ? e : -1;
            }
        } else {
            for (int t = warp; t < tokens; t += W) {
                int id;
                float w;
                choose<VPT, BF16, WIDE>(a, t0 + t, lane, &id, &w);
                if (lane < k) {
                    s_id[t * k + lane] = id;
                    a.ids[(t0 + t) * k + lane] = id;
                    a.weights[(t0 + t) * k + lane] = w;
                }
            }
        }
        __syncthreads();
        const int seg = (pairs + W * 32 - 1) / (W * 32) * 32, lo = min(warp * seg, pairs), hi = min(lo + seg, pairs);
        for (int i0 = lo; i0 < hi; i0 += 32) {
            const int i = i0 + lane, e = i < hi ? s_id[i] : -1;
            const unsigned same = __match_any_sync(kFull, e);
            int before = 0;
            if (e >= 0) {
                before = cnt[warp * E + e];
                s_rank[i] = before + __popc(same & ((1u << lane) - 1));
            }
            __syncwarp();
            if (e >= 0 && lane == __ffs(same) - 1) cnt[warp * E + e] = (uint16_t)(before + __popc(same));
            __syncwarp();
        }
        __syncthreads();
        for (int e = threadIdx.x; e < E; e += THREADS) {
            int s = 0;
            for (int w = 0; w < W; w++) {
                const int c = cnt[w * E + e];
                cnt[w * E + e] = (uint16_t)s;
                s += c;
            }
            cnt[W * E + e] = (uint16_t)s;
            if (one) start[e] = s;
        }
        if (one) scan_experts(start, start, E);  // (one round: the counts are the whole)
        else __syncthreads();
        for (int i = lo + lane; i < hi; i += 32) {
            const int e = s_id[i], at = e >= 0 ? start[e] + cnt[warp * E + e] + s_rank[i] : -1;
            a.pos[t0 * k + i] = at;
            if (one && e >= 0) a.order[at] = i;
        }
        __syncthreads();
        if (!one)
            for (int e = threadIdx.x; e < E; e += THREADS) start[e] += cnt[W * E + e];
        __syncthreads();
    }
    if (one)
        for (int e = threadIdx.x; e <= E; e += THREADS) a.offsets[e] = start[e];
    else
        for (int e = threadIdx.x; e < E; e += THREADS) a.hist[(size_t)blockIdx.x * E + e] = start[e];
}

// The second launch: where each block's share of an expert begins, then the places.  Shared memory: two counts per expert and part of
// the blocks.
constexpr int kPlaceThreads = 1024;
__global__ void __launch_bounds__(kPlaceThreads) moe_place_kernel(const MoeRouteArgs a, int chunk) {
    extern __shared__ int smem[];
    const int E = a.experts, B = gridDim.x, EP = (E + 31) & ~31, parts = kPlaceThreads / EP;  // (EP <= 1024)
    int* all = smem;                    // [E + 1]
    int* mine = all + E + 1;            // [E]: of the blocks before this one
    int* part = mine + E;               // [2][parts][E]
    wait_previous();
    // thread (q, e): blocks [q*B/parts, (q+1)*B/parts) of expert e
    const int e = threadIdx.x % EP, q = threadIdx.x / EP;
    if (q < parts && e < E) {
        const int lo = q * B / parts, hi = (q + 1) * B / parts;
        int before = 0, sum = 0;
#pragma unroll 16
        for (int b = lo; b < hi; b++) {
            const int c = __ldcg(a.hist + (size_t)b * E + e);
            sum += c;
            before += b < (int)blockIdx.x ? c : 0;
        }
        part[q * E + e] = sum;
        part[(parts + q) * E + e] = before;
    }
    __syncthreads();
    if (threadIdx.x < E) {
        int before = 0, sum = 0;
        for (int i = 0; i < parts; i++) {
            sum += part[i * E + threadIdx.x];
            before += part[(parts + i) * E + threadIdx.x];
        }
        all[threadIdx.x] = sum;
        mine[threadIdx.x] = before;
    }
    scan_experts(all, all, E);
    const size_t k = a.top_k, lo = (size_t)blockIdx.x * chunk * k, hi = min(lo + (size_t)chunk * k, a.tokens * k);
    for (size_t p = lo + threadIdx.x; p < hi; p += kPlaceThreads) {
        const int rank = a.pos[p];
        if (rank < 0) continue;
        const int id = a.ids[p], at = all[id] + mine[id] + rank;
        a.pos[p] = at;
        a.order[at] = (int)p;
    }
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i <= E; i += kPlaceThreads) a.offsets[i] = all[i];
}

// ---- the weighted sum -------------------------------------------------------------------------------------------------
template <bool BF16>
__device__ __forceinline__ float load1(const void* p, size_t i) {
    if (BF16) return __uint_as_float((uint32_t) reinterpret_cast<const uint16_t*>(p)[i] << 16);
    return reinterpret_cast<const float*>(p)[i];
}
// V neighbouring elements (8 from a 16-byte boundary, or one)
template <int V, bool BF16>
struct Piece {
    uint4 raw[BF16 ? 1 : 2];
    __device__ __forceinline__ void load(const void* p, size_t i) {
        if constexpr (V == 1) {
            raw[0].x = __float_as_uint(load1<BF16>(p, i));
        } else if constexpr (BF16) {
            raw[0] = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p) + i);
        } else {
            const uint4* q = reinterpret_cast<const uint4*>(reinterpret_cast<const float*>(p) + i);
            raw[0] = q[0];
            raw[1] = q[1];
        }
    }
    __device__ __forceinline__ float at(int j) const {
        if constexpr (V == 1) return __uint_as_float(raw[0].x);
        const uint32_t* w = &raw[0].x;
        if constexpr (BF16) return __uint_as_float(j & 1 ? w[j >> 1] & 0xFFFF0000u : w[j >> 1] << 16);
        return __uint_as_float(w[j]);
    }
};
template <int V, bool YB, bool OB>
__global__ void __launch_bounds__(256) moe_combine_kernel(const MoeCombineArgs a) {
    wait_previous();
    const size_t per_row = (a.dim + V - 1) / V, i = (size_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= per_row * a.tokens) return;
    const size_t t = per_row * a.tokens <= 0xffffffffu ? (uint32_t)i / (uint32_t)per_row : i / per_row, col = (i - t * per_row) * V;
    constexpr int U = YB || V == 1 ? 8 : 4;  // slots whose loads are under way together
    float s[V];
    Piece<V, OB> r;
    if (a.residual) r.load(a.residual, t * a.dim + col);
#pragma unroll
    for (int j = 0; j < V; j++) s[j] = a.residual ? r.at(j) : 0.0f;
    for (int j0 = 0; j0 < a.top_k; j0 += U) {
        Piece<V, YB> y[U];
        float w[U];
        bool there[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const size_t p = t * a.top_k + j0 + u;
            const bool slot = j0 + u < a.top_k;
            const int at = slot ? a.pos[p] : -1;
            there[u] = at >= 0 && (size_t)at < a.y_rows;
            w[u] = slot && a.weights ? a.weights[p] : 1.0f;
            if (there[u]) y[u].load(a.y, (size_t)at * a.dim + col);
        }
#pragma unroll
        for (int u = 0; u < U; u++)
            if (there[u]) {
#pragma unroll
                for (int j = 0; j < V; j++) s[j] = fmaf(w[u], y[u].at(j), s[j]);
            }
    }
    const size_t o = t * a.dim + col;
    if constexpr (V == 1) {
        if (OB) reinterpret_cast<__nv_bfloat16*>(a.out)[o] = __float2bfloat16_rn(s[0]);
        else reinterpret_cast<float*>(a.out)[o] = s[0];
    } else if constexpr (OB) {
        uint4 v;
        uint32_t* w = &v.x;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(s[2 * j], s[2 * j + 1]);
            w[j] = *reinterpret_cast<const uint32_t*>(&b);
        }
        *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(a.out) + o) = v;
    } else {
        float4* q = reinterpret_cast<float4*>(reinterpret_cast<float*>(a.out) + o);
        q[0] = make_float4(s[0], s[1], s[2], s[3]);
        q[1] = make_float4(s[4], s[5], s[6], s[7]);
    }
}

cudaLaunchConfig_t config(unsigned grid, unsigned threads, size_t smem, cudaStream_t stream, bool overlap_prev, cudaLaunchAttribute* attr) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    attr->id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr->val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = overlap_prev ? 1 : 0;
    return cfg;
}

constexpr size_t route_smem(int experts, int warps) { return ((size_t)experts + 1 + 2 * kRoundPairs) * 4 + ((size_t)warps + 1) * experts * 2; }

template <int VPT, bool BF16, bool WIDE>
cudaError_t launch_route_t(const MoeRouteArgs& a, int blocks, int chunk, cudaStream_t stream, bool overlap_prev) {
    constexpr int THREADS = VPT > 8 || WIDE ? 512 : 1024;  // (registers for up to 32 logits a lane)
    auto kern = moe_route_kernel<VPT, BF16, WIDE, THREADS>;
    static std::atomic<bool> attr_set[64];
    if (cudaError_t e = allow_smem(kern, (int)route_smem(LUX_CUDA_MAX_EXPERTS, THREADS / 32), attr_set)) return e;
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg = config(blocks, THREADS, route_smem(a.experts, THREADS / 32), stream, overlap_prev, &attr);
    return cudaLaunchKernelEx(&cfg, kern, a, chunk, blocks == 1);
}
template <int VPT>
cudaError_t launch_route_v(const MoeRouteArgs& a, int blocks, int chunk, cudaStream_t stream, bool overlap_prev) {
    if (a.bias) return a.logits_bf16 ? launch_route_t<VPT, true, true>(a, blocks, chunk, stream, overlap_prev) : launch_route_t<VPT, false, true>(a, blocks, chunk, stream, overlap_prev);
    return a.logits_bf16 ? launch_route_t<VPT, true, false>(a, blocks, chunk, stream, overlap_prev) : launch_route_t<VPT, false, false>(a, blocks, chunk, stream, overlap_prev);
}

}  // namespace

// One block: as long as its warps have no more than two tokens each and the pairs fit a round.
int moe_route_blocks(const MoeRouteArgs& a, int sm_count) {
    if (a.tokens <= 64 && a.tokens * a.top_k <= (size_t)kRoundPairs) return 1;
    const size_t per = std::max<size_t>(16, (a.tokens + sm_count - 1) / sm_count);
    const size_t blocks = (a.tokens + per - 1) / per;
    return (int)std::max<size_t>(blocks, 2);
}
size_t moe_route_workspace_bytes(int sm_count) { return (size_t)sm_count * LUX_CUDA_MAX_EXPERTS * sizeof(int); }

cudaError_t launch_moe_route(const MoeRouteArgs& a, int sm_count, cudaStream_t stream, bool overlap_prev, int* launches) {
    const int blocks = moe_route_blocks(a, sm_count), chunk = std::max(1, (int)((a.tokens + blocks - 1) / blocks));
    cudaError_t e;
    *launches = 1;
    if (!a.logits) e = launch_route_t<0, false, false>(a, blocks, chunk, stream, overlap_prev);
    else if (a.experts <= 32) e = launch_route_v<1>(a, blocks, chunk, stream, overlap_prev);
    else if (a.experts <= 64) e = launch_route_v<2>(a, blocks, chunk, stream, overlap_prev);
    else if (a.experts <= 128) e = launch_route_v<4>(a, blocks, chunk, stream, overlap_prev);
    else if (a.experts <= 256) e = launch_route_v<8>(a, blocks, chunk, stream, overlap_prev);
    else if (a.experts <= 512) e = launch_route_v<16>(a, blocks, chunk, stream, overlap_prev);
    else e = launch_route_v<32>(a, blocks, chunk, stream, overlap_prev);
    if (e != cudaSuccess || blocks == 1) return e;
    *launches = 2;
    cudaLaunchAttribute attr;
    const int parts = kPlaceThreads / ((a.experts + 31) & ~31);
    const cudaLaunchConfig_t cfg = config(blocks, kPlaceThreads, ((size_t)2 * a.experts + 1 + 2 * (size_t)parts * a.experts) * 4, stream, true, &attr);
    return cudaLaunchKernelEx(&cfg, moe_place_kernel, a, chunk);
}

cudaError_t launch_moe_combine(const MoeCombineArgs& a, cudaStream_t stream, bool overlap_prev) {
    const size_t pieces = (a.vec ? a.dim / 8 : a.dim) * a.tokens;
    const unsigned threads = pieces >= 148 * 256 ? 256 : 64;  // (few pieces: more blocks, on more SMs)
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg = config((unsigned)((pieces + threads - 1) / threads), threads, 0, stream, overlap_prev, &attr);
    void (*kern)(MoeCombineArgs) = a.vec ? (a.y_bf16 ? (a.out_bf16 ? moe_combine_kernel<8, true, true> : moe_combine_kernel<8, true, false>)
                                                     : (a.out_bf16 ? moe_combine_kernel<8, false, true> : moe_combine_kernel<8, false, false>))
                                         : (a.y_bf16 ? (a.out_bf16 ? moe_combine_kernel<1, true, true> : moe_combine_kernel<1, true, false>)
                                                     : (a.out_bf16 ? moe_combine_kernel<1, false, true> : moe_combine_kernel<1, false, false>));
    return cudaLaunchKernelEx(&cfg, kern, a);
}

}  // namespace luxcuda
