// Around the products of a layer of experts: the router with the sorting of its answers (moe_route), and the weighted sum of a
// token's expert outputs (moe_combine).
//
// moe_route.  One warp takes a token: lane l holds the logits of experts l, l + 32, ... as unsigned keys in the order of the numbers (0: not to
// be chosen); those above a threshold that the lanes' largest give are ranked among themselves (choose).  Then a counting sort that keeps
// the order of the pairs: a block ranks its own pairs (ballots of equal experts within 32 pairs, counts per warp and expert in shared memory),
// and adds where its share of each expert begins.
//   * Few tokens: one block does it all, one launch.
//   * More: a block takes as many neighbouring tokens as it has warps (more where that would be more blocks than SMs) and leaves its counts per
//     expert in a workspace; a second launch adds them up along the blocks, for 32 experts a block; a third puts the pairs in their places.  Up to
//     kFewBlocks blocks the last two are one launch, whose blocks each add up for themselves.  No atomics: a pair's rank must not depend
//     on who comes first.
// Bytes: tokens * experts logits once, 16 bytes a pair out.  Bound by the instructions of the choice (about a thousand a token at 256 experts, best
// 8; 60 % of the issue slots): 8192 tokens 18.2 us, with sigmoid and bias 20.0.  Few tokens: by the latency of a launch, 4 us.
//
// moe_combine.  HBM-bound: a thread takes 8 neighbouring columns of a token, with the loads of up to 8 slots under way (4096 tokens x 8 x 4096,
// fp32 stream: 64 us, 6.1 TB/s); rows that are no whole pieces of 8 on 16-byte boundaries go in several of 4, 2 or 1 (1.3 to 2.9 times the floor,
// 2 x 5003 bf16 the worst).
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
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }
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

// One round of a choice (whole warp): the expert with the largest key, the lowest of equals, is taken out of the lanes' keys; key i of a lane is
// expert lane + 32 i's.  -1: all keys are 0.
template <int VPT, class Key>
__device__ __forceinline__ int take_best(Key (&key)[VPT], int lane) {
    Key best = 0;
    int at = 0;
#pragma unroll
    for (int i = 0; i < VPT; i++)
        if (key[i] > best) { best = key[i]; at = lane + 32 * i; }
    const Key top = warp_max(best);
    if (!top) return -1;
    const int e = (int)__reduce_min_sync(kFull, best == top ? (uint32_t)at : 0x7fffffffu);
#pragma unroll
    for (int i = 0; i < VPT; i++)
        if (lane + 32 * i == e) key[i] = 0;
    return e;
}
__device__ __forceinline__ double wide_score(float v, float bias) { return 1.0 / (1.0 + exp(-(double)v)) + (double)bias; }

// The experts of one token (whole warp).  A lane gets an expert, its slot (-1: none of the top_k) and weight.  VPT: logits per lane.
//
// A threshold first: the top_k-th largest of the lanes' largest keys.  The chosen are among the experts that reach it, mostly two or three more
// than top_k of them; they are gathered, one a lane, in the order of their numbers, and each counts those ahead of it.  Where more reach
// it than a warp has lanes: top_k rounds over all keys.  (Always the rounds: 8192 tokens x 256 experts, best 8: 19 us of a launch.)
//
// WIDE: by sigmoid + bias in fp64; in fp32 two experts next to a border could change places with the rounding of the exponential.  The fp32 keys
// are off by less than 1e-6 (1 + |key|) (the machine's exponential: |v| / 4 + 1/2 U of e^-v's share of at most 1/4, U each from quotient and sums),
// so the chosen are among those that come within twice that of the threshold; only these are looked at in fp64.
template <int VPT, bool BF16, bool WIDE>
__device__ __forceinline__ void choose(const MoeRouteArgs& a, size_t token, int lane, uint32_t* room, int* id, int* slot, float* weight) {
    const size_t row = token * a.ld;
    uint32_t key[VPT], best = 0;
    float mine[WIDE ? 1 : VPT];
#pragma unroll
    for (int i = 0; i < VPT; i++) {
        const int e = lane + 32 * i;
        const float v = e < a.experts ? load_logit<BF16>(a.logits, row + e) : -INFINITY;
        key[i] = order_key(v);
        if constexpr (WIDE) {
            if (key[i]) key[i] = order_key(__fdividef(1.0f, 1.0f + __expf(-v)) + a.bias[e]);
        } else {
            mine[i] = v;
        }
        best = max(best, key[i]);
    }
    uint32_t least = best;
    for (int j = 1; j < a.top_k; j++) {  // (one lane out per round, of equals the lowest)
        const uint32_t top = __reduce_max_sync(kFull, least);
        if (!top) break;
        if (lane == __ffs(__ballot_sync(kFull, least == top)) - 1) least = 0;
    }
    least = max(__reduce_max_sync(kFull, least), 1u);
    if (WIDE && least > 1) {
        const float t = key_value(least);
        least = max(order_key(t - 2e-6f * (1.0f + fabsf(t))), 1u);
    }
    int n = 0;  // experts that reach it
#pragma unroll
    for (int i = 0; i < VPT; i++) {
        const unsigned there = __ballot_sync(kFull, key[i] >= least);
        const int at = n + __popc(there & ((1u << lane) - 1));
        if (key[i] >= least && at < 32) {
            room[at] = key[i];
            room[32 + at] = lane + 32 * i;
        }
        n += __popc(there);
    }
    __syncwarp();
    *id = -1;
    if (n <= 32) {
        if (lane < n) *id = (int)room[32 + lane];
        int ahead = 0;
        if constexpr (WIDE) {
            const unsigned long long w = *id >= 0 ? order_key(wide_score(load_logit<BF16>(a.logits, row + *id), a.bias[*id])) : 0ull;
            for (int j = 0; j < n; j++) {
                const unsigned long long other = __shfl_sync(kFull, w, j);
                ahead += other > w || (other == w && j < lane);
            }
            if (!w) ahead = 32;
        } else {
            const uint32_t w = lane < n ? room[lane] : 0u;
            for (int j = 0; j < n; j++) {
                const uint32_t other = __shfl_sync(kFull, w, j);
                ahead += other > w || (other == w && j < lane);
            }
        }
        *slot = *id >= 0 && ahead < a.top_k ? ahead : -1;
    } else {
        using Key = std::conditional_t<WIDE, unsigned long long, uint32_t>;
        Key all[VPT];
#pragma unroll
        for (int i = 0; i < VPT; i++) {
            if constexpr (WIDE) all[i] = key[i] >= least ? order_key(wide_score(load_logit<BF16>(a.logits, row + lane + 32 * i), a.bias[lane + 32 * i])) : 0ull;
            else all[i] = key[i];
        }
        for (int j = 0; j < a.top_k; j++) {
            const int e = take_best<VPT>(all, lane);
            if (e < 0) break;
            if (lane == j) *id = e;
        }
        *slot = *id >= 0 ? lane : -1;
    }
    __syncwarp();  // (room has been read)
    const bool got = *slot >= 0;
    const float v = got ? load_logit<BF16>(a.logits, row + *id) : 0.0f;
    float w = 0.0f, total = 1.0f;
    if (a.score == LUX_CUDA_SCORE_SIGMOID) {
        w = got ? 1.0f / (1.0f + expf(-v)) : 0.0f;
        if (a.renorm) total = warp_sum(w);
    } else {
        const unsigned first = __ballot_sync(kFull, *slot == 0);  // slot 0 has the largest (or there is none at all)
        const float top = __shfl_sync(kFull, v, first ? __ffs(first) - 1 : 0);
        w = got ? (v == top ? 1.0f : expf(v - top)) : 0.0f;
        if (a.renorm) {
            total = warp_sum(w);
        } else if constexpr (!WIDE) {  // (a bias goes with sigmoids only)
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
    extern __shared__ int smem[];
    const int E = a.experts, k = a.top_k, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, threads = blockDim.x, W = threads >> 5;
    int* start = smem;              // [E + 1]
    int* s_id = start + E + 1;      // [kRoundPairs]
    int* s_rank = s_id + kRoundPairs;
    uint16_t* cnt = reinterpret_cast<uint16_t*>(s_rank + kRoundPairs);  // [W + 1][E]; the last row: the round's counts
    for (int e = threadIdx.x; e <= E; e += threads) start[e] = 0;
    wait_previous();
    const size_t t_lo = (size_t)blockIdx.x * chunk, t_hi = min(t_lo + (size_t)chunk, a.tokens);
    const int per_round = min(chunk, kRoundPairs / k);
    for (size_t t0 = t_lo; t0 < t_hi; t0 += per_round) {
        const int tokens = (int)min((size_t)per_round, t_hi - t0), pairs = tokens * k;
        const int seg = (pairs + W * 32 - 1) / (W * 32) * 32, used = (pairs + seg - 1) / seg;  // pairs a warp ranks; warps that have any
        for (int i = threadIdx.x; i < used * E; i += threads) cnt[i] = 0;
        if constexpr (VPT == 0) {
            for (int i = threadIdx.x; i < pairs; i += threads) {
                const int e = a.ids[t0 * k + i];
                s_id[i] = e >= 0 && e < E ? e : -1;
            }
        } else {
            for (int t = warp; t < tokens; t += W) {
                int id, slot;
                float w;
                choose<VPT, BF16, WIDE>(a, t0 + t, lane, reinterpret_cast<uint32_t*>(s_rank) + warp * 64, &id, &slot, &w);
                const int n = __popc(__ballot_sync(kFull, slot >= 0));  // slots 0 .. n-1
                if (slot >= 0) {
                    s_id[t * k + slot] = id;
                    a.ids[(t0 + t) * k + slot] = id;
                    a.weights[(t0 + t) * k + slot] = w;
                }
                if (lane >= n && lane < k) {  // slots without an expert
                    s_id[t * k + lane] = -1;
                    a.ids[(t0 + t) * k + lane] = -1;
                    a.weights[(t0 + t) * k + lane] = 0.0f;
                }
            }
        }
        __syncthreads();
        const int lo = min(warp * seg, pairs), hi = min(lo + seg, pairs);
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
        for (int e = threadIdx.x; e < E; e += threads) {
            int s = 0;
            for (int w0 = 0; w0 < used; w0 += 8) {
                int c[8];
#pragma unroll
                for (int w = 0; w < 8; w++) c[w] = w0 + w < used ? cnt[(w0 + w) * E + e] : 0;
#pragma unroll
                for (int w = 0; w < 8; w++) {
                    if (w0 + w < used) cnt[(w0 + w) * E + e] = (uint16_t)s;
                    s += c[w];
                }
            }
            if (one) start[e] = s;
            else cnt[W * E + e] = (uint16_t)s;
        }
        if (one) scan_experts(start, start, E);  // (one round: the counts are the whole)
        else __syncthreads();
        for (int i = lo + lane; i < hi; i += 32) {
            const int e = s_id[i], at = e >= 0 ? start[e] + cnt[warp * E + e] + s_rank[i] : -1;
            a.pos[t0 * k + i] = at;
            if (one && e >= 0) a.order[at] = i;
        }
        if (!one) {
            __syncthreads();
            for (int e = threadIdx.x; e < E; e += threads) start[e] += cnt[W * E + e];
            __syncthreads();
        }
    }
    if (one)
        for (int e = threadIdx.x; e <= E; e += threads) a.offsets[e] = start[e];
    else
        for (int e = threadIdx.x; e < E; e += threads) a.hist[(size_t)blockIdx.x * E + e] = start[e];
}

// The second launch: 32 experts a block, warp w a run of the B blocks' counts.  Behind it hist[b][e] is the sum of the blocks before b, hist[B][e] that of
// all.
constexpr int kMaxBlocks = 160;  // (one on each SM, whose registers hold one of 1024 threads: in two rounds, 8192 x 256 22.6 us against 20.0)
__global__ void __launch_bounds__(1024) moe_count_kernel(int* hist, int E, int B) {
    __shared__ int part[32][33];
    wait_previous();
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, e = blockIdx.x * 32 + lane;
    const int lo = w * B / 32, hi = (w + 1) * B / 32;
    int c[(kMaxBlocks + 31) / 32], sum = 0;
#pragma unroll
    for (int i = 0; i < (kMaxBlocks + 31) / 32; i++) c[i] = e < E && lo + i < hi ? __ldcg(hist + (size_t)(lo + i) * E + e) : 0;
#pragma unroll
    for (int i = 0; i < (kMaxBlocks + 31) / 32; i++) sum += c[i];
    part[w][lane] = sum;
    __syncthreads();
    int before = 0;
    for (int i = 0; i < w; i++) before += part[i][lane];
    if (e >= E) return;
#pragma unroll
    for (int i = 0; i < (kMaxBlocks + 31) / 32; i++)
        if (lo + i < hi) {
            hist[(size_t)(lo + i) * E + e] = before;
            before += c[i];
        }
    if (w == 31) hist[(size_t)B * E + e] = before;
}

// The last: the places.
constexpr int kPlaceThreads = 512;
__global__ void __launch_bounds__(kPlaceThreads) moe_place_kernel(const MoeRouteArgs a, int chunk, int B) {
    extern __shared__ int all[];  // [E + 1]
    const int E = a.experts;
    wait_previous();
    for (int e = threadIdx.x; e < E; e += kPlaceThreads) all[e] = __ldcg(a.hist + (size_t)B * E + e);
    scan_experts(all, all, E);
    const uint32_t per = (uint32_t)chunk * a.top_k, pairs = (uint32_t)a.tokens * a.top_k;  // (below 2^31)
    for (uint32_t p = blockIdx.x * kPlaceThreads + threadIdx.x; p < pairs; p += gridDim.x * kPlaceThreads) {
        const int rank = a.pos[p];
        if (rank < 0) continue;
        const int id = a.ids[p], at = all[id] + __ldcg(a.hist + (size_t)(p / per) * E + id) + rank;
        a.pos[p] = at;
        a.order[at] = (int)p;
    }
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i <= E; i += kPlaceThreads) a.offsets[i] = all[i];
}
// Few blocks: every block adds up the counts itself, for its own pairs.  One launch less (with 147 blocks 2.5 us more than it saves).
constexpr int kFewBlocks = 64, kCountThreads = 1024;
__global__ void __launch_bounds__(kCountThreads) moe_count_place_kernel(const MoeRouteArgs a, int chunk) {
    extern __shared__ int smem[];
    const int E = a.experts, B = gridDim.x, EP = (E + 31) & ~31, parts = kCountThreads / EP;  // (EP <= 1024)
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
    for (size_t p = lo + threadIdx.x; p < hi; p += kCountThreads) {
        const int rank = a.pos[p];
        if (rank < 0) continue;
        const int id = a.ids[p], at = all[id] + mine[id] + rank;
        a.pos[p] = at;
        a.order[at] = (int)p;
    }
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i <= E; i += kCountThreads) a.offsets[i] = all[i];
}

// ---- the weighted sum -------------------------------------------------------------------------------------------------
// V neighbouring elements, on a boundary of as many bytes as they have (16 at most)
template <int V, bool BF16>
struct Piece {
    static constexpr int kWords = BF16 ? (V + 1) / 2 : V;
    uint32_t raw[kWords];
    __device__ __forceinline__ void load(const void* p, size_t i) {
        const char* q = static_cast<const char*>(p) + i * (BF16 ? 2 : 4);
        if constexpr (kWords >= 4) {
#pragma unroll
            for (int k = 0; k < kWords; k += 4) {
                const uint4 v = reinterpret_cast<const uint4*>(q)[k / 4];
                raw[k] = v.x; raw[k + 1] = v.y; raw[k + 2] = v.z; raw[k + 3] = v.w;
            }
        } else if constexpr (kWords == 2) {
            const uint2 v = *reinterpret_cast<const uint2*>(q);
            raw[0] = v.x; raw[1] = v.y;
        } else if constexpr (BF16 && V == 1) {
            raw[0] = *reinterpret_cast<const uint16_t*>(q);
        } else {
            raw[0] = *reinterpret_cast<const uint32_t*>(q);
        }
    }
    __device__ __forceinline__ float at(int j) const {
        if constexpr (BF16) return __uint_as_float(j & 1 ? raw[j >> 1] & 0xFFFF0000u : raw[j >> 1] << 16);
        return __uint_as_float(raw[j]);
    }
    __device__ __forceinline__ void put(const float (&v)[V]) {
        if constexpr (BF16) {
#pragma unroll
            for (int j = 0; j < V; j += 2) {
                const __nv_bfloat162 b = __floats2bfloat162_rn(v[j], V > 1 ? v[j + (V > 1)] : 0.0f);
                raw[j / 2] = *reinterpret_cast<const uint32_t*>(&b);
            }
        } else {
#pragma unroll
            for (int j = 0; j < V; j++) raw[j] = __float_as_uint(v[j]);
        }
    }
    __device__ __forceinline__ void store(void* p, size_t i) const {
        char* q = static_cast<char*>(p) + i * (BF16 ? 2 : 4);
        if constexpr (kWords >= 4) {
#pragma unroll
            for (int k = 0; k < kWords; k += 4) reinterpret_cast<uint4*>(q)[k / 4] = make_uint4(raw[k], raw[k + 1], raw[k + 2], raw[k + 3]);
        } else if constexpr (kWords == 2) {
            *reinterpret_cast<uint2*>(q) = make_uint2(raw[0], raw[1]);
        } else if constexpr (BF16 && V == 1) {
            *reinterpret_cast<uint16_t*>(q) = (uint16_t)raw[0];
        } else {
            *reinterpret_cast<uint32_t*>(q) = raw[0];
        }
    }
};
// A thread: R pieces of V columns of a token, `groups` pieces apart; U: slots whose loads are under way together.
template <int V, int R, int U, bool YB, bool OB>
__global__ void __launch_bounds__(256) moe_combine_kernel(const MoeCombineArgs a, size_t groups) {
    wait_previous();
    const size_t pieces = a.dim / V, i = (size_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= groups * a.tokens) return;
    const size_t t = groups * a.tokens <= 0xffffffffu ? (uint32_t)i / (uint32_t)groups : i / groups, c0 = i - t * groups;
    float s[R][V];
    bool in[R];
    Piece<V, OB> o[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
        in[r] = R == 1 || c0 + r * groups < pieces;
        if (a.residual && in[r]) o[r].load(a.residual, t * a.dim + (c0 + r * groups) * V);
    }
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
        for (int j = 0; j < V; j++) s[r][j] = a.residual && in[r] ? o[r].at(j) : 0.0f;
    for (int j0 = 0; j0 < a.top_k; j0 += U) {
        Piece<V, YB> y[U][R];
        float w[U];
        bool there[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const size_t p = t * a.top_k + j0 + u;
            const bool slot = j0 + u < a.top_k;
            const int at = slot ? a.pos[p] : -1;
            there[u] = at >= 0 && (size_t)at < a.y_rows;
            w[u] = slot && a.weights ? a.weights[p] : 1.0f;
#pragma unroll
            for (int r = 0; r < R; r++)
                if (there[u] && in[r]) y[u][r].load(a.y, (size_t)at * a.dim + (c0 + r * groups) * V);
        }
#pragma unroll
        for (int u = 0; u < U; u++)
            if (there[u]) {
#pragma unroll
                for (int r = 0; r < R; r++)
#pragma unroll
                    for (int j = 0; j < V; j++) s[r][j] = in[r] ? fmaf(w[u], y[u][r].at(j), s[r][j]) : 0.0f;
            }
    }
#pragma unroll
    for (int r = 0; r < R; r++)
        if (in[r]) {
            o[r].put(s[r]);
            o[r].store(a.out, t * a.dim + (c0 + r * groups) * V);
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

constexpr int route_warps(int experts) { return experts > 256 ? 16 : 32; }  // of a block (registers for up to 32 logits a lane)
template <int VPT, bool BF16, bool WIDE>
cudaError_t launch_route_t(const MoeRouteArgs& a, int blocks, int chunk, cudaStream_t stream, bool overlap_prev) {
    constexpr int THREADS = 32 * route_warps(VPT * 32);
    auto kern = moe_route_kernel<VPT, BF16, WIDE, THREADS>;
    static std::atomic<bool> attr_set[64];
    if (cudaError_t e = allow_smem(kern, (int)route_smem(LUX_CUDA_MAX_EXPERTS, 32), attr_set)) return e;
    cudaLaunchAttribute attr;
    // few tokens: few warps, whose barriers and prefix sums are short (one token, 64 experts: 5.0 us with 32)
    const int threads = blocks > 1 ? THREADS : std::min(THREADS, 32 * std::max(4, chunk));
    const cudaLaunchConfig_t cfg = config(blocks, threads, route_smem(a.experts, threads / 32), stream, overlap_prev, &attr);
    return cudaLaunchKernelEx(&cfg, kern, a, chunk, blocks == 1);
}
template <int VPT>
cudaError_t launch_route_v(const MoeRouteArgs& a, int blocks, int chunk, cudaStream_t stream, bool overlap_prev) {
    if (a.bias) return a.logits_bf16 ? launch_route_t<VPT, true, true>(a, blocks, chunk, stream, overlap_prev) : launch_route_t<VPT, false, true>(a, blocks, chunk, stream, overlap_prev);
    return a.logits_bf16 ? launch_route_t<VPT, true, false>(a, blocks, chunk, stream, overlap_prev) : launch_route_t<VPT, false, false>(a, blocks, chunk, stream, overlap_prev);
}

}  // namespace

// One block: up to 32 tokens, a token a warp, or two above 256 experts, where a block has 16 warps (64 tokens of 64 experts, two a warp: 10.4 us against 9.0 in
// several blocks), and pairs that fit a round.
int moe_route_blocks(const MoeRouteArgs& a, int sm_count) {
    if (a.tokens <= 32 && a.tokens * a.top_k <= (size_t)kRoundPairs) return 1;
    const size_t most = std::min(sm_count, kMaxBlocks), per = std::max<size_t>(route_warps(a.experts), (a.tokens + most - 1) / most);
    return (int)std::max<size_t>((a.tokens + per - 1) / per, 2);
}
size_t moe_route_workspace_bytes() { return (size_t)(kMaxBlocks + 1) * LUX_CUDA_MAX_EXPERTS * sizeof(int); }

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
    cudaLaunchAttribute attr;
    if (blocks <= kFewBlocks) {
        *launches = 2;
        const int parts = kCountThreads / ((a.experts + 31) & ~31);
        const cudaLaunchConfig_t cfg = config(blocks, kCountThreads, ((size_t)2 * a.experts + 1 + 2 * (size_t)parts * a.experts) * 4, stream, true, &attr);
        return cudaLaunchKernelEx(&cfg, moe_count_place_kernel, a, chunk);
    }
    *launches = 3;
    const cudaLaunchConfig_t count = config((a.experts + 31) / 32, 1024, 0, stream, true, &attr);
    if ((e = cudaLaunchKernelEx(&count, moe_count_kernel, a.hist, a.experts, blocks)) != cudaSuccess) return e;
    const unsigned grid = (unsigned)std::min<size_t>(2 * (size_t)sm_count, (a.tokens * a.top_k + kPlaceThreads - 1) / kPlaceThreads);
    const cudaLaunchConfig_t place = config(grid, kPlaceThreads, ((size_t)a.experts + 1) * 4, stream, true, &attr);
    return cudaLaunchKernelEx(&place, moe_place_kernel, a, chunk, blocks);
}

namespace {
template <int V, int R, int U>
cudaError_t launch_combine_t(const MoeCombineArgs& a, int sm_count, cudaStream_t stream, bool overlap_prev) {
    const size_t groups = (a.dim / V + R - 1) / R, all = groups * a.tokens;
    const unsigned threads = all >= (size_t)sm_count * 256 ? 256 : 64;  // (few: more blocks, on more SMs)
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg = config((unsigned)((all + threads - 1) / threads), threads, 0, stream, overlap_prev, &attr);
    constexpr int UF = V == 8 ? (U + 1) / 2 : U;  // (fp32: as many bytes)
    void (*kern)(MoeCombineArgs, size_t) = a.y_bf16 ? (a.out_bf16 ? moe_combine_kernel<V, R, U, true, true> : moe_combine_kernel<V, R, U, true, false>)
                                                    : (a.out_bf16 ? moe_combine_kernel<V, R, UF, false, true> : moe_combine_kernel<V, R, UF, false, false>);
    return cudaLaunchKernelEx(&cfg, kern, a, groups);
}
}  // namespace

// Rows of whole pieces of eight: eight slots under way, or two and more columns where there are no more slots.  Others: two slots of more columns, which
// leaves room for more threads and wastes less on slots that are not there (3565 x 6 x 7684 bf16 90 us, eight slots 123, one column a thread
// 284; 4463 x 2 x 7772 62, eight 135, 329); eight where there are no more columns than the card has threads (16 x 8 x 5003 4.2 us, two slots 5.1;
// 128 x 8 x 4098 6.6, two slots 5.8).
cudaError_t launch_moe_combine(const MoeCombineArgs& a, int sm_count, cudaStream_t stream, bool overlap_prev) {
    const bool two = a.top_k <= 2 || a.dim * a.tokens > (size_t)sm_count * 2048;
    switch (a.vec) {
        case 8: return a.top_k <= 2 ? launch_combine_t<8, 2, 2>(a, sm_count, stream, overlap_prev) : launch_combine_t<8, 1, 8>(a, sm_count, stream, overlap_prev);
        case 4: return two ? launch_combine_t<4, 4, 2>(a, sm_count, stream, overlap_prev) : launch_combine_t<4, 2, 8>(a, sm_count, stream, overlap_prev);
        case 2: return two ? launch_combine_t<2, 8, 2>(a, sm_count, stream, overlap_prev) : launch_combine_t<2, 4, 8>(a, sm_count, stream, overlap_prev);
        default: return two ? launch_combine_t<1, 8, 2>(a, sm_count, stream, overlap_prev) : launch_combine_t<1, 4, 8>(a, sm_count, stream, overlap_prev);
    }
}

}  // namespace luxcuda
