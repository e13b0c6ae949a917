// Product of two microscaled 4-bit operands (mx4.cuh):  y[M,N] = alpha * x[M,K] . W[N,K]^T, fp32 accumulation in tensor memory.
//
// The tensor cores take the format as it lies: tcgen05.mma with block scales multiplies 64 codes of each operand's row at a time
// with the scales of their blocks, which it reads from tensor memory.  Nothing is dequantised: weights, activations and scales go
// by the copy engine into shared memory, the scale tiles from there by tcgen05.cp into tensor memory, and the tile
// D[n, m] = sum_k W[n, k] x[m, k] (128 rows of W x bm rows of x) accumulates there.
//
// Few rows of x (mx4_tile_kernel): HBM-bound on the weights (K/2 + K/block bytes per row of W), and on the latency of a launch where
// they are few.  With few tiles K is cut over a cluster of up to eight CTAs; each leaves its fp32 tile in its shared memory and all
// add up an equal share of it in the order of K, out of one another's shared memory: no workspace, no atomics, and the sum's order
// follows from the shape alone.  A launch fills its ring with weights while the kernels before it still run.
//   16 x 8192 x 28672, E4M3: 23.5 us, 5.7 TB/s.  One after another, each with its own weights: 1 x 4096 x 11008 6.7 us (floor 3.7),
//   8 x 4096 x 22016 10.7 (7.4), 1 x 1024 x 1024 2.4; 1 x 4096 x 11008 with its quantisation 8.2, 7.6 where
//   that runs beside the product before.
// Many rows (mx4_pair_kernel, further down): bound by what shared memory and L2 give the tensor cores.
//   4096 x 8192 x 28672 304-318 us, 6.1-6.3 PFLOP/s while the chip is cool (under its power limit: 390); 2048 x 4096 x 4096 16.2 us,
//   4.2 PFLOP/s (two rounds of tiles for 1.7 rounds' worth).
#include <cuda.h>

#include <algorithm>
#include <atomic>

#include "internal.h"
#include "mx4.cuh"
#include "mx4_plan.h"

namespace luxcuda {

namespace {

using namespace mx4_plan;

constexpr int kThreads = 128;
constexpr uint32_t kWaitClocks = 4000000000u;

// scale tiles along K per stage
constexpr int stage_tiles(int format) { return kStageK / (4 * mx4_block(format)); }

__device__ __forceinline__ uint32_t s32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint32_t b, uint32_t n) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(b), "r"(n)); }
__device__ __forceinline__ void bar_expect(uint32_t b, uint32_t n) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(b), "r"(n) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t b, uint32_t parity) {
    uint32_t ok;
    asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3; selp.u32 %0, 1, 0, p; }"
                 : "=r"(ok) : "r"(b), "r"(parity), "r"(20000u) : "memory");
    return ok != 0;
}
// Bounded wait (about two seconds of SM clock).  False: it ran out, or another role has given up; *abort is set.
__device__ __forceinline__ bool bar_wait(uint32_t b, uint32_t parity, volatile int* abort) {
    if (bar_try(b, parity)) return true;
    const uint32_t t0 = clock();
    do {
#pragma unroll 1
        for (int i = 0; i < 64; i++)
            if (bar_try(b, parity)) return true;
    } while (!*abort && (uint32_t)clock() - t0 < kWaitClocks);
    *abort = 1;
    return false;
}
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(r));
    return r != 0;
}
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// a scale tile (32 rows of 16 bytes, one behind the other) into four columns, the same in all four quarters of the lanes
__device__ __forceinline__ void tc_copy_scales(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
template <int FMT>
__device__ __forceinline__ void tc_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb, uint32_t accumulate) {
    if (FMT == LUX_CUDA_MX4_E8M0)
        asm volatile("{ .reg .pred p; setp.ne.b32 p, %6, 0;\n"
                     "  tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p; }"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate) : "memory");
    else
        asm volatile("{ .reg .pred p; setp.ne.b32 p, %6, 0;\n"
                     "  tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p; }"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate) : "memory");
}
// Shared-memory descriptors: rows of 128 bytes under the 128-byte swizzle, eight rows 1024 bytes apart; and a scale tile,
// unswizzled, eight rows of 16 bytes 128 bytes apart.
__device__ __forceinline__ uint64_t desc_sw128(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
__device__ __forceinline__ uint64_t desc_scales(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | (uint64_t)(128 >> 4) << 32 | (uint64_t)1 << 46;
}
// Instruction descriptor of the block-scaled 4-bit kinds: A = B = E2M1, D fp32, both K-major, 128 x n; the scale type; which
// bytes of a scale word the MMA takes (E8M0: two of the four).
template <int FMT>
__device__ __forceinline__ constexpr uint32_t mma_idesc(uint32_t n, uint32_t byte) {
    return 1u << 7 | 1u << 10 | (n >> 3) << 17 | (FMT == LUX_CUDA_MX4_E8M0 ? 1u << 23 : 0u) | (kTileN >> 7) << 27 | byte << 29 | byte << 4;
}
__device__ __forceinline__ void tmem_ld16_async(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    tmem_ld16_async(taddr, r);
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 16; i++) asm volatile("" : "+r"(r[i]));
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// shared memory of the cluster's CTA `rank` at this CTA's address
__device__ __forceinline__ float4 lds_cluster(uint32_t addr, uint32_t rank) {
    uint32_t a;
    float4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
    return v;
}

__device__ __forceinline__ float lds_cluster_f32(uint32_t addr, uint32_t rank) {
    uint32_t a;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
}

struct Params {
    const uint8_t *xs, *ws;  // scale tiles
    void* y;
    int* error;
    int M, K, N, y_bf16, y_vec;  // y_vec: y on a 16-byte boundary, N a multiple of 4
    int x_early;                 // x is not being written by a kernel before this one
    float alpha;
    int m_tiles, bm, split;  // tiles along M of bm rows of x (a multiple of 16); CTAs per cluster = parts of K
    int tiles_k;             // scale tiles along K
    int nst, stages, stage_bytes, b_off, sa_off, sb_off, bar_off;
    uint32_t tmem_cols, sf_col;
};

// Rows m = first, first + step, ... below m_cnt of the tile, the sum of what the cluster's CTAs hold of them (in the order of their
// parts of K), to y: a warp per row; a lane takes four neighbouring columns where they can be stored together (VEC), else every
// 32nd.  S: CTAs, at most; U: rows whose loads are under way together.
template <int S, int U, bool VEC>
__device__ __forceinline__ void store_rows(const Params& p, uint32_t part, int first, int step, int m_cnt, int m0, int n0) {
    const int lane = threadIdx.x & 31, n = n0 + (VEC ? lane * 4 : lane), stride = VEC ? 1 : 32;
    for (int m = first; m < m_cnt; m += U * step) {
        float4 v[U][S];
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int j = 0; j < S; j++) {
                v[u][j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (j < p.split && m + u * step < m_cnt) {
                    const uint32_t at = part + (m + u * step) * (kTileN * 4);
                    v[u][j] = VEC ? lds_cluster(at + lane * 16, j)
                                  : make_float4(lds_cluster_f32(at + lane * 4, j), lds_cluster_f32(at + lane * 4 + 128, j), lds_cluster_f32(at + lane * 4 + 256, j),
                                                lds_cluster_f32(at + lane * 4 + 384, j));
                }
            }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (m + u * step >= m_cnt || n >= p.N) continue;
            float4 s = v[u][0];
#pragma unroll
            for (int j = 1; j < S; j++) { s.x += v[u][j].x; s.y += v[u][j].y; s.z += v[u][j].z; s.w += v[u][j].w; }
            const float e[4] = {s.x * p.alpha, s.y * p.alpha, s.z * p.alpha, s.w * p.alpha};
            const size_t at = (size_t)(m0 + m + u * step) * p.N + n;
            if (p.y_bf16) {
                __nv_bfloat16* y = static_cast<__nv_bfloat16*>(p.y) + at;
                if (VEC) {
                    const __nv_bfloat162 lo = __floats2bfloat162_rn(e[0], e[1]), hi = __floats2bfloat162_rn(e[2], e[3]);
                    *reinterpret_cast<uint2*>(y) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (n + i * stride < p.N) y[i * stride] = __float2bfloat16_rn(e[i]);
                }
            } else {
                float* y = static_cast<float*>(p.y) + at;
                if (VEC) {
                    *reinterpret_cast<float4*>(y) = make_float4(e[0], e[1], e[2], e[3]);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (n + i * stride < p.N) y[i * stride] = e[i];
                }
            }
        }
    }
}
template <bool VEC>
__device__ __forceinline__ void store_tile(const Params& p, uint32_t part, int first, int step, int m_cnt, int m0, int n0) {
    if (p.split <= 2) store_rows<2, 8, VEC>(p, part, first, step, m_cnt, m0, n0);
    else if (p.split <= 4) store_rows<4, 4, VEC>(p, part, first, step, m_cnt, m0, n0);
    else store_rows<kMaxSplit, 2, VEC>(p, part, first, step, m_cnt, m0, n0);
}

// A stage's scales into tensor memory and its MMAs.  WHOLE: all of its K is there.
template <int FMT, bool WHOLE>
__device__ __forceinline__ void issue_stage(const Params& p, int st, uint32_t d, uint64_t da, uint64_t db, uint64_t dsa, uint64_t dsb, uint32_t sf, uint32_t idesc,
                                            bool accumulate) {
    constexpr int ST = stage_tiles(FMT);
    const int tiles = WHOLE ? ST : min(ST, p.tiles_k - st * ST), mmas = WHOLE ? kStageK / kMmaK : (p.K - st * kStageK + kMmaK - 1) / kMmaK;
#pragma unroll
    for (int i = 0; i < ST; i++)
        if (WHOLE || i < tiles) {
            tc_copy_scales(sf + i * kScaleCols, dsa + i * (kScaleTile >> 4));
            tc_copy_scales(sf + (ST + i) * kScaleCols, dsb + i * (kScaleTile >> 4));
        }
#pragma unroll
    for (int i = 0; i < kStageK / kMmaK; i++)
        if (WHOLE || i < mmas) {
            const int t = FMT == LUX_CUDA_MX4_E8M0 ? i >> 1 : i;
            const uint32_t byte = FMT == LUX_CUDA_MX4_E8M0 ? (i & 1) * 2 : 0;
            tc_mma<FMT>(d, da + 2 * i, db + 2 * i, idesc | byte << 29 | byte << 4, sf + t * kScaleCols, sf + (ST + t) * kScaleCols, (i > 0 || accumulate) ? 1u : 0u);
        }
}

template <int FMT>
__global__ void __launch_bounds__(kThreads) mx4_tile_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                                                            const __grid_constant__ Params p) {
    constexpr int ST = stage_tiles(FMT);
    extern __shared__ unsigned char smem_raw[];
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort;
    const uint32_t ring = (s32(smem_raw) + 1023u) & ~1023u;
    volatile int* abort = &s_abort;
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const uint32_t full = ring + p.bar_off, empty = full + 8 * kMaxStages, done = empty + 8 * kMaxStages;
    const int rank = p.split == 1 ? 0 : blockIdx.x % p.split, tile = blockIdx.x / p.split;
    const int tm = tile % p.m_tiles, tn = tile / p.m_tiles, m0 = tm * p.bm, n0 = tn * kTileN;
    const int s_lo = p.nst * rank / p.split, s_hi = p.nst * (rank + 1) / p.split, first = min(p.stages, s_hi - s_lo);
    if (tid == 0) {
        for (int i = 0; i < p.stages; i++) {
            bar_init(full + 8 * i, 1);
            bar_init(empty + 8 * i, 1);
        }
        bar_init(done, 1);
        s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s32(&s_tmem)), "r"(p.tmem_cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0);
    const int m_cnt = min(p.bm, p.M - m0);
    const uint32_t n_mma = (uint32_t)(m_cnt + 15) & ~15u;  // rows of x that the MMAs take

    if (warp == 0) {
        if (lane == 0) {
            asm volatile("prefetch.tensormap [%0];" ::"l"(&map_w) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
            auto scales = [&](int st) { return (uint32_t)min(ST, p.tiles_k - st * ST) * kScaleTile; };
            auto load_w = [&](int st, int slot) {
                const uint32_t bar = full + 8 * slot, base = ring + slot * p.stage_bytes, sc = scales(st);
                bar_expect(bar, kABytes + p.bm * 128 + 2 * sc);
                tma_load_2d(base, &map_w, st * 128, n0, bar);
                bulk_load(base + p.sa_off, p.ws + ((size_t)tn * p.tiles_k + st * ST) * kScaleTile, sc, bar);
            };
            auto load_x = [&](int st, int slot) {
                const uint32_t bar = full + 8 * slot, base = ring + slot * p.stage_bytes;
                tma_load_2d(base + p.b_off, &map_x, st * 128, m0, bar);
                bulk_load(base + p.sb_off, p.xs + ((size_t)(m0 >> 7) * p.tiles_k + st * ST) * kScaleTile, scales(st), bar);
            };
            // what lies ahead of the wait for the previous kernel of the stream touches weights only, and x where that kernel leaves it
            for (int i = 0; i < first; i++) load_w(s_lo + i, i);
            if (p.x_early)
                for (int i = 0; i < first; i++) load_x(s_lo + i, i);
            asm volatile("griddepcontrol.wait;" ::: "memory");
            asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
            if (!p.x_early)
                for (int i = 0; i < first; i++) load_x(s_lo + i, i);
            int slot = 0;
            uint32_t ph = 0;
            for (int st = s_lo + first; st < s_hi; st++) {
                if (!bar_wait(empty + 8 * slot, ph, abort)) break;
                load_w(st, slot);
                load_x(st, slot);
                if (++slot == p.stages) { slot = 0; ph ^= 1; }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // (the clock of a bounded wait must not start before the previous kernel has ended: it may itself be waiting, for a peer, for as
        // long as its caller allows)
        const int wait_at = p.x_early ? s_lo + first : s_lo;  // (behind what is loaded ahead of the loader's own wait)
        // The whole warp walks the stages and one elected lane issues: what the instructions take then lives in uniform registers.  (With
        // loops of one lane's own around them a stage took 630 cycles, whatever its loads did: 1 x 4096 x 4096 out of L2, not split,
        // 7.8 us.)
        int slot = 0;
        uint32_t ph = 0;
        bool ok = true;
        const uint32_t stage16 = (uint32_t)p.stage_bytes >> 4, sf0 = tmem + p.sf_col, idesc = mma_idesc<FMT>(n_mma, 0);
        const uint64_t da = desc_sw128(ring), db = desc_sw128(ring + p.b_off), dsa = desc_scales(ring + p.sa_off), dsb = desc_scales(ring + p.sb_off);
        for (int st = s_lo; st < s_hi; st++) {
            if (st == wait_at) asm volatile("griddepcontrol.wait;" ::: "memory");
            if (!__all_sync(0xffffffffu, bar_wait(full + 8 * slot, ph, abort))) { ok = false; break; }
            tc_fence_after();
            const uint32_t at = slot * stage16, sf = sf0 + slot * (2 * ST * kScaleCols);
            const bool whole = (st + 1) * kStageK <= p.K;
            if (elect_one()) {
                if (whole) issue_stage<FMT, true>(p, st, tmem, da + at, db + at, dsa + at, dsb + at, sf, idesc, st > s_lo);
                else issue_stage<FMT, false>(p, st, tmem, da + at, db + at, dsa + at, dsb + at, sf, idesc, st > s_lo);
                tc_commit(empty + 8 * slot);
                if (st + 1 == s_hi) tc_commit(done);
            }
            __syncwarp();
            if (++slot == p.stages) { slot = 0; ph ^= 1; }
        }
        if (!ok) *abort = 1;
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    // every warp: 32 lanes (rows of W) of the tile
    const bool ok = __all_sync(0xffffffffu, bar_wait(done, 0, abort));
    tc_fence_after();
    // The ring is idle (everything that went into it has been consumed): this CTA's sums go there, [row of x][row of W].
    if (ok)
        for (int c0 = 0; c0 < m_cnt; c0 += 16) {
            uint32_t v[16];
            __syncwarp();
            tmem_ld16(tmem + ((uint32_t)(warp * 32) << 16) + c0, v);
#pragma unroll
            for (int j = 0; j < 16; j++) asm volatile("st.shared.u32 [%0], %1;" ::"r"(ring + ((c0 + j) * kTileN + tid) * 4), "r"(v[j]) : "memory");
        }
    // Tensor memory goes back before this CTA waits for another: one that is still waiting for room in it (tcgen05.alloc has no limit)
    // waits only for CTAs that need nothing but their own copies and MMAs, whatever else lies on the SM.
    tc_fence_before();
    __syncthreads();
    if (s_abort) {  // copies and MMAs in flight get two milliseconds to land
        const uint32_t t0 = clock();
        while ((uint32_t)clock() - t0 < 4000000u) __nanosleep(1000);
        if (tid == 0 && p.error) *p.error = 1;
        __syncthreads();
    }
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(p.tmem_cols) : "memory");
    }
    if (p.split > 1) cluster_sync();
    if (ok) {
        const int first = rank + p.split * warp, step = p.split * (kThreads / 32);
        if (p.y_vec) store_tile<true>(p, ring, first, step, m_cnt, m0, n0);
        else store_tile<false>(p, ring, first, step, m_cnt, m0, n0);
    }
    __syncwarp();
    if (p.split > 1) cluster_sync();  // nobody leaves while another may still read its shared memory
}

// ---- many rows of x: pairs of CTAs (cta_group::2) ----------------------------------------------------------------------------
// Two CTAs of a cluster share one stream of MMAs: 256 rows of x (128 from each) times 256 rows of W, of which each stages half.  A
// stage of 256 codes is 32 KB of codes per CTA for 512 cycles of the tensor core at its rate (it takes 700, the tensor pipe is busy
// two thirds of the time and L2 gives 13 TB/s); with tiles of 128 x 128 on single CTAs L2 would have to bring the same in 256.  Rows of codes on
// odd 16-byte boundaries (K / 32 odd) touch five sectors for four: 59.5 us at 3829 x 10272 x 3232, 47.4 at K = 10304.  D takes 256 columns of tensor memory, the scales of the stages in flight the others: those
// of the CTA's own rows of x, and of all 256 rows of W in both CTAs.
//
// One pair per pair of SMs, tiles round robin, x innermost.  10 warps: 0-7 epilogue (warp w: lanes 32*(w%4).., half w/4 of the columns;
// y leaves through shared memory by the copy engine, or, where a row of y is no multiple of 16 bytes, by the warps), 8 loads, 9 MMAs.
constexpr int kPairStages = 5, kPairN = 256, kEpiWarps = 8;
constexpr int kPairThreads = (kEpiWarps + 2) * 32;
constexpr int kPairRowBytes = 128;                        // a row of a block of y on its way out: 64 bf16 or 32 fp32, swizzled
constexpr int kPairBlockBytes = kTileN * kPairRowBytes;   // and the block: 128 rows; two of them, filled and emptied in turn
constexpr int kPairYBytes = 2 * kPairBlockBytes;          // (room for the whole tile would cost a stage: 41.7 us against 40.0 at 2048 x 4096 x 11008)
constexpr uint32_t kPeerBitMask = 0xFEFFFFFFu;            // a shared::cluster address with this bit cleared is CTA 0's copy
constexpr int kEpiBar = 1;

struct PairParams {
    void* y;
    int* error;
    int M, K, N, y_tma;
    float alpha;
    int m_tiles, tiles;   // of 256 rows of x; pairs' tiles
    int tiles_k, nst;
};
constexpr int pair_stage_bytes(int format) { return 2 * kABytes + 3 * stage_tiles(format) * kScaleTile; }
constexpr int pair_smem(int format) { return kPairStages * pair_stage_bytes(format) + kPairYBytes + 8 * (2 * kPairStages + 2) + 1024; }
static_assert(pair_smem(LUX_CUDA_MX4_E4M3) <= kSmemMax - 1024 && pair_smem(LUX_CUDA_MX4_E8M0) <= kSmemMax - 1024, "shared memory of the pair kernel");
static_assert(256 + kPairStages * 3 * stage_tiles(LUX_CUDA_MX4_E4M3) * kScaleCols <= 512, "tensor memory of the pair kernel");

__device__ __forceinline__ void bar_arrive_cta0(uint32_t b) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(b & kPeerBitMask) : "memory");
}
// into this CTA's shared memory, completion counted on CTA 0's barrier
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar & kPeerBitMask) : "memory");
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, uint32_t src, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x), "r"(y), "r"(src) : "memory");
}
// arrives on the barrier at this offset in both CTAs when what was issued so far has completed
__device__ __forceinline__ void tc_commit_pair(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3) : "memory");
}
// in both CTAs, each from its own shared memory into its own tensor memory
__device__ __forceinline__ void tc_copy_scales_pair(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
template <int FMT>
__device__ __forceinline__ void tc_mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb, uint32_t accumulate) {
    if (FMT == LUX_CUDA_MX4_E8M0)
        asm volatile("{ .reg .pred p; setp.ne.b32 p, %6, 0;\n"
                     "  tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p; }"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate) : "memory");
    else
        asm volatile("{ .reg .pred p; setp.ne.b32 p, %6, 0;\n"
                     "  tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p; }"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate) : "memory");
}
// as mma_idesc, 256 x 256
template <int FMT>
__device__ __forceinline__ constexpr uint32_t pair_idesc(uint32_t byte) {
    return 1u << 7 | 1u << 10 | (kPairN >> 3) << 17 | (FMT == LUX_CUDA_MX4_E8M0 ? 1u << 23 : 0u) | (2 * kTileN >> 7) << 27 | byte << 29 | byte << 4;
}
// 32 columns of this thread's lane; the caller waits (tmem_ld_wait) before it uses them
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
// The loads above have arrived.  (The registers pass through it: nothing that uses them moves ahead of the wait.)
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[128]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 128; i++) asm volatile("" : "+r"(r[i]));
}
__device__ __forceinline__ uint32_t lds_u16(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=r"(v) : "r"(a));
    return v;
}
__device__ __forceinline__ uint32_t lds_u32(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a));
    return v;
}
__device__ __forceinline__ void sts_v4(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

// as issue_stage; scales in shared memory and in tensor memory: ST tiles of x; in shared memory then ST tiles of the first 128 rows of W and ST
// of the others, in tensor memory the two side by side
template <int FMT, bool WHOLE>
__device__ __forceinline__ void issue_stage_pair(const PairParams& p, int st, uint32_t d, uint64_t da, uint64_t db, uint64_t ds, uint32_t sf) {
    constexpr int ST = stage_tiles(FMT);
    const int mmas = WHOLE ? kStageK / kMmaK : (p.K - st * kStageK + kMmaK - 1) / kMmaK;
    const uint32_t sb = sf + ST * kScaleCols;
#pragma unroll
    for (int i = 0; i < ST; i++) {  // (past the last tile of a row: whatever lies there, for MMAs that are not issued)
        tc_copy_scales_pair(sf + i * kScaleCols, ds + i * (kScaleTile >> 4));
        tc_copy_scales_pair(sb + 2 * i * kScaleCols, ds + (ST + i) * (kScaleTile >> 4));
        tc_copy_scales_pair(sb + (2 * i + 1) * kScaleCols, ds + (2 * ST + i) * (kScaleTile >> 4));
    }
#pragma unroll
    for (int i = 0; i < kStageK / kMmaK; i++)
        if (WHOLE || i < mmas) {
            const int t = FMT == LUX_CUDA_MX4_E8M0 ? i >> 1 : i;
            tc_mma_pair<FMT>(d, da + 2 * i, db + 2 * i, pair_idesc<FMT>(FMT == LUX_CUDA_MX4_E8M0 ? (i & 1) * 2 : 0), sf + t * kScaleCols, sb + 2 * t * kScaleCols,
                             (st > 0 || i > 0) ? 1u : 0u);
        }
}

template <int FMT, bool YBF16>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
mx4_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_xs,
                const __grid_constant__ CUtensorMap map_ws, const __grid_constant__ CUtensorMap map_y, const __grid_constant__ PairParams p) {
    constexpr int ST = stage_tiles(FMT), STAGE = pair_stage_bytes(FMT), SA = 2 * kABytes, SB = SA + ST * kScaleTile;
    constexpr int SLOT = 3 * ST * kScaleCols;  // columns of scales per stage: ST tiles of x, 2 * ST of W
    extern __shared__ unsigned char smem_raw[];
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort;
    const uint32_t ring = (s32(smem_raw) + 1023u) & ~1023u, stage_y = ring + kPairStages * STAGE, full = stage_y + kPairYBytes;
    const uint32_t empty = full + 8 * kPairStages, tmem_full = empty + 8 * kPairStages, tmem_empty = tmem_full + 8;
    volatile int* abort = &s_abort;
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    uint32_t rank;  // of this CTA in its pair: 0 issues the MMAs of both
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    if (tid == 0) {
        for (int i = 0; i < kPairStages; i++) {
            bar_init(full + 8 * i, 1);   // (CTA 0's) its loader's arrival, with the bytes of both CTAs
            bar_init(empty + 8 * i, 1);  // a commit, in both CTAs
        }
        bar_init(tmem_full, 1);
        bar_init(tmem_empty, 2 * kEpiWarps);  // (CTA 0's) the epilogue warps of both
        s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kEpiWarps + 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s32(&s_tmem)), "n"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // the peer's barriers are there before anything arrives on them
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0);
    // No clock of a bounded wait starts before the previous kernel has ended; ahead of that the loader alone is at work, on weights.
    if (warp != kEpiWarps) asm volatile("griddepcontrol.wait;" ::: "memory");

    if (warp == kEpiWarps) {
        if (lane == 0) {
            asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"(&map_w) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"(&map_xs) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"(&map_ws) : "memory");
            auto load_w = [&](int st, int tn, int slot) {
                const uint32_t bar = full + 8 * slot, base = ring + slot * STAGE;
                if (rank == 0) bar_expect(bar, 2 * STAGE);
                tma_load_2d_pair(base + kABytes, &map_w, st * 128, (tn + (int)rank) * kTileN, bar);
                tma_load_2d_pair(base + SB, &map_ws, 0, tn * p.tiles_k + st * ST, bar);
                tma_load_2d_pair(base + SB + ST * kScaleTile, &map_ws, 0, (tn + 1) * p.tiles_k + st * ST, bar);
            };
            const int first = min(kPairStages, p.nst);  // stages of the first tile whose weights are fetched ahead
            for (int st = 0; st < first; st++) load_w(st, pair / p.m_tiles * 2, st);
            asm volatile("griddepcontrol.wait;" ::: "memory");
            asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
            int slot = 0;
            uint32_t ph = 1;
            bool ok = true;
            for (int tile = pair; tile < p.tiles && ok; tile += pairs) {
                const int tm = tile % p.m_tiles * 2 + (int)rank, tn = tile / p.m_tiles * 2;  // this CTA's tile of x, the pair's first of W (128 rows each)
                for (int st = 0; st < p.nst; st++) {
                    if (tile != pair || st >= first) {
                        if (!bar_wait(empty + 8 * slot, ph, abort)) { ok = false; break; }
                        load_w(st, tn, slot);
                    }
                    tma_load_2d_pair(ring + slot * STAGE, &map_x, st * 128, tm * kTileN, full + 8 * slot);
                    tma_load_2d_pair(ring + slot * STAGE + SA, &map_xs, 0, tm * p.tiles_k + st * ST, full + 8 * slot);
                    if (++slot == kPairStages) { slot = 0; ph ^= 1; }
                }
            }
        }
        __syncwarp();
    } else if (warp == kEpiWarps + 1) {
        if (rank == 0) {
            int slot = 0;
            uint32_t ph = 0, tile_i = 0;
            bool ok = true;
            const uint64_t da = desc_sw128(ring), db = desc_sw128(ring + kABytes), ds = desc_scales(ring + SA);
            for (int tile = pair; tile < p.tiles && ok; tile += pairs, tile_i++) {
                if (!__all_sync(0xffffffffu, bar_wait(tmem_empty, (tile_i & 1) ^ 1, abort))) break;
                tc_fence_after();
                for (int st = 0; st < p.nst; st++) {
                    if (!__all_sync(0xffffffffu, bar_wait(full + 8 * slot, ph, abort))) { ok = false; break; }
                    tc_fence_after();
                    const uint32_t at = slot * (STAGE >> 4), sf = tmem + 256 + slot * SLOT;
                    const bool whole = (st + 1) * kStageK <= p.K;
                    if (elect_one()) {
                        if (whole) issue_stage_pair<FMT, true>(p, st, tmem, da + at, db + at, ds + at, sf);
                        else issue_stage_pair<FMT, false>(p, st, tmem, da + at, db + at, ds + at, sf);
                        tc_commit_pair(empty + 8 * slot);
                        if (st + 1 == p.nst) tc_commit_pair(tmem_full);
                    }
                    __syncwarp();
                    if (++slot == kPairStages) { slot = 0; ph ^= 1; }
                }
            }
        }
    } else {
        // This thread's row of the CTA's 128 rows of x; its columns: half of each block of y that leaves as one.  All 128 of them come into
        // registers first, so that the accumulator is free again after the time of the loads and the next tile's MMAs run while this
        // one is converted and stored.  (Block by block out of tensor memory: 333 us against 322 at 4096 x 8192 x 28672.)
        const int q = warp & 3, half = warp >> 2, row = q * 32 + lane;
        constexpr int kCols = kPairRowBytes / (YBF16 ? 2 : 4), kBlocks = kPairN / kCols, kMine = kCols / 2;
        uint32_t tile_i = 0;
        for (int tile = pair; tile < p.tiles; tile += pairs, tile_i++) {
            const int m0 = (tile % p.m_tiles * 2 + (int)rank) * kTileN, n0 = tile / p.m_tiles * kPairN;
            // (one answer for all of these warps, which meet at a barrier below: some may still have seen the tile when others gave up)
            uint32_t all;
            asm volatile("{ .reg .pred p, q; setp.ne.u32 q, %1, 0; bar.red.and.pred p, %2, %3, q; selp.u32 %0, 1, 0, p; }"
                         : "=r"(all) : "r"((uint32_t)bar_wait(tmem_full, tile_i & 1, abort)), "n"(kEpiBar), "n"(kEpiWarps * 32) : "memory");
            if (!all) break;
            tc_fence_after();
            uint32_t v[128];
            __syncwarp();
            const uint32_t d_lane = tmem + ((uint32_t)(q * 32) << 16) + half * kMine;
#pragma unroll
            for (int b = 0; b < kBlocks; b++) {
                if (YBF16) tmem_ld32(d_lane + b * kCols, v + b * kMine);
                else tmem_ld16_async(d_lane + b * kCols, v + b * kMine);
            }
            tmem_ld_wait(v);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive_cta0(tmem_empty);  // the accumulator may be overwritten
#pragma unroll
            for (int b = 0; b < kBlocks; b++) {
                const uint32_t block = stage_y + (b & 1) * kPairBlockBytes, line = block + row * kPairRowBytes;
                const int c0 = b * kCols;
                uint32_t w[16];  // 64 bytes of the row: pieces 4 * half .. 4 * half + 3
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    if (YBF16)
                        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(__uint_as_float(v[(b * kMine + 2 * i + 1) % 128]) * p.alpha), "f"(__uint_as_float(v[(b * kMine + 2 * i) % 128]) * p.alpha));
                    else
                        w[i] = __float_as_uint(__uint_as_float(v[b * kMine + i]) * p.alpha);
                }
                // the block that this one takes the place of, two back, has been read
                if (p.y_tma && tid == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
                asm volatile("bar.sync %0, %1;" ::"n"(kEpiBar), "n"(kEpiWarps * 32) : "memory");
#pragma unroll
                for (int j = 0; j < 4; j++) sts_v4(line + (((4 * half + j) ^ (row & 7)) << 4), w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
                if (p.y_tma) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // these writes, then the copy engine's reads
                asm volatile("bar.sync %0, %1;" ::"n"(kEpiBar), "n"(kEpiWarps * 32) : "memory");
                if (p.y_tma) {
                    if (tid == 0) {
                        if (m0 < p.M && n0 + c0 < p.N) tma_store_2d(&map_y, block, n0 + c0, m0);
                        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                    }
                } else if (n0 + c0 < p.N) {
                    // sixteen rows per warp, lanes side by side; eight rows' loads under way before the first store
                    constexpr int kPer = kCols / 32;
                    const int r0 = warp * (kTileN / kEpiWarps), rows = p.M - m0 - r0, left = p.N - n0 - c0;
#pragma unroll
                    for (int i0 = 0; i0 < kTileN / kEpiWarps; i0 += 8) {
                        uint32_t e[8][kPer];
#pragma unroll
                        for (int i = 0; i < 8; i++)
#pragma unroll
                            for (int h = 0; h < kPer; h++) {
                                const int r = r0 + i0 + i;
                                const uint32_t src = block + r * kPairRowBytes;
                                if (YBF16) e[i][h] = lds_u16(src + (((4 * h + (lane >> 3)) ^ (r & 7)) << 4) + (lane & 7) * 2);
                                else e[i][h] = lds_u32(src + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4);
                            }
                        const size_t at = (size_t)(m0 + r0 + i0) * p.N + n0 + c0 + lane;
#pragma unroll
                        for (int i = 0; i < 8; i++)
#pragma unroll
                            for (int h = 0; h < kPer; h++)
                                if (i0 + i < rows && 32 * h + lane < left) {
                                    if (YBF16) static_cast<uint16_t*>(p.y)[at + (size_t)i * p.N + 32 * h] = (uint16_t)e[i][h];
                                    else static_cast<uint32_t*>(p.y)[at + (size_t)i * p.N + 32 * h] = e[i][h];
                                }
                    }
                }
            }
        }
        if (tid == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");  // the last block has left
    }
    tc_fence_before();
    __syncthreads();
    if (s_abort) {  // copies and MMAs in flight get two milliseconds to land
        const uint32_t t0 = clock();
        while ((uint32_t)clock() - t0 < 4000000u) __nanosleep(1000);
        if (tid == 0 && p.error) *p.error = 1;
        __syncthreads();
    }
    cluster_sync();  // neither CTA leaves (or frees tensor memory) while the other may still reach into it
    if (warp == kEpiWarps + 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512) : "memory");
    }
}

// codes [rows][K/2 bytes], boxes of 128 bytes x box_rows under the 128-byte swizzle; past the ends they read as zeros
bool encode_codes(const void* codes, int rows, int K, int box_rows, CUtensorMap* map) {
    const EncodeTiledFn encode = encode_tiled_fn();
    if (!encode) {
        set_last_error("mx4_matmul: the driver has no cuTensorMapEncodeTiled");
        return false;
    }
    const cuuint64_t dims[2] = {(cuuint64_t)K / 2, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)K / 2};
    const cuuint32_t box[2] = {128, (cuuint32_t)box_rows}, estr[2] = {1, 1};
    const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(codes), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) set_last_error("cuTensorMapEncodeTiled (codes) failed (%d)", (int)r);
    return r == CUDA_SUCCESS;
}

template <int FMT>
cudaError_t launch_tile(const Mx4MatmulArgs& a, int sm_count, cudaStream_t stream, bool overlap_prev, const char** name) {
    constexpr int ST = stage_tiles(FMT);
    const TilePlan t = plan_tile(a.M, a.K, a.N, ST, sm_count);
    Params p = {};
    p.xs = a.xs; p.ws = a.ws; p.y = a.y; p.error = a.error ? a.error : device_error_word();
    p.M = a.M; p.K = a.K; p.N = a.N; p.y_bf16 = a.y_dtype == LUX_DTYPE_BFLOAT16; p.y_vec = ((uintptr_t)a.y & 15) == 0 && a.N % 4 == 0; p.alpha = a.alpha; p.x_early = overlap_prev && a.x_stable;
    p.bm = t.bm; p.m_tiles = t.m_tiles; p.split = t.split;
    p.tiles_k = mx4_tiles_k(a.K, FMT);
    p.nst = (a.K + kStageK - 1) / kStageK;
    p.b_off = kABytes;
    p.sa_off = p.b_off + p.bm * 128;
    p.sb_off = p.sa_off + ST * kScaleTile;
    p.stages = t.stages; p.stage_bytes = t.stage_bytes;
    p.bar_off = p.stages * p.stage_bytes;
    p.sf_col = t.sf_col; p.tmem_cols = t.tmem_cols;
    const int smem = t.smem;
    if (p.stages > kMaxStages || p.tmem_cols > 512 || smem > kSmemMax - 1024 || t.tiles * p.split > 0x7fffffffll) return cudaErrorInvalidValue;
    CUtensorMap map_x, map_w;
    if (!encode_codes(a.xq, a.M, a.K, p.bm, &map_x) || !encode_codes(a.wq, a.N, a.K, kTileN, &map_w)) return cudaErrorInvalidValue;
    auto kern = mx4_tile_kernel<FMT>;
    static std::atomic<bool> attr_set[64];
    if (cudaError_t e = allow_smem(kern, kSmemMax - 1024, attr_set)) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(t.tiles * p.split));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = p.split;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = overlap_prev ? 2 : 1;
    if (name) *name = FMT == LUX_CUDA_MX4_E8M0 ? "mx4_tile<e8m0>" : "mx4_tile<e4m3>";
    return cudaLaunchKernelEx(&cfg, kern, map_x, map_w, p);
}

// scales as rows of 512 bytes, a box the tiles of one stage
bool encode_scales(const void* scales, long long tiles, int box_tiles, CUtensorMap* map) {
    const cuuint64_t dims[2] = {kScaleTile / 4, (cuuint64_t)tiles}, strides[1] = {kScaleTile};
    const cuuint32_t box[2] = {kScaleTile / 4, (cuuint32_t)box_tiles}, estr[2] = {1, 1};
    const CUresult r = encode_tiled_fn()(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<void*>(scales), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                         CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) set_last_error("cuTensorMapEncodeTiled (scales) failed (%d)", (int)r);
    return r == CUDA_SUCCESS;
}

template <int FMT, bool YBF16>
cudaError_t launch_pair(const Mx4MatmulArgs& a, int sm_count, cudaStream_t stream, bool overlap_prev, const char** name) {
    constexpr int ST = stage_tiles(FMT);
    PairParams p = {};
    p.y = a.y; p.error = a.error ? a.error : device_error_word();
    p.M = a.M; p.K = a.K; p.N = a.N; p.alpha = a.alpha;
    p.m_tiles = (a.M - 1) / (2 * kTileN) + 1;
    const long long tiles = (long long)p.m_tiles * ((a.N - 1) / kPairN + 1);
    p.tiles_k = mx4_tiles_k(a.K, FMT);
    p.nst = (a.K + kStageK - 1) / kStageK;
    const long long x_tiles = (long long)((a.M - 1) / kTileN + 1) * p.tiles_k, w_tiles = (long long)((a.N - 1) / kTileN + 1) * p.tiles_k;
    if (tiles > 0x7fffffff || x_tiles > 0x7fffffff || w_tiles > 0x7fffffff) return cudaErrorInvalidValue;
    p.tiles = (int)tiles;
    CUtensorMap map_x, map_w, map_xs, map_ws, map_y;
    if (!encode_codes(a.xq, a.M, a.K, kTileN, &map_x) || !encode_codes(a.wq, a.N, a.K, kTileN, &map_w) || !encode_scales(a.xs, x_tiles, ST, &map_xs) ||
        !encode_scales(a.ws, w_tiles, ST, &map_ws))
        return cudaErrorInvalidValue;
    const cuuint64_t row_bytes = (cuuint64_t)a.N * (YBF16 ? 2 : 4);
    p.y_tma = row_bytes % 16 == 0 && ((uintptr_t)a.y & 15) == 0;
    map_y = map_x;
    if (p.y_tma) {
        const cuuint64_t dims[2] = {(cuuint64_t)a.N, (cuuint64_t)a.M}, strides[1] = {row_bytes};
        const cuuint32_t box[2] = {(cuuint32_t)(kPairRowBytes / (YBF16 ? 2 : 4)), kTileN}, estr[2] = {1, 1};
        const CUresult r = encode_tiled_fn()(&map_y, YBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, a.y, dims, strides, box, estr,
                                             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        if (r != CUDA_SUCCESS) {
            set_last_error("cuTensorMapEncodeTiled (y) failed (%d)", (int)r);
            return cudaErrorInvalidValue;
        }
    }
    auto kern = mx4_pair_kernel<FMT, YBF16>;
    static std::atomic<bool> attr_set[64];
    if (cudaError_t e = allow_smem(kern, kSmemMax - 1024, attr_set)) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(2 * std::min<long long>(sm_count / 2, tiles)));
    cfg.blockDim = dim3(kPairThreads);
    cfg.dynamicSmemBytes = pair_smem(FMT);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = overlap_prev ? 1 : 0;
    if (name) *name = FMT == LUX_CUDA_MX4_E8M0 ? "mx4_pairs<e8m0>" : "mx4_pairs<e4m3>";
    return cudaLaunchKernelEx(&cfg, kern, map_x, map_w, map_xs, map_ws, map_y, p);
}

// Pairs or single CTAs, by estimates in microseconds whose constants were chosen for the best choices over 62 shapes (129 .. 4096 rows, K
// 512 .. 11008, N 256 .. 28672, both formats; the worst choice costs 15%, the mean half a percent).  A round of tiles costs a pair by its
// stages of K, and more where y is fp32 or its rows are no multiple of 16 bytes; a wave of single CTAs by the stages of a part.
// Measured, us, pairs | single:
//   129 x 4096 x 4096 8.9 | 7.8     256 x 4096 x 11008 11.1 | 12.1     1024 x 4096 x 4096 10.6 | 12.1    3207 x 10272 x 465 20.9 | 21.5
//   200 x 4096 x 4096 8.9 | 7.9     300 x 4096 x 11008 15.1 | 12.1     2048 x 4096 x 4096 16.2 | 23.0    3340 x 4256 x 24487 186 | 330
//   512 x 4096 x 4096 9.2 | 10.2    777 x 2880 x 5003 15.0 | 13.5      158 x 1856 x 498 fp32 9.9 | 5.8   2635 x 1248 x 23907 66 | 139
bool pairs_pay(const Mx4MatmulArgs& a, int sm_count) {
    if (a.M <= kTileN) return false;
    const TilePlan t = plan_tile(a.M, a.K, a.N, stage_tiles(a.format), sm_count);
    const bool f32 = a.y_dtype == LUX_DTYPE_FLOAT32, odd = (long long)a.N * (f32 ? 4 : 2) % 16 != 0;
    const long long nst = (a.K + kStageK - 1) / kStageK, slots = (long long)sm_count * std::max(1, t.per_sm);
    const long long pair_tiles = ((a.M + 255ll) / 256) * ((a.N + 255ll) / 256), rounds = (pair_tiles + sm_count / 2 - 1) / (sm_count / 2);
    const long long waves = (t.tiles * t.split + slots - 1) / slots;
    return 3.4 + rounds * (0.26 * nst + 1.8 + 1.1 * f32 + 1.5 * odd) < waves * (0.66 * ((nst + t.split - 1) / t.split) + 6.8) - 3.4;
}

}  // namespace

cudaError_t launch_mx4_matmul(const Mx4MatmulArgs& a, int sm_count, cudaStream_t stream, bool overlap_prev, const char** name) {
    if (!a.M || !a.N) return cudaSuccess;
    if (pairs_pay(a, sm_count)) {
        auto launch = a.y_dtype == LUX_DTYPE_BFLOAT16 ? (a.format == LUX_CUDA_MX4_E8M0 ? launch_pair<LUX_CUDA_MX4_E8M0, true> : launch_pair<LUX_CUDA_MX4_E4M3, true>)
                                                      : (a.format == LUX_CUDA_MX4_E8M0 ? launch_pair<LUX_CUDA_MX4_E8M0, false> : launch_pair<LUX_CUDA_MX4_E4M3, false>);
        return launch(a, sm_count, stream, overlap_prev, name);
    }
    return a.format == LUX_CUDA_MX4_E8M0 ? launch_tile<LUX_CUDA_MX4_E8M0>(a, sm_count, stream, overlap_prev, name)
                                         : launch_tile<LUX_CUDA_MX4_E4M3>(a, sm_count, stream, overlap_prev, name);
}

}  // namespace luxcuda
