// Product of two microscaled 4-bit operands (mx4.cuh):  y[M,N] = alpha * x[M,K] . W[N,K]^T, fp32 accumulation in tensor memory.
//
// The tensor cores take the format as it lies: tcgen05.mma with block scales multiplies 64 codes of each operand's row at a time
// with the scales of their blocks, which it reads from tensor memory.  Nothing is dequantised: weights, activations and scales go
// by the copy engine into shared memory, the scale tiles from there by tcgen05.cp into tensor memory, and the tile
// D[n, m] = sum_k W[n, k] x[m, k] (128 rows of W x bm rows of x) accumulates there.
//
// Few rows of x: HBM-bound on the weights (K/2 + K/block bytes per row of W).  With few tiles K is cut over a cluster of up to
// eight CTAs; each leaves its fp32 tile in its shared memory and all add up an equal share of it in the order of K, out of one
// another's shared memory: no workspace, no atomics, and the sum's order follows from the shape alone.
#include <cuda.h>

#include <algorithm>
#include <atomic>

#include "internal.h"
#include "mx4.cuh"

namespace luxcuda {

namespace {

constexpr int kStageK = 256;              // codes along K per stage: 128 bytes of a row, one swizzle span
constexpr int kTileN = 128;               // rows of W per tile
constexpr int kTileM = 128;               // rows of x per tile, at most
constexpr int kMmaK = 64;                 // codes along K per MMA
constexpr int kMaxStages = 6;
constexpr int kMaxSplit = 8;              // CTAs of a cluster
constexpr int kThreads = 128;
constexpr int kScaleTile = 512;           // bytes of a scale tile (128 rows x 4 blocks)
constexpr int kScaleCols = 4;             // and its columns of tensor memory
constexpr int kABytes = kTileN * 128;
constexpr uint32_t kWaitClocks = 4000000000u;
constexpr int kSmemMax = 227 * 1024;

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
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float lds_cluster(uint32_t addr, uint32_t rank) {
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
    int M, K, N, y_bf16;
    float alpha;
    int m_tiles, bm, split;  // tiles along M of bm rows of x (a multiple of 16); CTAs per cluster = parts of K
    int tiles_k;             // scale tiles along K
    int nst, stages, stage_bytes, b_off, sa_off, sb_off, bar_off;
    uint32_t tmem_cols, sf_col;
};

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
    const int s_lo = p.nst * rank / p.split, s_hi = p.nst * (rank + 1) / p.split;
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
            // what lies ahead of the wait for the previous kernel of the stream touches weights only
            const int first = min(p.stages, s_hi - s_lo);
            for (int i = 0; i < first; i++) load_w(s_lo + i, i);
            asm volatile("griddepcontrol.wait;" ::: "memory");
            asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
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
        int slot = 0;
        uint32_t ph = 0;
        bool ok = true;
        for (int st = s_lo; st < s_hi; st++) {
            if (!__all_sync(0xffffffffu, bar_wait(full + 8 * slot, ph, abort))) { ok = false; break; }
            tc_fence_after();
            if (elect_one()) {
                const uint32_t base = ring + slot * p.stage_bytes;
                const uint32_t sa = tmem + p.sf_col + slot * (2 * ST * kScaleCols), sb = sa + ST * kScaleCols;
                const int tiles = min(ST, p.tiles_k - st * ST), mmas = min(kStageK / kMmaK, (p.K - st * kStageK + kMmaK - 1) / kMmaK);
                for (int i = 0; i < tiles; i++) {
                    tc_copy_scales(sa + i * kScaleCols, desc_scales(base + p.sa_off + i * kScaleTile));
                    tc_copy_scales(sb + i * kScaleCols, desc_scales(base + p.sb_off + i * kScaleTile));
                }
                const uint64_t da = desc_sw128(base), db = desc_sw128(base + p.b_off);
                for (int i = 0; i < mmas; i++) {
                    const int t = FMT == LUX_CUDA_MX4_E8M0 ? i >> 1 : i;
                    const uint32_t byte = FMT == LUX_CUDA_MX4_E8M0 ? (i & 1) * 2 : 0;
                    tc_mma<FMT>(tmem, da + 2 * i, db + 2 * i, mma_idesc<FMT>(n_mma, byte), sa + t * kScaleCols, sb + t * kScaleCols, (st > s_lo || i > 0) ? 1u : 0u);
                }
                tc_commit(empty + 8 * slot);
                if (st + 1 == s_hi) tc_commit(done);
            }
            __syncwarp();
            if (++slot == p.stages) { slot = 0; ph ^= 1; }
        }
        if (!ok) *abort = 1;
    }
    // every warp: 32 lanes (rows of W) of the tile
    const bool ok = __all_sync(0xffffffffu, bar_wait(done, 0, abort));
    tc_fence_after();
    const int nl = warp * 32 + lane, n = n0 + nl;
    const uint32_t d_lane = tmem + ((uint32_t)(warp * 32) << 16);
    auto put = [&](int m, float v) {
        v *= p.alpha;
        const size_t at = (size_t)(m0 + m) * p.N + n;
        if (p.y_bf16) static_cast<__nv_bfloat16*>(p.y)[at] = __float2bfloat16_rn(v);
        else static_cast<float*>(p.y)[at] = v;
    };
    if (p.split == 1) {
        if (ok)
            for (int c0 = 0; c0 < m_cnt; c0 += 16) {
                uint32_t v[16];
                __syncwarp();
                tmem_ld16(d_lane + c0, v);
                if (n < p.N) {
#pragma unroll
                    for (int j = 0; j < 16; j++)
                        if (c0 + j < m_cnt) put(c0 + j, __uint_as_float(v[j]));
                }
            }
    } else {
        // the ring is idle (everything that went into it has been consumed): this CTA's part of the sums, [row of x][row of W]
        if (ok)
            for (int c0 = 0; c0 < m_cnt; c0 += 16) {
                uint32_t v[16];
                __syncwarp();
                tmem_ld16(d_lane + c0, v);
#pragma unroll
                for (int j = 0; j < 16; j++) asm volatile("st.shared.u32 [%0], %1;" ::"r"(ring + ((c0 + j) * kTileN + nl) * 4), "r"(v[j]) : "memory");
            }
        cluster_sync();
        if (ok && n < p.N)
            for (int m = rank; m < m_cnt; m += p.split) {
                float v[kMaxSplit], s = 0.0f;
#pragma unroll
                for (int j = 0; j < kMaxSplit; j++)
                    if (j < p.split) v[j] = lds_cluster(ring + (m * kTileN + nl) * 4, j);
#pragma unroll
                for (int j = 0; j < kMaxSplit; j++)
                    if (j < p.split) s += v[j];
                put(m, s);
            }
        cluster_sync();  // nobody leaves while another may still read its shared memory
    }
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
    Params p = {};
    p.xs = a.xs; p.ws = a.ws; p.y = a.y; p.error = a.error ? a.error : device_error_word();
    p.M = a.M; p.K = a.K; p.N = a.N; p.y_bf16 = a.y_dtype == LUX_DTYPE_BFLOAT16; p.alpha = a.alpha;
    p.bm = std::min(kTileM, (a.M + 15) & ~15);
    p.m_tiles = (a.M + p.bm - 1) / p.bm;
    p.tiles_k = mx4_tiles_k(a.K, FMT);
    p.nst = (a.K + kStageK - 1) / kStageK;
    const long long tiles = (long long)p.m_tiles * ((a.N + kTileN - 1) / kTileN);
    p.split = (int)std::max(1ll, std::min({(long long)kMaxSplit, (long long)p.nst / 2, 2ll * sm_count / tiles}));
    p.b_off = kABytes;
    p.sa_off = p.b_off + p.bm * 128;
    p.sb_off = p.sa_off + ST * kScaleTile;
    p.stage_bytes = (p.sb_off + ST * kScaleTile + 1023) & ~1023;
    // two CTAs per SM; the parts of the sums take the ring's place
    p.stages = std::max(2, std::min({kMaxStages, (kSmemMax / 2 - 3072) / p.stage_bytes, (p.nst + p.split - 1) / p.split}));
    if (p.split > 1)
        while (p.stages * p.stage_bytes < kTileN * p.bm * 4) p.stages++;
    p.bar_off = p.stages * p.stage_bytes;
    p.sf_col = (p.bm + 31) & ~31;
    p.tmem_cols = 32;
    while (p.tmem_cols < p.sf_col + p.stages * 2 * ST * kScaleCols) p.tmem_cols *= 2;
    const int smem = p.bar_off + 8 * (2 * kMaxStages + 1) + 1024;
    if (p.stages > kMaxStages || p.tmem_cols > 512 || smem > kSmemMax || tiles * p.split > 0x7fffffffll) return cudaErrorInvalidValue;
    CUtensorMap map_x, map_w;
    if (!encode_codes(a.xq, a.M, a.K, p.bm, &map_x) || !encode_codes(a.wq, a.N, a.K, kTileN, &map_w)) return cudaErrorInvalidValue;
    auto kern = mx4_tile_kernel<FMT>;
    static std::atomic<bool> attr_set[64];
    if (cudaError_t e = allow_smem(kern, kSmemMax - 1024, attr_set)) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(tiles * p.split));
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

}  // namespace

cudaError_t launch_mx4_matmul(const Mx4MatmulArgs& a, int sm_count, cudaStream_t stream, bool overlap_prev, const char** name) {
    if (!a.M || !a.N) return cudaSuccess;
    return a.format == LUX_CUDA_MX4_E8M0 ? launch_tile<LUX_CUDA_MX4_E8M0>(a, sm_count, stream, overlap_prev, name)
                                         : launch_tile<LUX_CUDA_MX4_E4M3>(a, sm_count, stream, overlap_prev, name);
}

}  // namespace luxcuda
