// Products grouped by expert for many rows an expert (qmatmul_experts), bf16 activations, affine weights:
//   y[i] = epilogue(x[row(i)] . dequant(Wq[e])^T + bias[e]),   offsets[e] <= i < offsets[e+1]
// The roles of qmm_tc.cu's one-CTA kernel on tiles of 128 rows of an expert's W against up to bm of its rows of x; tensor-bound where experts
// have 150 rows and more, bound by dequantisation below (a k-stage of 128 takes 0.45 us of it whatever the rows).
//   * The tiles follow from the offsets in device memory: every CTA scans them at its start (an expert's rows are cut into as few tiles as
//     bm allows, all of one height), then takes every gridDim.x-th tile of the whole list; neighbouring CTAs share an expert's weights or
//     rows of x at the same time.
//   * The matrix instruction's N is the tile's own height, rounded up to 16: a tile of 40 rows takes 48 rows' time.
//   * Rows of x: sorted ones by TMA boxes of 16 rows, a box per lane; gathered ones by TMA gathers of 4 rows each, whose indices the lanes hold
//     for the tile.  (A row of x that does not exist has an index past the tensor's end, which reads as zeros.)
//   * Gated: a tile is eight groups of eight rows of gate and the eight of up that go with them, one TMA box of the weights seen as
//     [expert][group of 8][half][8][byte].  Tensor memory is then read in the shape that leaves a row and the row eight further on in one
//     thread: no exchange between the two halves.
#include <algorithm>
#include <atomic>

#include "epilogue.cuh"
#include "groups.cuh"
#include "qmm_roles.cuh"

namespace luxcuda {

namespace {

constexpr int kBoxRows = 16;    // rows of x per TMA box
constexpr int kGatherRows = 4;  // ... and per gather
static_assert(kDqGroups == kStagesB, "a group always owns the same slot");

struct ExpertGemm {
    const __nv_bfloat16* scales;
    const __nv_bfloat16* biases;
    const float* bias;
    const int *offsets, *order;
    void* y;
    int* error;
    int experts, rows, x_rows, K, N, gshift, act, y_bf16, y_vec;
    int bm, n_tiles, w_slots, most;  // rows of x per tile, at most; tiles along N; tiles in all, at most
    uint32_t top_k;
};

struct Control {
    uint64_t full[kStagesB], empty[kStagesB], wfull[kDqGroups * kMaxWSlots], wempty[kDqGroups * kMaxWSlots], tmem_full, tmem_empty;
    uint32_t tmem_base;
    int abort_flag;
};
static_assert(sizeof(Control) <= kGemmCtlBytes, "the plan's share of shared memory");

// Tiles of an expert with n rows: how many along its rows, and their height.
__device__ __forceinline__ int row_tiles(int n, int bm) { return (n + bm - 1) / bm; }

// The CTA's tiles (the interface of TileIter), each with its expert and rows.
struct GroupTiles {
    const int *off, *first;  // [experts + 1] in shared memory: first rows, first tiles
    int tile_, nst, e, nt, m0, rows;
    __device__ __forceinline__ void init(const ExpertGemm& p, const int* tables, int nst_) {
        off = tables;
        first = tables + p.experts + 1;
        nst = nst_;
        tile_ = blockIdx.x;
        e = 0;
        if (valid(p)) locate(p);
    }
    __device__ __forceinline__ bool valid(const ExpertGemm& p) const { return tile_ < first[p.experts]; }
    __device__ __forceinline__ void locate(const ExpertGemm& p) {
        while (first[e + 1] <= tile_) e++;
        const int n = off[e + 1] - off[e], mt = row_tiles(n, p.bm), at = tile_ - first[e], m = at % mt;
        const int h = ((n + mt - 1) / mt + 15) & ~15;
        nt = at / mt;
        m0 = off[e] + m * h;
        rows = min(h, n - m * h);
    }
    __device__ __forceinline__ void next(const ExpertGemm& p) {
        tile_ += gridDim.x;
        if (valid(p)) locate(p);
    }
};
// ... as weight_producer and dequant_role want it
struct GroupSeg : GroupTiles {
    const ExpertGemm* p;
    __device__ __forceinline__ bool valid() const { return GroupTiles::valid(*p); }
    __device__ __forceinline__ int s_lo() const { return 0; }
    __device__ __forceinline__ int s_hi() const { return nst; }
    __device__ __forceinline__ void next() { GroupTiles::next(*p); }
};

__device__ __forceinline__ void tma_load_5d(void* dst, const CUtensorMap* map, int a, int b, int c, int d, int e, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];"
        ::"r"(s32(dst)), "l"(map), "r"(a), "r"(b), "r"(c), "r"(d), "r"(e), "r"(s32(bar)) : "memory");
}
__device__ __forceinline__ void tma_gather4(uint32_t dst, const CUtensorMap* map, int x, const int (&row)[4], uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];"
        ::"r"(dst), "l"(map), "r"(x), "r"(row[0]), "r"(row[1]), "r"(row[2]), "r"(row[3]), "r"(s32(bar)) : "memory");
}
// Lanes 16 .. of a quarter of tensor memory, 16 columns: thread t gets row t/4, columns 2(t%4) and the next in r[0..1], row t/4 + 8 in r[2..3], and
// the same of the eight columns behind in r[4..7].
__device__ __forceinline__ void tmem_ld_16x256b_x2(uint32_t taddr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr));
}

template <int BITS, bool GATED, bool GATHER>
__global__ void __launch_bounds__(kNumThreads, 1)
qmm_experts_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ ExpertGemm p) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    unsigned char* sB = smem;  // [kStagesB][kSub][bm rows][128 B], swizzled (TMA)
    const uint32_t b_bytes = (uint32_t)p.bm * 128;
    unsigned char* sW = sB + (size_t)kStagesB * kSub * b_bytes;  // [kDqGroups][w_slots][128 rows][64 B], 64-byte swizzle (TMA)
    unsigned char* sEpi = sW + (size_t)kDqGroups * p.w_slots * kWUnitBytes;  // [kEpiWarps][16 rows of x][32 columns] bf16
    Control* ctl = reinterpret_cast<Control*>(sEpi + (size_t)kEpiWarps * kEpiStageBytes);
    int* off = reinterpret_cast<int*>(reinterpret_cast<unsigned char*>(ctl) + kGemmCtlBytes);  // tables of GroupTiles
    int* first = off + p.experts + 1;
    volatile int* abort_flag = &ctl->abort_flag;

    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // (uniform for the compiler too)
    const int nks = p.K / kBK, nst = (nks + kSub - 1) / kSub;

    if (tid == 0) {
        for (int s = 0; s < kStagesB; s++) {
            mbar_init(&ctl->full[s], 4 + 1);  // the owning group's four warps + the producer of x (with its byte count)
            mbar_init(&ctl->empty[s], 1);     // one tcgen05.commit
        }
        for (int g = 0; g < kDqGroups * kMaxWSlots; g++) {
            mbar_init(&ctl->wfull[g], 1);
            mbar_init(&ctl->wempty[g], 4);
        }
        mbar_init(&ctl->tmem_full, 1);
        mbar_init(&ctl->tmem_empty, kEpiWarps);
        ctl->abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // (tensor memory behind the wait: a kernel before this one may still want it)
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (warp == kMmaWarp) tmem_alloc(&ctl->tmem_base, kTmemCols);
    tc_fence_before();
    group_tables(off, first, p.offsets, p.experts, p.rows, p.most, [&](int n) { return row_tiles(n, p.bm) * p.n_tiles; });
    tc_fence_after();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t tmem_base = __shfl_sync(0xffffffffu, ctl->tmem_base, 0);
    GroupSeg seg;
    seg.p = &p;
    seg.init(p, off, nst);

    if (warp == kTmaWarp) {
        // ---------------- rows of x: the whole warp, a box (or four gathers) per lane and stage ----------------
        if (lane == 0) {
            asm volatile("prefetch.tensormap [%0];" ::"l"(&tmap_x) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"(&tmap_w) : "memory");
        }
        uint32_t slot = 0, ph = 1;
        bool ok = true;
        for (; seg.valid() && ok; seg.next()) {
            constexpr int PER = GATHER ? kGatherRows : kBoxRows, L = GATHER ? 2 : 1;  // rows a load; loads a lane and sub-block, at most
            const int loads = (seg.rows + PER - 1) / PER;
            int row[L][4];
            if constexpr (GATHER) {
#pragma unroll
                for (int l = 0; l < L; l++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int m = (lane + 32 * l) * 4 + i;
                        int at = m < seg.rows ? __ldcg(p.order + seg.m0 + m) : -1;
                        if (at >= 0) at = (uint32_t)at / p.top_k;
                        row[l][i] = at >= 0 && at < p.x_rows ? at : p.x_rows;  // (past the end: zeros)
                    }
            }
            for (int st = 0; st < nst; st++) {
                const int nsub = min(kSub, nks - st * kSub);
                ok = __all_sync(0xffffffffu, mbar_wait(&ctl->empty[slot], ph, abort_flag));
                if (!ok) break;
                if (lane == 0) mbar_expect_tx(&ctl->full[slot], (uint32_t)(loads * PER * 128 * nsub));
                __syncwarp();
                if constexpr (GATHER) {
                    for (int u = 0; u < nsub; u++)
#pragma unroll
                        for (int l = 0; l < L; l++)
                            if (lane + 32 * l < loads)
                                tma_gather4(s32(sB) + (slot * kSub + u) * b_bytes + (lane + 32 * l) * 512, &tmap_x, (st * kSub + u) * kBK, row[l], &ctl->full[slot]);
                } else {
                    const int u = lane >> 4, b = lane & 15;
                    if (u < nsub && b < loads)
                        tma_load_2d(sB + (slot * kSub + u) * b_bytes + b * (kBoxRows * 128), &tmap_x, (st * kSub + u) * kBK, seg.m0 + b * kBoxRows, &ctl->full[slot]);
                }
                __syncwarp();
                if (++slot == kStagesB) { slot = 0; ph ^= 1; }
            }
        }
    } else if (warp == kMmaWarp) {
        // ---------------- MMA issuer: the whole warp, one elected lane issues ----------------
        uint32_t tile_i = 0, slot = 0, phase = 0;
        const uint64_t db0 = umma_desc_sw128(s32(sB));
        bool ok = true;
        for (; seg.valid() && ok; seg.next(), tile_i++) {
            const uint32_t idesc = umma_idesc(kTileN, (seg.rows + 15) & ~15);
            if (!mbar_wait_warp(&ctl->tmem_empty, (tile_i & 1) ^ 1, abort_flag)) break;
            tc_fence_after();
            for (int st = 0; st < nst; st++) {
                if (!mbar_wait_warp(&ctl->full[slot], phase, abort_flag)) { ok = false; break; }
                tc_fence_after();
                const uint64_t db = db0 + (uint64_t)(slot * (kSub * b_bytes >> 4));
                const uint32_t a_tmem = tmem_base + kAColBase + slot * kAColsPerSlot;
                if (elect_one()) {
#pragma unroll
                    for (int kk = 0; kk < kBK / 16; kk++) tc_mma_ts(tmem_base, a_tmem + 8 * kk, db + 2 * kk, idesc, (kk > 0 || st != 0) ? 1u : 0u);
                    if (st * kSub + 1 < nks) {  // (the last stage of an odd K has one sub-block)
#pragma unroll
                        for (int kk = 0; kk < kBK / 16; kk++)
                            tc_mma_ts(tmem_base, a_tmem + kAColsPerSub + 8 * kk, db + (b_bytes >> 4) + 2 * kk, idesc, 1u);
                    }
                    tc_commit(&ctl->empty[slot]);
                }
                __syncwarp();
                if (++slot == kStagesB) { slot = 0; phase ^= 1; }
            }
            if (ok && elect_one()) tc_commit(&ctl->tmem_full);
            __syncwarp();
        }
    } else if (warp == kWWarp) {
        // ---------------- packed weights ----------------
        if (lane == 0)
            weight_producer<BITS>(p, seg, nks, sW, ctl->wfull, ctl->wempty, abort_flag,
                                  [&](const GroupSeg& s) { return GATED ? make_int2(s.nt * 8, s.e) : make_int2(s.e * p.N + s.nt * kTileN, 0); },
                                  [&](void* dst, int x, int2 at, uint64_t* bar) {
                                      if constexpr (GATED) tma_load_5d(dst, &tmap_w, x, 0, 0, at.x, at.y, bar);
                                      else tma_load_2d(dst, &tmap_w, x, at.x, bar);
                                  });
    } else if (warp >= kEpiWarps) {
        // ---------------- dequantisers ----------------
        const int q = warp & 3, grp = (warp - kEpiWarps) >> 2;
        dequant_role<BITS>(p, seg, grp, q * 32 + lane, nks, sW + (size_t)grp * p.w_slots * kWUnitBytes, &ctl->wfull[grp * kMaxWSlots],
                           &ctl->wempty[grp * kMaxWSlots], &ctl->empty[grp],
                           tmem_base + ((uint32_t)(q * 32) << 16) + kAColBase + grp * kAColsPerSlot, abort_flag,
                           // (rows past the expert's last: the last one's scales, for lanes whose results are not stored)
                           [&](const GroupSeg& s, int r) {
                               if constexpr (GATED) {
                                   const int f = min(s.nt * 64 + (r >> 4) * 8 + (r & 7), (p.N >> 1) - 1);
                                   return s.e * p.N + (r & 8 ? p.N >> 1 : 0) + f;
                               } else {
                                   return s.e * p.N + min(s.nt * kTileN + r, p.N - 1);
                               }
                           },
                           [&]() { mbar_arrive(&ctl->full[grp]); });
    } else {
        // ---------------- epilogue: warp w reads a quarter of the lanes, half of the columns (rows of x), 16 at a time ----------------
        const int q = warp & 3, half = warp >> 2;
        const uint32_t quarter = tmem_base + ((uint32_t)(q * 32) << 16);
        unsigned char* stg = sEpi + (size_t)warp * kEpiStageBytes;
        uint32_t tile_i = 0;
        for (; seg.valid(); seg.next(), tile_i++) {
            const int blocks = (seg.rows + 15) >> 4, lo = half ? (blocks + 1) >> 1 : 0, hi = half ? blocks : (blocks + 1) >> 1;
            const size_t ld = GATED ? p.N >> 1 : p.N;
            if constexpr (GATED) {
                // this thread: columns f[0], f[1] of y
                const int F = p.N >> 1;
                int f[2];
                float bg[2] = {0.0f, 0.0f}, bu[2] = {0.0f, 0.0f};
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    f[j] = seg.nt * 64 + q * 16 + j * 8 + (lane >> 2);
                    if (p.bias && f[j] < F) {
                        bg[j] = __ldg(p.bias + (size_t)seg.e * p.N + f[j]);
                        bu[j] = __ldg(p.bias + (size_t)seg.e * p.N + F + f[j]);
                    }
                }
                if (!mbar_wait(&ctl->tmem_full, tile_i & 1, abort_flag)) break;
                tc_fence_after();
                for (int blk = lo; blk < hi; blk++) {
                    uint32_t v[2][8];
                    __syncwarp();
                    tmem_ld_16x256b_x2(quarter + blk * 16, v[0]);
                    tmem_ld_16x256b_x2(quarter + (16u << 16) + blk * 16, v[1]);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    float o[2][4];  // rows of x: 2(t%4), the next, and those eight further on
#pragma unroll
                    for (int j = 0; j < 2; j++)
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const int at = (i >> 1) * 4 + (i & 1);
                            o[j][i] = activate(p.act, __uint_as_float(v[j][at]) + bg[j]) * (__uint_as_float(v[j][at + 2]) + bu[j]);
                        }
                    const int m = seg.m0 + blk * 16, rows = seg.rows - blk * 16;
                    if (p.y_vec) {
                        // [16 rows of x][16 columns] through shared memory: a lane stores eight columns of a row
#pragma unroll
                        for (int j = 0; j < 2; j++)
#pragma unroll
                            for (int i = 0; i < 4; i++)
                                *reinterpret_cast<__nv_bfloat16*>(stg + ((i >> 1) * 8 + (lane & 3) * 2 + (i & 1)) * 32 + j * 16 + (lane >> 2) * 2) = __float2bfloat16_rn(o[j][i]);
                        __syncwarp();
                        const int row = lane >> 1, col = seg.nt * 64 + q * 16 + (lane & 1) * 8;
                        if (row < rows && col < F)
                            *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.y) + (size_t)(m + row) * ld + col) = *reinterpret_cast<const uint4*>(stg + row * 32 + (lane & 1) * 16);
                    } else {
#pragma unroll
                        for (int j = 0; j < 2; j++)
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                const int row = (i >> 1) * 8 + (lane & 3) * 2 + (i & 1);
                                if (row >= rows || f[j] >= F) continue;
                                const size_t at = (size_t)(m + row) * ld + f[j];
                                if (p.y_bf16) static_cast<__nv_bfloat16*>(p.y)[at] = __float2bfloat16_rn(o[j][i]);
                                else static_cast<float*>(p.y)[at] = o[j][i];
                            }
                    }
                }
            } else {
                const int n = seg.nt * kTileN + q * 32 + lane;
                const float b = p.bias && n < p.N ? __ldg(p.bias + (size_t)seg.e * p.N + n) : 0.0f;
                if (!mbar_wait(&ctl->tmem_full, tile_i & 1, abort_flag)) break;
                tc_fence_after();
                for (int blk = lo; blk < hi; blk++) {
                    uint32_t v[16];
                    __syncwarp();
                    tmem_ld16(quarter + blk * 16, v);
                    const int m = seg.m0 + blk * 16, rows = seg.rows - blk * 16;
#pragma unroll
                    for (int j = 0; j < 16; j++) v[j] = __float_as_uint(activate(p.act, __uint_as_float(v[j]) + b));
                    if (p.y_vec) {
#pragma unroll
                        for (int j = 0; j < 16; j++) *reinterpret_cast<__nv_bfloat16*>(stg + j * 64 + lane * 2) = __float2bfloat16_rn(__uint_as_float(v[j]));
                        __syncwarp();
                        const int col = seg.nt * kTileN + q * 32 + (lane & 3) * 8;
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            const int row = i * 8 + (lane >> 2);
                            if (row < rows && col < p.N)
                                *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.y) + (size_t)(m + row) * ld + col) = *reinterpret_cast<const uint4*>(stg + row * 64 + (lane & 3) * 16);
                        }
                    } else if (n < p.N) {
#pragma unroll
                        for (int j = 0; j < 16; j++) {
                            if (j >= rows) continue;
                            const size_t at = (size_t)(m + j) * ld + n;
                            if (p.y_bf16) static_cast<__nv_bfloat16*>(p.y)[at] = __float2bfloat16_rn(__uint_as_float(v[j]));
                            else static_cast<float*>(p.y)[at] = __uint_as_float(v[j]);
                        }
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&ctl->tmem_empty);
        }
    }
    // ---------------- teardown ----------------
    tc_fence_before();
    __syncthreads();
    settle_after_abort(abort_flag);
    if (tid == 0 && ctl->abort_flag) *p.error = 1;
    if (warp == kMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tmem_base, kTmemCols);
    }
}

struct Plan {
    int bm, w_slots;
    size_t smem;
};
// bm: an expert of twice the average still takes one tile, as far as there is room; lower tiles leave shared memory to L1, which holds the rows'
// scales.  Weight rings as in qmm_plan.h.
bool make_plan(const ExpertsArgs& a, Plan* pl) {
    const size_t mean = (a.rows + a.experts - 1) / a.experts;
    pl->bm = (int)std::min<size_t>(kMaxBM, std::max<size_t>(32, (2 * mean + 15) / 16 * 16));
    for (;; pl->bm -= 16) {
        const size_t fixed = 1024 + kGemmCtlBytes + (size_t)kStagesB * kSub * pl->bm * 128 + (size_t)kEpiWarps * kEpiStageBytes + (size_t)8 * (a.experts + 1);
        pl->w_slots = (int)std::min<size_t>(a.bits == 8 ? 2 : 1, fixed < (size_t)kGemmSmemLimit ? (kGemmSmemLimit - fixed) / (kDqGroups * kWUnitBytes) : 0);
        pl->smem = fixed + (size_t)kDqGroups * pl->w_slots * kWUnitBytes;
        if (pl->w_slots) return true;
    }
}

template <int BITS, bool GATED, bool GATHER>
cudaError_t launch_t(const CUtensorMap& tmap_x, const CUtensorMap& tmap_w, const ExpertGemm& p, size_t smem, int grid, cudaStream_t stream, bool overlap_prev) {
    auto kern = qmm_experts_kernel<BITS, GATED, GATHER>;
    static std::atomic<bool> attr_set[64];
    if (cudaError_t e = allow_smem(kern, kGemmSmemLimit, attr_set)) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(kNumThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = overlap_prev ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kern, tmap_x, tmap_w, p);
}
template <int BITS>
cudaError_t launch_b(const ExpertsArgs& a, const CUtensorMap& tmap_x, const CUtensorMap& tmap_w, const ExpertGemm& p, size_t smem, int grid, cudaStream_t stream, bool overlap_prev) {
    if (a.gated) return a.order ? launch_t<BITS, true, true>(tmap_x, tmap_w, p, smem, grid, stream, overlap_prev) : launch_t<BITS, true, false>(tmap_x, tmap_w, p, smem, grid, stream, overlap_prev);
    return a.order ? launch_t<BITS, false, true>(tmap_x, tmap_w, p, smem, grid, stream, overlap_prev) : launch_t<BITS, false, false>(tmap_x, tmap_w, p, smem, grid, stream, overlap_prev);
}

}  // namespace

// K in whole sub-blocks; a row of x at least; tiles and groups counted in 32 bits
bool qmm_experts_supported(const ExpertsArgs& a) {
    const long long n_tiles = ((long long)a.N + kTileN - 1) / kTileN;
    return a.K % kBK == 0 && a.x_rows > 0 && (long long)(a.rows / 16 + a.experts) * n_tiles < (1ll << 30) && encode_tiled_fn() != nullptr;
}

cudaError_t launch_qmm_experts(const ExpertsArgs& a, int sm_count, cudaStream_t stream, bool overlap_prev, const char** name) {
    Plan pl;
    if (!make_plan(a, &pl)) return cudaErrorInvalidValue;
    int* err = a.error ? a.error : device_error_word();
    if (!err) return cudaErrorMemoryAllocation;
    const EncodeTiledFn encode = encode_tiled_fn();
    const cuuint32_t estr[5] = {1, 1, 1, 1, 1};
    CUtensorMap tmap_x, tmap_w;
    const cuuint64_t xdims[2] = {(cuuint64_t)a.K, (cuuint64_t)a.x_rows}, xstrides[1] = {(cuuint64_t)a.K * 2};
    const cuuint32_t xbox[2] = {(cuuint32_t)kBK, a.order ? 1u : (cuuint32_t)kBoxRows};
    CUresult r = encode(&tmap_x, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(a.x), xdims, xstrides, xbox, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r == CUDA_SUCCESS) {
        const cuuint64_t row = (cuuint64_t)a.K * a.bits / 8, F = (cuuint64_t)a.N / 2;
        if (a.gated) {
            const cuuint64_t dims[5] = {row, 8, 2, F / 8, (cuuint64_t)a.experts}, strides[4] = {row, F * row, 8 * row, 2 * F * row};
            const cuuint32_t box[5] = {64, 8, 2, kTileN / 16, 1};
            r = encode(&tmap_w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 5, const_cast<uint32_t*>(a.wq), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                       CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        } else {
            const cuuint64_t dims[2] = {row, (cuuint64_t)a.experts * a.N}, strides[1] = {row};
            const cuuint32_t box[2] = {64, kTileN};
            r = encode(&tmap_w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint32_t*>(a.wq), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                       CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        }
    }
    if (r != CUDA_SUCCESS) {
        set_last_error("cuTensorMapEncodeTiled (experts) failed (%d)", (int)r);
        return cudaErrorInvalidValue;
    }
    ExpertGemm p;
    p.scales = (const __nv_bfloat16*)a.scales; p.biases = (const __nv_bfloat16*)a.biases; p.bias = a.bias;
    p.offsets = a.offsets; p.order = a.order; p.y = a.y; p.error = err;
    p.experts = a.experts; p.rows = (int)a.rows; p.x_rows = (int)a.x_rows; p.K = a.K; p.N = a.N;
    p.gshift = a.group == 32 ? 5 : (a.group == 64 ? 6 : 7);
    p.act = a.act; p.y_bf16 = a.y_dtype == LUX_DTYPE_BFLOAT16;
    p.y_vec = p.y_bf16 && ((uintptr_t)a.y & 15) == 0 && (a.gated ? a.N / 2 : a.N) % 8 == 0;
    p.bm = pl.bm; p.w_slots = pl.w_slots; p.n_tiles = (a.N + kTileN - 1) / kTileN; p.top_k = a.order ? a.top_k : 1;
    *name = a.bits == 4 ? "qmm_experts<4>" : "qmm_experts<8>";
    const long long tiles = (long long)(a.rows / pl.bm + a.experts) * p.n_tiles;  // (at most)
    p.most = (int)tiles;
    const int grid = (int)std::min<long long>(sm_count, tiles);
    return a.bits == 4 ? launch_b<4>(a, tmap_x, tmap_w, p, pl.smem, grid, stream, overlap_prev) : launch_b<8>(a, tmap_x, tmap_w, p, pl.smem, grid, stream, overlap_prev);
}

}  // namespace luxcuda
