// Products grouped by expert for many rows an expert (qmatmul_experts), bf16 activations, affine weights:
//   y[i] = epilogue(x[row(i)] . dequant(Wq[e])^T + bias[e]),   offsets[e] <= i < offsets[e+1]
// The roles of qmm_tc.cu's kernels on tiles of 128 rows of an expert's W (on pairs of CTAs: two neighbouring ones) against up to bm of its rows of x;
// bound by dequantisation for few rows (32 an expert: a k-stage of 128 takes 0.34 us at 4 bit, 0.53 at 8, the tensor pipe is active 12 and 10 % of the time), by
// that and by last rounds of tiles that are not full for more (16 experts, 4096 x 2816 gated, 4 bit: 128 rows 41 % of the tensor pipe and 925 TFLOP/s, 256
// rows 51 % and 1121, 512 rows 65 % and 1278; 256 rows at 8 bit 41 % and 865).
//   * The tiles follow from the offsets in device memory: every CTA scans them at its start (an expert's rows are cut into as few tiles as
//     bm allows, all of one height), then takes every gridDim.x-th tile of the whole list; neighbouring CTAs share an expert's weights or
//     rows of x at the same time.
//   * Many rows an expert: pairs of CTAs (cta_group::2), each with half of the rows of x and 128 rows of W of its own; the finished tile goes through
//     shared memory, so that the next one's MMAs run while it is stored.  Fewer: single CTAs with two accumulators.
//   * The matrix instruction's N is the tile's own height, rounded up to 16: a tile of 40 rows takes 48 rows' time.
//   * Rows of x come by TMA, a box of 16 to 64 rows per lane of a warp.  With an order they are copied side by side first, a launch of its own
//     (2048 tokens x 8 experts x 4096: 134 MB, 27 us).  Fetched by index in here they cost more, since every tile of W does it again: TMA gathers of
//     four rows take 29 ns each, 128 of them a stage of 256 rows (1692 us for the 4096 x 2816 product); 16-byte copies by two warps 588, and on pairs of
//     CTAs 690 (their writes have to be waited for and fenced before the MMAs, two stages instead of three are under way).
//   * The sums are the tensor cores' fp32 accumulators, which cut off instead of rounding: fp32 y is off by 1 to 3e-6 (2-norm).  Shorter sums added
//     up outside would cost a second accumulator for every tile, in registers or memory.
//   * Gated: a tile is eight groups of eight rows of gate and the eight of up that go with them, one TMA box of the weights seen as
//     [expert][group of 8][half][8][byte].  Tensor memory is then read in the shape that leaves a row and the row eight further on in one
//     thread: no exchange between the two halves.
#include <algorithm>
#include <atomic>
#include <cstdlib>

#include "epilogue.cuh"
#include "experts_plan.h"
#include "groups.cuh"
#include "qmm_roles.cuh"

namespace luxcuda {

namespace {

// Four groups of dequantising warps and four epilogue warps (qmm_tc.cu: three and eight, as many threads): what bounds tiles that are not high is how
// fast a group gets through a stage (64 experts x 8 rows, 4096 x 2816: without the tensor cores' part 5 % less time, without the arithmetic on codes
// 12 %, with all weights in L2 no less; the rest are the instructions of the hand-overs), and the epilogue has a second accumulator or a copy
// in shared memory to run beside.  Stages as groups: A in tensor memory, 64 columns each, behind the accumulators.
constexpr int kGroups = 4, kStages = kGroups, kEpis = 4;
constexpr int kXWarp = kEpis + 4 * kGroups, kIssueWarp = kXWarp + 1, kFetchWarp = kXWarp + 2, kThreads = (kXWarp + 3) * 32;
static_assert(kStages == kExpertStages && kGroups == kExpertGroups && kEpis == kExpertEpis, "the plan's");
constexpr uint32_t kACol = 256;  // one accumulator of up to 256 columns, or two
static_assert(kACol + kStages * kAColsPerSlot <= kTmemCols, "tensor memory");

struct ExpertGemm {
    const __nv_bfloat16* scales;
    const __nv_bfloat16* biases;
    const float* bias;
    const int* offsets;
    void* y;
    int* error;
    int experts, rows, K, N, gshift, act, y_bf16, y_vec;
    int box;                         // rows of x per TMA box, a divisor of bm
    int bm, n_tiles, w_slots, most;  // rows of x per tile, at most; tiles along N; tiles in all, at most
    int y_staged;  // pairs: the tile goes through shared memory (bf16 y, 16-byte pieces of its rows)
};

struct Control {
    uint64_t full[kStages], empty[kStages], wfull[kGroups * kMaxWSlots], wempty[kGroups * kMaxWSlots], tmem_full[2], tmem_empty[2];
    uint32_t tmem_base;
    int abort_flag;
};
static_assert(sizeof(Control) <= kGemmCtlBytes, "the plan's share of shared memory");

// Tiles of an expert with n rows: how many along its rows, and their height.
__device__ __forceinline__ int row_tiles(int n, int bm) { return (n + bm - 1) / bm; }

// The CTA's tiles (the interface of TileIter), each with its expert and rows.
struct GroupTiles {
    const int *off, *first;  // [experts + 1] in shared memory: first rows, first tiles
    int tile_, step, align, nst, e, nt, m0, rows;
    __device__ __forceinline__ void init(const ExpertGemm& p, const int* tables, int nst_, int start, int step_, int align_) {
        off = tables;
        first = tables + p.experts + 1;
        nst = nst_;
        tile_ = start;
        step = step_;
        align = align_;
        e = 0;
        if (valid(p)) locate(p);
    }
    __device__ __forceinline__ bool valid(const ExpertGemm& p) const { return tile_ < first[p.experts]; }
    __device__ __forceinline__ void locate(const ExpertGemm& p) {
        while (first[e + 1] <= tile_) e++;
        const int n = off[e + 1] - off[e], mt = row_tiles(n, p.bm), at = tile_ - first[e], m = at % mt;
        const int h = ((n + mt - 1) / mt + align - 1) & -align;
        nt = at / mt;
        m0 = off[e] + m * h;
        rows = min(h, n - m * h);
    }
    __device__ __forceinline__ void next(const ExpertGemm& p) {
        tile_ += step;
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
// Lanes 16 .. of a quarter of tensor memory, 16 columns: thread t gets row t/4, columns 2(t%4) and the next in r[0..1], row t/4 + 8 in r[2..3], and
// the same of the eight columns behind in r[4..7].
__device__ __forceinline__ void tmem_ld_16x256b_x2(uint32_t taddr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr));
}

template <int BITS, bool GATED, bool PAIR>
__device__ __forceinline__ void experts_body(const CUtensorMap& tmap_x, const CUtensorMap& tmap_w, const ExpertGemm& p) {
    constexpr int kCtas = PAIR ? 2 : 1, kAlign = 16 * kCtas;
    const int rank = PAIR ? (int)(blockIdx.x & 1) : 0;  // of this CTA in its pair: 0 issues the MMAs of both
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    unsigned char* sB = smem;  // [kStages][kSub][bm rows (pair: half of them)][128 B], swizzled (TMA)
    const uint32_t b_bytes = (uint32_t)(p.bm / kCtas) * 128;
    unsigned char* sW = sB + (size_t)kStages * kSub * b_bytes;  // [kGroups][w_slots][128 rows][64 B], 64-byte swizzle (TMA)
    unsigned char* sEpi = sW + (size_t)kGroups * p.w_slots * kWUnitBytes;  // [kEpis][16 rows of x][32 columns] bf16
    // (pairs: [bm rows of x][kYPitch bytes]: a finished tile on its way out; the pitch keeps the rows on different banks)
    constexpr int kYCols = GATED ? kTileN / 2 : kTileN, kYPitch = y_pitch(GATED);
    Control* ctl = reinterpret_cast<Control*>(sEpi + (PAIR ? (size_t)(p.y_staged ? p.bm * kYPitch : 0) : (size_t)kEpis * kEpiStageBytes));
    int* off = reinterpret_cast<int*>(reinterpret_cast<unsigned char*>(ctl) + kGemmCtlBytes);  // tables of GroupTiles
    int* first = off + p.experts + 1;
    volatile int* abort_flag = &ctl->abort_flag;

    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // (uniform for the compiler too)
    const int nks = p.K / kBK, nst = (nks + kSub - 1) / kSub;

    if (tid == 0) {
        for (int s = 0; s < kStages; s++) {
            // (pairs: used in CTA 0 only) the owning group's four warps in each CTA + CTA 0's producer of x, whose byte count covers both halves
            mbar_init(&ctl->full[s], 4 * kCtas + 1);
            mbar_init(&ctl->empty[s], 1);  // one tcgen05.commit (pairs: multicast to both CTAs)
        }
        for (int g = 0; g < kGroups * kMaxWSlots; g++) {
            mbar_init(&ctl->wfull[g], 1);
            mbar_init(&ctl->wempty[g], 4);
        }
        for (int b = 0; b < 2; b++) {
            mbar_init(&ctl->tmem_full[b], 1);
            mbar_init(&ctl->tmem_empty[b], kEpis * kCtas);
        }
        ctl->abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // (tensor memory behind the wait: a kernel before this one may still want it)
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (warp == kIssueWarp) {
        if constexpr (PAIR) tmem_alloc_pair(&ctl->tmem_base, kTmemCols);
        else tmem_alloc(&ctl->tmem_base, kTmemCols);
    }
    tc_fence_before();
    group_tables(off, first, p.offsets, p.experts, p.rows, p.most, [&](int n) { return row_tiles(n, p.bm) * p.n_tiles; });
    if constexpr (PAIR) cluster_sync();  // the peer's barriers are initialised before anything arrives on them
    tc_fence_after();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t tmem_base = __shfl_sync(0xffffffffu, ctl->tmem_base, 0);
    // accumulator and phase of the CTA's i-th tile
    auto acc_of = [](uint32_t i) { return PAIR ? 0u : i & 1; };
    auto phase_of = [](uint32_t i) { return (PAIR ? i : i >> 1) & 1; };
    GroupSeg seg;
    seg.p = &p;
    seg.init(p, off, nst, blockIdx.x / kCtas, gridDim.x / kCtas, kAlign);
    // tile of 128 rows of W that is this CTA's
    auto n_tile = [&](const GroupSeg& s) { return PAIR ? s.nt * 2 + rank : s.nt; };
    auto arrive_full = [&](int s) {
        if constexpr (PAIR) mbar_arrive_cta0(&ctl->full[s]);
        else mbar_arrive(&ctl->full[s]);
    };

    if (warp == kXWarp) {
        // ---------------- rows of x: the whole warp, a box per lane and stage ----------------
        if (lane == 0) asm volatile("prefetch.tensormap [%0];" ::"l"(&tmap_x) : "memory");
        uint32_t slot = 0, ph = 1;
        bool ok = true;
        for (; seg.valid() && ok; seg.next()) {
            // (pairs: both halves whole, so that either CTA knows the other's bytes)
            const int half = ((seg.rows + 31) & ~31) >> 1, loads = ((PAIR ? half : seg.rows) + p.box - 1) / p.box, from = seg.m0 + (PAIR ? rank * half : 0);
            for (int st = 0; st < nst; st++) {
                const int nsub = min(kSub, nks - st * kSub);
                ok = __all_sync(0xffffffffu, mbar_wait(&ctl->empty[slot], ph, abort_flag));
                if (!ok) break;
                if (lane == 0 && rank == 0) mbar_expect_tx(&ctl->full[slot], (uint32_t)(kCtas * loads * p.box * 128 * nsub));
                __syncwarp();
                const int u = lane >> 4, b = lane & 15;
                if (u < nsub && b < loads) {
                    unsigned char* dst = sB + (slot * kSub + u) * b_bytes + b * (p.box * 128);
                    if constexpr (PAIR) tma_load_2d_pair(dst, &tmap_x, (st * kSub + u) * kBK, from + b * p.box, &ctl->full[slot]);
                    else tma_load_2d(dst, &tmap_x, (st * kSub + u) * kBK, from + b * p.box, &ctl->full[slot]);
                }
                __syncwarp();
                if (++slot == kStages) { slot = 0; ph ^= 1; }
            }
        }
    } else if (warp == kIssueWarp) {
        // ---------------- MMA issuer: the whole warp, one elected lane issues ----------------
        auto mma = [](uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
            if constexpr (PAIR) tc_mma_ts_pair(d, a, b, idesc, acc);
            else tc_mma_ts(d, a, b, idesc, acc);
        };
        auto commit = [](uint64_t* bar) {
            if constexpr (PAIR) tc_commit_pair(bar);
            else tc_commit(bar);
        };
        uint32_t tile_i = 0, slot = 0, phase = 0;
        const uint64_t db0 = umma_desc_sw128(s32(sB));
        bool ok = true;
        for (; rank == 0 && seg.valid() && ok; seg.next(), tile_i++) {
            const uint32_t idesc = umma_idesc(kTileN * kCtas, (seg.rows + kAlign - 1) & -kAlign);
            const uint32_t acc = acc_of(tile_i), d_tmem = tmem_base + acc * kLowRows;
            if (!mbar_wait_warp(&ctl->tmem_empty[acc], phase_of(tile_i) ^ 1, abort_flag)) break;
            tc_fence_after();
            for (int st = 0; st < nst; st++) {
                if (!mbar_wait_warp(&ctl->full[slot], phase, abort_flag)) { ok = false; break; }
                tc_fence_after();
                const uint64_t db = db0 + (uint64_t)(slot * (kSub * b_bytes >> 4));
                const uint32_t a_tmem = tmem_base + kACol + slot * kAColsPerSlot;
                if (elect_one()) {
#pragma unroll
                    for (int kk = 0; kk < kBK / 16; kk++) mma(d_tmem, a_tmem + 8 * kk, db + 2 * kk, idesc, (kk > 0 || st != 0) ? 1u : 0u);
                    if (st * kSub + 1 < nks) {  // (the last stage of an odd K has one sub-block)
#pragma unroll
                        for (int kk = 0; kk < kBK / 16; kk++)
                            mma(d_tmem, a_tmem + kAColsPerSub + 8 * kk, db + (b_bytes >> 4) + 2 * kk, idesc, 1u);
                    }
                    commit(&ctl->empty[slot]);
                }
                __syncwarp();
                if (++slot == kStages) { slot = 0; phase ^= 1; }
            }
            if (ok && elect_one()) commit(&ctl->tmem_full[acc]);
            __syncwarp();
        }
    } else if (warp == kFetchWarp) {
        // ---------------- packed weights ----------------
        if (lane == 0) {
            asm volatile("prefetch.tensormap [%0];" ::"l"(&tmap_w) : "memory");
            weight_producer<BITS, kGroups>(p, seg, nks, sW, ctl->wfull, ctl->wempty, abort_flag,
                                  [&](const GroupSeg& s) { return GATED ? make_int2(n_tile(s) * 8, s.e) : make_int2(s.e * p.N + n_tile(s) * kTileN, 0); },
                                  [&](void* dst, int x, int2 at, uint64_t* bar) {
                                      if constexpr (GATED) tma_load_5d(dst, &tmap_w, x, 0, 0, at.x, at.y, bar);
                                      else tma_load_2d(dst, &tmap_w, x, at.x, bar);
                                  });
        }
    } else if (warp >= kEpis) {
        // ---------------- dequantisers ----------------
        const int q = warp & 3, grp = (warp - kEpis) >> 2;
        dequant_role<BITS, kGroups>(p, seg, grp, q * 32 + lane, nks, sW + (size_t)grp * p.w_slots * kWUnitBytes, &ctl->wfull[grp * kMaxWSlots],
                           &ctl->wempty[grp * kMaxWSlots], &ctl->empty[grp],
                           tmem_base + ((uint32_t)(q * 32) << 16) + kACol + grp * kAColsPerSlot, abort_flag,
                           // (rows past the expert's last: the last one's scales, for lanes whose results are not stored)
                           [&](const GroupSeg& s, int r) {
                               if constexpr (GATED) {
                                   const int f = min(n_tile(s) * 64 + (r >> 4) * 8 + (r & 7), (p.N >> 1) - 1);
                                   return s.e * p.N + (r & 8 ? p.N >> 1 : 0) + f;
                               } else {
                                   return s.e * p.N + min(n_tile(s) * kTileN + r, p.N - 1);
                               }
                           },
                           [&]() { arrive_full(grp); });
    } else {
        // ---------------- epilogue: a warp reads a quarter of the lanes, 16 columns (rows of x) at a time ----------------
        const int q = warp;
        unsigned char* stg = sEpi + (size_t)warp * kEpiStageBytes;
        const bool staged = PAIR && p.y_staged;
        constexpr int kEpiBar = 1;  // named barrier of these warps
        auto wait_tile = [&](uint32_t acc, uint32_t i) {  // (staged: and the previous tile has left)
            return staged ? mbar_wait_epis<kEpiBar, kEpis>(&ctl->tmem_full[acc], phase_of(i), abort_flag) : mbar_wait_epi(&ctl->tmem_full[acc], phase_of(i), abort_flag);
        };
        uint32_t tile_i = 0;
        for (; seg.valid(); seg.next(), tile_i++) {
            const int tile_n = n_tile(seg);
            const int blocks = (seg.rows + 15) >> 4;
            const size_t ld = GATED ? p.N >> 1 : p.N;
            const uint32_t acc = acc_of(tile_i), quarter = tmem_base + ((uint32_t)(q * 32) << 16) + acc * kLowRows;
            if constexpr (GATED) {
                // this thread: columns f[0], f[1] of y
                const int F = p.N >> 1;
                int f[2];
                float bg[2] = {0.0f, 0.0f}, bu[2] = {0.0f, 0.0f};
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    f[j] = tile_n * 64 + q * 16 + j * 8 + (lane >> 2);
                    if (p.bias && f[j] < F) {
                        bg[j] = __ldcg(p.bias + (size_t)seg.e * p.N + f[j]);
                        bu[j] = __ldcg(p.bias + (size_t)seg.e * p.N + F + f[j]);
                    }
                }
                if (!wait_tile(acc, tile_i)) break;
                tc_fence_after();
                for (int blk = 0; blk < blocks; blk++) {
                    uint32_t v[2][8];
                    __syncwarp();
                    tmem_ld_16x256b_x2(quarter + blk * 16, v[0]);
                    tmem_ld_16x256b_x2(quarter + (16u << 16) + blk * 16, v[1]);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    float o[8];  // two columns of y times rows of x: 2(t%4), the next, and those eight further on
#pragma unroll
                    for (int k = 0; k < 8; k++) o[k] = __uint_as_float(v[k >> 2][(k >> 1 & 1) * 4 + (k & 1)]) + bg[k >> 2];
                    activate(p.act, o);
#pragma unroll
                    for (int k = 0; k < 8; k++) o[k] *= __uint_as_float(v[k >> 2][(k >> 1 & 1) * 4 + (k & 1) + 2]) + bu[k >> 2];
                    const int m = seg.m0 + blk * 16, rows = seg.rows - blk * 16;
                    if (staged) {
#pragma unroll
                        for (int j = 0; j < 2; j++)
#pragma unroll
                            for (int i = 0; i < 4; i++)
                                *reinterpret_cast<__nv_bfloat16*>(sEpi + (blk * 16 + (i >> 1) * 8 + (lane & 3) * 2 + (i & 1)) * kYPitch + (q * 16 + j * 8 + (lane >> 2)) * 2) = __float2bfloat16_rn(o[4 * j + i]);
                    } else if (!PAIR && p.y_vec) {
                        // [16 rows of x][16 columns] through shared memory: a lane stores eight columns of a row
#pragma unroll
                        for (int j = 0; j < 2; j++)
#pragma unroll
                            for (int i = 0; i < 4; i++)
                                *reinterpret_cast<__nv_bfloat16*>(stg + ((i >> 1) * 8 + (lane & 3) * 2 + (i & 1)) * 32 + j * 16 + (lane >> 2) * 2) = __float2bfloat16_rn(o[4 * j + i]);
                        __syncwarp();
                        const int row = lane >> 1, col = tile_n * 64 + q * 16 + (lane & 1) * 8;
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
                                if (p.y_bf16) static_cast<__nv_bfloat16*>(p.y)[at] = __float2bfloat16_rn(o[4 * j + i]);
                                else static_cast<float*>(p.y)[at] = o[4 * j + i];
                            }
                    }
                }
            } else {
                const int n = tile_n * kTileN + q * 32 + lane;
                const float b = p.bias && n < p.N ? __ldcg(p.bias + (size_t)seg.e * p.N + n) : 0.0f;
                if (!wait_tile(acc, tile_i)) break;
                tc_fence_after();
                for (int blk = 0; blk < blocks; blk++) {
                    uint32_t v[16];
                    __syncwarp();
                    tmem_ld16(quarter + blk * 16, v);
                    const int m = seg.m0 + blk * 16, rows = seg.rows - blk * 16;
                    float o[16];
#pragma unroll
                    for (int j = 0; j < 16; j++) o[j] = __uint_as_float(v[j]) + b;
                    activate(p.act, o);
                    if (staged) {
#pragma unroll
                        for (int j = 0; j < 16; j++) *reinterpret_cast<__nv_bfloat16*>(sEpi + (blk * 16 + j) * kYPitch + (q * 32 + lane) * 2) = __float2bfloat16_rn(o[j]);
                    } else if (!PAIR && p.y_vec) {
#pragma unroll
                        for (int j = 0; j < 16; j++) *reinterpret_cast<__nv_bfloat16*>(stg + j * 64 + lane * 2) = __float2bfloat16_rn(o[j]);
                        __syncwarp();
                        const int col = tile_n * kTileN + q * 32 + (lane & 3) * 8;
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
                            if (p.y_bf16) static_cast<__nv_bfloat16*>(p.y)[at] = __float2bfloat16_rn(o[j]);
                            else static_cast<float*>(p.y)[at] = o[j];
                        }
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if constexpr (PAIR) mbar_arrive_cta0(&ctl->tmem_empty[acc]);
                else mbar_arrive(&ctl->tmem_empty[acc]);
            }
            if (staged) {  // the accumulator is free: the tile leaves, 16 bytes a store, while the next one's MMAs run
                asm volatile("bar.sync %0, %1;" ::"n"(kEpiBar), "n"(kEpis * 32) : "memory");
                constexpr int kPieces = kYCols / 8;
                const int piece = tid % kPieces, col = tile_n * kYCols + piece * 8;
                if (col < (int)ld)
                    for (int row = tid / kPieces; row < seg.rows; row += kEpis * 32 / kPieces)
                        *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.y) + (size_t)(seg.m0 + row) * ld + col) = *reinterpret_cast<const uint4*>(sEpi + row * kYPitch + piece * 16);
            }
        }
    }
    // ---------------- teardown ----------------
    tc_fence_before();
    __syncthreads();
    settle_after_abort(abort_flag);
    if constexpr (PAIR) cluster_sync();  // neither CTA leaves (or frees tensor memory) while the other may still reach into it
    if (tid == 0 && ctl->abort_flag) *p.error = 1;
    if (warp == kIssueWarp) {
        tc_fence_after();
        if constexpr (PAIR) tmem_dealloc_pair(tmem_base, kTmemCols);
        else tmem_dealloc(tmem_base, kTmemCols);
    }
}

template <int BITS, bool GATED>
__global__ void __launch_bounds__(kThreads, 1)
qmm_experts_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ ExpertGemm p) {
    experts_body<BITS, GATED, false>(tmap_x, tmap_w, p);
}
template <int BITS, bool GATED>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
qmm_experts_pair_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ ExpertGemm p) {
    experts_body<BITS, GATED, true>(tmap_x, tmap_w, p);
}

bool y_in_pieces(const ExpertsArgs& a) { return a.y_dtype == LUX_DTYPE_BFLOAT16 && ((uintptr_t)a.y & 15) == 0 && (a.gated ? a.N / 2 : a.N) % 8 == 0; }
template <int BITS, bool GATED, bool PAIR>
cudaError_t launch_t(const CUtensorMap& tmap_x, const CUtensorMap& tmap_w, const ExpertGemm& p, size_t smem, int grid, cudaStream_t stream, bool overlap_prev) {
    auto kern = PAIR ? qmm_experts_pair_kernel<BITS, GATED> : qmm_experts_kernel<BITS, GATED>;
    static std::atomic<bool> attr_set[64];
    if (cudaError_t e = allow_smem(kern, kGemmSmemLimit, attr_set)) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = overlap_prev ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kern, tmap_x, tmap_w, p);
}
template <int BITS, bool PAIR>
cudaError_t launch_b(const ExpertsArgs& a, const CUtensorMap& tmap_x, const CUtensorMap& tmap_w, const ExpertGemm& p, size_t smem, int grid, cudaStream_t stream, bool overlap_prev) {
    return a.gated ? launch_t<BITS, true, PAIR>(tmap_x, tmap_w, p, smem, grid, stream, overlap_prev) : launch_t<BITS, false, PAIR>(tmap_x, tmap_w, p, smem, grid, stream, overlap_prev);
}

// Rows of x side by side: row i of out is row order[i] / top_k of x, zeros where there is none (which behind the last pair is anything).  A warp takes
// a row at a time, 64 bytes a lane under way.  (Loads past L1, here and of what the GEMM reads besides weights: the kernel before may have written it while
// this one was already on the SM.)
__global__ void __launch_bounds__(256) gather_rows_kernel(const uint4* x, uint4* out, const int* order, int rows, int x_rows, int pieces, uint32_t top_k) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int lane = threadIdx.x & 31;
    for (long long i = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); i < rows; i += (long long)gridDim.x * 8) {
        int from = __ldcg(order + i);
        if (from >= 0) from = (uint32_t)from / top_k;
        const bool there = from >= 0 && from < x_rows;
        const uint4* src = x + (size_t)(there ? from : 0) * pieces;
        uint4* dst = out + (size_t)i * pieces;
        for (int c = lane; c < pieces; c += 128) {
            uint4 v[4];
#pragma unroll
            for (int u = 0; u < 4; u++) v[u] = there && c + 32 * u < pieces ? __ldcg(src + c + 32 * u) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int u = 0; u < 4; u++)
                if (c + 32 * u < pieces) dst[c + 32 * u] = v[u];
        }
    }
}

}  // namespace

// K in whole sub-blocks; a row of x at least; tiles and groups counted in 32 bits
size_t qmm_experts_workspace_bytes(const ExpertsArgs& a) { return a.order ? a.rows * a.K * 2 : 0; }
bool qmm_experts_supported(const ExpertsArgs& a) {
    const long long n_tiles = ((long long)a.N + kTileN - 1) / kTileN;
    return a.K % kBK == 0 && a.x_rows > 0 && (long long)(a.rows / 16 + a.experts) * n_tiles < (1ll << 30) && encode_tiled_fn() != nullptr;
}

cudaError_t launch_qmm_experts(const ExpertsArgs& a, void* workspace, int sm_count, cudaStream_t stream, bool overlap_prev, const char** name) {
    const char* force = getenv("LUXCUDA_EXPERTS_PAIR");  // "0" | "1" (experiments)
    const ExpertsPlan pl = plan_experts({a.rows, a.experts, a.K, a.N, a.bits, a.order != nullptr}, a.gated, y_in_pieces(a), sm_count, force ? force[0] == '1' : -1);
    int* err = a.error ? a.error : device_error_word();
    if (!err) return cudaErrorMemoryAllocation;
    const EncodeTiledFn encode = encode_tiled_fn();
    const cuuint32_t estr[5] = {1, 1, 1, 1, 1};
    CUtensorMap tmap_x, tmap_w;
    if (a.order) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)std::min<size_t>((size_t)sm_count * 8, (a.rows + 7) / 8));
        cfg.blockDim = dim3(256);
        cfg.stream = stream;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = overlap_prev ? 1 : 0;
        if (cudaError_t e = cudaLaunchKernelEx(&cfg, gather_rows_kernel, (const uint4*)a.x, (uint4*)workspace, a.order, (int)a.rows, (int)a.x_rows,
                                               a.K / 8, (uint32_t)a.top_k))
            return e;
        overlap_prev = true;  // (behind that launch in any case)
    }
    const void* x = a.order ? workspace : a.x;
    const cuuint64_t xdims[2] = {(cuuint64_t)a.K, (cuuint64_t)(a.order ? a.rows : a.x_rows)}, xstrides[1] = {(cuuint64_t)a.K * 2};
    const cuuint32_t xbox[2] = {(cuuint32_t)kBK, (cuuint32_t)pl.box};
    CUresult r = encode(&tmap_x, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(x), xdims, xstrides, xbox, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
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
    p.offsets = a.offsets; p.y = a.y; p.error = err;
    p.experts = a.experts; p.rows = (int)a.rows; p.K = a.K; p.N = a.N;
    p.gshift = a.group == 32 ? 5 : (a.group == 64 ? 6 : 7);
    p.act = a.act; p.y_bf16 = a.y_dtype == LUX_DTYPE_BFLOAT16;
    p.y_vec = y_in_pieces(a); p.y_staged = pl.y_staged;
    p.box = pl.box; p.bm = pl.bm; p.w_slots = pl.w_slots; p.n_tiles = pl.n_tiles;
    *name = a.bits == 4 ? (pl.pair ? "qmm_experts<4,pairs>" : "qmm_experts<4>") : (pl.pair ? "qmm_experts<8,pairs>" : "qmm_experts<8>");
    const long long tiles = (long long)(a.rows / pl.bm + a.experts) * p.n_tiles;  // (at most)
    p.most = (int)tiles;
    const int grid = pl.pair ? 2 * (int)std::min<long long>(sm_count / 2, tiles) : (int)std::min<long long>(sm_count, tiles);
    auto launch = a.bits == 4 ? (pl.pair ? launch_b<4, true> : launch_b<4, false>) : (pl.pair ? launch_b<8, true> : launch_b<8, false>);
    return launch(a, tmap_x, tmap_w, p, pl.smem, grid, stream, overlap_prev);
}

}  // namespace luxcuda
