// Prefill-regime quantized GEMM for bf16 activations (M > 16):
//   y[M,N] = x[M,K] . dequant(Wq[N,K])^T,  w^ = RNE_bf16(s*q + b)  (one bf16 FMA)
// on the 5th-generation tensor cores: tcgen05.mma with the fp32 accumulator in
// tensor memory, operands in shared memory.
//
// Tensor-bound: 2*M*N*K flop per launch; the packed weights (N*K*bits/8 bytes)
// are re-read M/BM times from L2, x (M*K*2 bytes) N/128 times.
//
// The MMA computes the TRANSPOSED tile  D[n, m] = sum_k W^[n, k] * x[m, k]:
//   A operand = 128 rows of W^ (dequantised bf16), written by the dequantising
//               warps straight into TENSOR MEMORY (tcgen05.st): it never
//               touches shared memory, whose bandwidth the B operand needs;
//   B operand = BM <= 256 rows of x (K-major, 128-byte swizzle) in shared
//               memory, brought in by TMA (cp.async.bulk.tensor, no multicast);
//   D         = 128 lanes x BM columns of fp32 in TMEM.
// With W on the 128-lane side a weight is dequantised once per BM = 256 rows of
// x, which keeps the integer pipe (the scarce one) at about a quarter load.
// TMEM (512 columns): D in columns [0, 256), a ring of A k-stages
// (64 weights = 32 columns each) from column 256 on, one slot per k-stage in
// flight.  Shared memory: the matching ring of B stages (32 KiB each).
//
// One persistent CTA per SM, 23 warps:
//   warps 0-7   epilogue: warp w reads TMEM lanes 32*(w%4).., half w/4 of the
//               columns, rounds to bf16/fp32, stores y[m][n];
//   warps 8-19  dequantisers in three groups of four warps (dequant_role): group j owns the
//               pipeline stages = j (mod 3); inside a group warp q owns TMEM lanes 32q..,
//               so thread (q, lane) owns row n0 + 32q + lane.  A unit of 128 rows x 64 packed
//               bytes comes through shared memory (64-byte swizzle, so the row-per-thread
//               reads are bank-conflict free; row-per-thread loads from global memory were one
//               L1 wavefront per lane).  Scales / biases of a stage are one small vector load
//               per thread, fetched one owned stage ahead.  32 TMEM columns per 64 weights;
//   warp 20     TMA producer for x;
//   warp 21     allocates TMEM, issues tcgen05.mma (one elected lane) and the
//               commits that release A slots / B stages and publish D;
//   warp 22     TMA producer for the packed weights (weight_producer).
// Hand-over uses mbarriers; every wait is bounded: on a time-out the kernel
// raises an error word (host-visible) and all roles drain and return.
#include <algorithm>
#include <atomic>

#include "epilogue.cuh"
#include "qmm_roles.cuh"

namespace luxcuda {

namespace {

constexpr uint32_t kSpinLimit = 1u << 22;  // polls of a flag in global memory, 100 ns and more apart
constexpr size_t kWsFlagBytes = 1024;  // flag words of the stream-K workspace (one per CTA), ahead of the partials

struct GemmParams {
    const uint32_t* wq;
    const __nv_bfloat16* scales;
    const __nv_bfloat16* biases;
    void* y;
    int* error;              // host-visible error word (0 = ok)
    int M, K, N, gshift, y_bf16;
    int world, ld, col0;     // copies of y to write (1 unless column-sharded), their row stride and this rank's first column
    void* y_all[kMaxShardWorld];
    int bm;                  // rows of x per tile (multiple of 16, <= 256)
    int w_slots;             // weight units in flight per dequantising group
    int n_tiles, m_tiles;
    float* ws;               // partial accumulators of tiles shared between CTAs: [CTA][bm][128] fp32
    int y_tma;               // pair kernel: y leaves through shared memory; 1: by a TMA store (bf16, one copy of y, N % 8 == 0),
                             // 2: by 16-byte stores into every rank's copy (column-sharded, ld and col0 multiples of 8)
    uint32_t* ws_flags;      // [CTA]: 1 while that CTA's partial waits to be added (zero between launches)
    const float* bias;       // epilogue (EPI): null where there is none
    const void* residual;    // as y: [M][N]
    int act, r_bf16;
};

// ---- the epilogue of qmatmul_epi: act(sum + bias) + residual ----
// The residual is the tile's size again in bytes, read by the warps that nothing overlaps: into L2 while the tile's MMAs run, then sixteen rows ahead
// of the accumulator.  (Neither, 32 rows at a time: 2048 x 4096 x 4096 onto an fp32 stream 117 us, without the stream 61.)
//
// All epilogue threads, ahead of their wait for the accumulator: the rows [m0, m0 + rows) of the tile's columns from n0 on into L2, a row per copy.
__device__ __forceinline__ void prefetch_residual(const GemmParams& p, int m0, int rows, int n0, int thread) {
    const size_t es = p.r_bf16 ? 2 : 4;
    if (!p.residual || n0 >= p.N || ((uintptr_t)p.residual | p.N * es) & 15) return;
    const uint32_t bytes = (uint32_t)(min(kTileN, p.N - n0) * es);  // (a multiple of 16, as the rows are)
    for (int row = thread; row < rows; row += kEpiWarps * 32)
        asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(static_cast<const char*>(p.residual) + ((size_t)(m0 + row) * p.N + n0) * es), "r"(bytes) : "memory");
}
__device__ __forceinline__ uint32_t ldg_u16_plain(const uint16_t* p) {  // (not .nc: y may be the residual)
    uint32_t v;
    asm volatile("ld.global.u16 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}
// Column n of the residual, rows m .. m + 15 (of which `rows` are there), as it lies: converted here, each load would be waited for ahead of the next
__device__ __forceinline__ void load_residual(const GemmParams& p, int m, int rows, int n, uint32_t (&r)[16]) {
    if (!p.residual || n >= p.N) return;
    const size_t at = (size_t)m * p.N + n;
    if (p.r_bf16) {
        const uint16_t* q = static_cast<const uint16_t*>(p.residual) + at;
#pragma unroll
        for (int j = 0; j < 16; j++, q += p.N) r[j] = j < rows ? ldg_u16_plain(q) : 0u;
    } else {
        const uint32_t* q = static_cast<const uint32_t*>(p.residual) + at;
#pragma unroll
        for (int j = 0; j < 16; j++, q += p.N) r[j] = j < rows ? *q : 0u;
    }
}
__device__ __forceinline__ void finish(const GemmParams& p, uint32_t* raw, const uint32_t (&r)[16], float bias) {
    float v[16];
#pragma unroll
    for (int j = 0; j < 16; j++) v[j] = __uint_as_float(raw[j]) + bias;
    activate(p.act, v);
    if (p.residual) {
#pragma unroll
        for (int j = 0; j < 16; j++) v[j] += __uint_as_float(r[j] << (p.r_bf16 ? 16 : 0));
    }
#pragma unroll
    for (int j = 0; j < 16; j++) raw[j] = __float_as_uint(v[j]);
}
// A warp's share of a tile, rows [c_lo, c_hi) of x (whole sixteens; m_end of the tile's rows are there) of its lanes' columns n: put(sums, row of the tile)
// takes sixteen at a time.
template <class Put>
__device__ __forceinline__ void finish_rows(const GemmParams& p, uint32_t lanes, int c_lo, int c_hi, int m0, int m_end, int n, const Put& put) {
    const float bias = p.bias && n < p.N ? __ldg(p.bias + n) : 0.0f;
    uint32_t r[16], next[16];
    load_residual(p, m0 + c_lo, m_end - c_lo, n, next);
    for (int c0 = c_lo; c0 < min(c_hi, m_end); c0 += 16) {
#pragma unroll
        for (int j = 0; j < 16; j++) r[j] = next[j];
        if (c0 + 16 < c_hi) load_residual(p, m0 + c0 + 16, m_end - c0 - 16, n, next);
        uint32_t v[16];
        __syncwarp();
        tmem_ld16(lanes + c0, v);
        finish(p, v, r, bias);
        put(v, c0);
    }
}
// sixteen rows straight to y (one copy of it)
__device__ __forceinline__ void put_direct(const GemmParams& p, const uint32_t* v, int m, int rows, int n) {
    if (n >= p.N) return;
    const size_t at = (size_t)m * p.N + n;
    if (p.y_bf16) {
        __nv_bfloat16* q = static_cast<__nv_bfloat16*>(p.y) + at;
#pragma unroll
        for (int j = 0; j < 16; j++, q += p.N)
            if (j < rows) *q = __float2bfloat16_rn(__uint_as_float(v[j]));
    } else {
        float* q = static_cast<float*>(p.y) + at;
#pragma unroll
        for (int j = 0; j < 16; j++, q += p.N)
            if (j < rows) *q = __uint_as_float(v[j]);
    }
}

// The work of a launch is the sequence of (tile, k-stage) units, tile after tile.  Two schedules:
//   * whole tiles, round robin: CTA c takes tiles c, c + G, c + 2G, ... (neighbouring CTAs work on neighbouring
//     tiles at the same k, which L2 likes); the launch lasts ceil(T/G) tiles;
//   * "stream-K": CTA c takes the units [U*c/G, U*(c+1)/G), so every SM gets the same number of k-stages
//     whatever the number of tiles, at the price of one more epilogue per CTA and of the exchange of partial
//     accumulators described next.  The host picks the cheaper one by a small cost model (make_gemm_plan).
// A CTA's range is a sequence of segments, each a run of stages [s_lo, s_hi) of one tile.  Only its first
// segment can start inside a tile (s_lo > 0): that partial accumulator goes to the CTA's slot of the
// workspace; the CTA that owns the tile's first stages (s_lo == 0) adds the partials of the CTAs after it
// (c+1 .. the owner of the tile's last stage) in its epilogue and writes y.  Those partials are produced
// either at the start of the neighbour's range or, when a range is shorter than a tile, at the same time
// as the head: the head's wait for them is short, and bounded.
struct SegIter {  // stream-K: the CTA's range of units, segment by segment
    long long u, u_hi;
    int nst;
    __device__ __forceinline__ void init(long long total_units, int nst_) {
        nst = nst_;
        u = total_units * blockIdx.x / gridDim.x;
        u_hi = total_units * (blockIdx.x + 1) / gridDim.x;
    }
    __device__ __forceinline__ bool valid() const { return u < u_hi; }
    __device__ __forceinline__ int tile() const { return (int)(u / nst); }
    __device__ __forceinline__ int s_lo() const { return (int)(u % nst); }
    __device__ __forceinline__ int s_hi() const { return (int)min((long long)nst, (long long)s_lo() + (u_hi - u)); }
    __device__ __forceinline__ void next() { u += (long long)(s_hi() - s_lo()); }
};
// the CTA whose range holds unit u
__device__ __forceinline__ int cta_of_unit(long long u, long long total_units) {
    return (int)(((u + 1) * gridDim.x - 1) / total_units);
}

struct SmemLayout {
    uint64_t full[kStagesB], empty[kStagesB], wfull[kDqGroups * kMaxWSlots], wempty[kDqGroups * kMaxWSlots], tmem_full, tmem_empty;
    uint32_t tmem_base;
    int abort_flag;
};

template <int BITS, bool EPI>
__global__ void __launch_bounds__(kNumThreads, 1)
qmm_tc_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w,
              const __grid_constant__ GemmParams p) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    unsigned char* sB = smem;  // [kStagesB][bm rows][128 B], swizzled (TMA)
    const uint32_t b_bytes = (uint32_t)p.bm * 128;
    unsigned char* sW = sB + (size_t)kStagesB * kSub * b_bytes;  // [kDqGroups][w_slots][128 rows][64 B], 64-byte swizzle (TMA)
    unsigned char* sEpi = sW + (size_t)kDqGroups * p.w_slots * kWUnitBytes;  // [kEpiWarps][16 rows of x][32 rows of the tile] bf16: the epilogue's transposer
    SmemLayout* sl = reinterpret_cast<SmemLayout*>(sEpi + (size_t)kEpiWarps * kEpiStageBytes);
    volatile int* abort_flag = &sl->abort_flag;

    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // (uniform for the compiler too)
    const int nks = p.K / kBK;                  // 64-weight sub-blocks along K
    const int nst = (nks + kSub - 1) / kSub;    // pipeline stages per tile
    const int total_tiles = p.n_tiles * p.m_tiles;
    const long long total_units = (long long)total_tiles * nst;

    if (tid == 0) {
        for (int s = 0; s < kStagesB; s++) {
            mbar_init(&sl->full[s], 4 + 1);  // the owning group's four warps + the TMA producer (with its byte count)
            mbar_init(&sl->empty[s], 1);        // one tcgen05.commit
        }
        for (int g = 0; g < kDqGroups * kMaxWSlots; g++) {
            mbar_init(&sl->wfull[g], 1);   // the weight producer's expect_tx
            mbar_init(&sl->wempty[g], 4);  // the group's four warps have read their rows
        }
        mbar_init(&sl->tmem_full, 1);
        mbar_init(&sl->tmem_empty, kEpiWarps * 32);
        sl->abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMmaWarp) tmem_alloc(&sl->tmem_base, kTmemCols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = __shfl_sync(0xffffffffu, sl->tmem_base, 0);

    if (warp == kTmaWarp) {
        // ---------------- TMA producer: x tiles ----------------
        if (lane == 0) {
            asm volatile("prefetch.tensormap [%0];" ::"l"(&tmap_x) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"(&tmap_w) : "memory");
            uint32_t it = 0;
            bool ok = true;
            SegIter seg;
            for (seg.init(total_units, nst); seg.valid() && ok; seg.next()) {
                const int tile = seg.tile(), s_hi = seg.s_hi();
                const int m0 = (tile % p.m_tiles) * p.bm;
                for (int st = seg.s_lo(); st < s_hi; st++, it++) {
                    const int sb = it % kStagesB;
                    const uint32_t ph = (it / kStagesB) & 1;
                    const int nsub = min(kSub, nks - st * kSub);
                    if (!mbar_wait(&sl->empty[sb], ph ^ 1, abort_flag)) { ok = false; break; }
                    mbar_expect_tx(&sl->full[sb], b_bytes * nsub);
                    for (int u = 0; u < nsub; u++)
                        tma_load_2d(sB + (sb * kSub + u) * b_bytes, &tmap_x, (st * kSub + u) * kBK, m0, &sl->full[sb]);
                }
            }
        }
    } else if (warp == kMmaWarp) {
        // ---------------- MMA issuer ----------------
        // The whole warp walks the stages and one elected lane issues: addresses and descriptors then live in uniform
        // registers, where the MMAs take them from.  (Walked by one lane, each MMA cost about 106 cycles of moves into
        // them, 850 of the 1210 cycles that a stage took whatever the tile's height; the MMAs of a 256-row tile need 1024.)
        {
            const uint32_t idesc = umma_idesc(kTileN, p.bm);
            uint32_t tile_i = 0, slot = 0, phase = 0;
            const uint64_t db0 = umma_desc_sw128(s32(sB));
            bool ok = true;
            SegIter seg;
            for (seg.init(total_units, nst); seg.valid() && ok; seg.next(), tile_i++) {
                const int s_lo = seg.s_lo(), s_hi = seg.s_hi();
                if (!mbar_wait_warp(&sl->tmem_empty, (tile_i & 1) ^ 1, abort_flag)) break;
                tc_fence_after();
                for (int st = s_lo; st < s_hi; st++) {
                    if (!mbar_wait_warp(&sl->full[slot], phase, abort_flag)) { ok = false; break; }
                    tc_fence_after();
                    const uint64_t db = db0 + (uint64_t)(slot * (kSub * b_bytes >> 4));
                    const uint32_t a_tmem = tmem_base + kAColBase + slot * kAColsPerSlot;
                    if (elect_one()) {
                        // 16 k per MMA = 8 TMEM columns of A, 32 bytes of each B row
#pragma unroll
                        for (int kk = 0; kk < kBK / 16; kk++) tc_mma_ts(tmem_base, a_tmem + 8 * kk, db + 2 * kk, idesc, (kk > 0 || st != s_lo) ? 1u : 0u);
                        if (st * kSub + 1 < nks) {  // (the last stage of an odd K has one sub-block)
#pragma unroll
                            for (int kk = 0; kk < kBK / 16; kk++)
                                tc_mma_ts(tmem_base, a_tmem + kAColsPerSub + 8 * kk, db + (b_bytes >> 4) + 2 * kk, idesc, 1u);
                        }
                        tc_commit(&sl->empty[slot]);  // arrives when the MMAs above have consumed their operands
                    }
                    __syncwarp();
                    if (++slot == kStagesB) { slot = 0; phase ^= 1; }
                }
                if (ok && elect_one()) tc_commit(&sl->tmem_full);
                __syncwarp();
            }
        }
    } else if (warp == kWWarp) {
        // ---------------- TMA producer: packed weights ----------------
        SegIter seg;
        seg.init(total_units, nst);
        if (lane == 0) weight_producer<BITS>(p, seg, nks, sW, sl->wfull, sl->wempty, abort_flag, [&](const auto& s) { return make_int2((s.tile() / p.m_tiles) * kTileN, 0); },
                                              [&](void* dst, int x, int2 at, uint64_t* bar) { tma_load_2d(dst, &tmap_w, x, at.x, bar); });
    } else if (warp >= kEpiWarps) {
        // ---------------- dequantisers ----------------
        const int q = warp & 3, grp = (warp - kEpiWarps) >> 2;
        SegIter seg;
        seg.init(total_units, nst);
        dequant_role<BITS>(p, seg, grp, q * 32 + lane, nks, sW + (size_t)grp * p.w_slots * kWUnitBytes, &sl->wfull[grp * kMaxWSlots],
                           &sl->wempty[grp * kMaxWSlots], &sl->empty[grp],
                           tmem_base + ((uint32_t)(q * 32) << 16) + kAColBase + grp * kAColsPerSlot, abort_flag,
                           [&](const auto& s, int r) { return min((s.tile() / p.m_tiles) * kTileN + r, p.N - 1); }, [&]() { mbar_arrive(&sl->full[grp]); });
    } else {
        // ---------------- epilogue: warp w reads TMEM lanes 32*(w%4).., half w/4 of the column blocks ----------------
        const int q = warp & 3, half = warp >> 2;
        const int nblk = (p.bm + 31) / 32, blk_lo = half ? (nblk + 1) / 2 : 0, blk_hi = half ? nblk : (nblk + 1) / 2;
        const int et = tid;                       // 0 .. 255: the epilogue threads are the first eight warps
        const int nl = q * 32 + lane;             // this thread's row of the tile (TMEM lane)
        constexpr int kEpiBar = 1 + kDqGroups;    // named barrier of the epilogue warps
        uint32_t tile_i = 0;
        bool ok = true;
        SegIter seg;
        for (seg.init(total_units, nst); seg.valid() && ok; seg.next(), tile_i++) {
            const int tile = seg.tile(), s_lo = seg.s_lo(), s_hi = seg.s_hi();
            const int n = (tile / p.m_tiles) * kTileN + nl;
            const int m0 = (tile % p.m_tiles) * p.bm;
            if (EPI && s_lo == 0) prefetch_residual(p, m0, min(p.bm, p.M - m0), n - nl, et);
            // (split tiles: these warps meet at a barrier below)
            if (!(s_lo != 0 || s_hi != nst ? mbar_wait_epis<kEpiBar, kEpiWarps>(&sl->tmem_full, tile_i & 1, abort_flag)
                                           : mbar_wait_epi(&sl->tmem_full, tile_i & 1, abort_flag)))
                break;
            tc_fence_after();
            const int m_end = min(p.bm, p.M - m0);
            if (s_lo != 0) {
                // The segment starts inside a tile: its accumulator is a partial sum, for the CTA that owns the
                // tile's first stages.  [row of x][row of the tile] fp32 in this CTA's slot, then the flag.
                float* ws = p.ws + (size_t)blockIdx.x * (kTileN * kMaxBM);
                for (int blk = blk_lo; blk < blk_hi; blk++) {
                    const int c0 = blk * 32;
                    uint32_t v[32];
                    __syncwarp();
                    tmem_ld32(tmem_base + ((uint32_t)(q * 32) << 16) + c0, v);
                    // (rows past the tile's last row of x are stored too: the slot has room for them and nobody adds them)
#pragma unroll
                    for (int j = 0; j < 32; j++) __stcg(ws + (size_t)(c0 + j) * kTileN + nl, __uint_as_float(v[j]));
                }
                // The stores of all epilogue threads are ordered before the barrier, the barrier before the release
                // of the flag: whoever acquires the flag sees them.  (No fence per thread: it would wait for the
                // stores, with the accumulator still held.)
                asm volatile("bar.sync %0, %1;" ::"n"(kEpiBar), "n"(kEpiWarps * 32) : "memory");
                if (et == 0) asm volatile("st.release.gpu.global.u32 [%0], %1;" ::"l"(p.ws_flags + blockIdx.x), "r"(1u) : "memory");
            } else {
                // The segment starts the tile.  If it does not also end it, the CTAs after this one hold the rest:
                // wait (bounded) for their partials, add them in CTA order, then write y.
                const int c_last = s_hi == nst ? (int)blockIdx.x : cta_of_unit((long long)(tile + 1) * nst - 1, total_units);
                const int parts = c_last - (int)blockIdx.x;
                if (parts > 0) {
                    bool got = true;
                    if (et < parts) {
                        const uint32_t* f = p.ws_flags + blockIdx.x + 1 + et;
                        uint32_t v = 0;
                        for (uint32_t i = 0; i < kSpinLimit; i++) {
                            asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(f) : "memory");
                            if (v || ((i & 1023u) == 1023u && *abort_flag)) break;
                            __nanosleep(100);
                        }
                        got = v != 0;
                    }
                    uint32_t all;
                    asm volatile(
                        "{ .reg .pred p, q; setp.ne.u32 q, %1, 0; bar.red.and.pred p, %2, %3, q; selp.u32 %0, 1, 0, p; }"
                        : "=r"(all) : "r"((uint32_t)got), "n"(kEpiBar), "n"(kEpiWarps * 32) : "memory");
                    if (!all) {
                        *abort_flag = 1;
                        ok = false;
                        break;
                    }
                }
                // y[m][n] for this thread's n and `cnt` consecutive rows m0 + c0 + j
                // bf16: the thread holds one column of y (its n) for consecutive rows, but y is contiguous along n.
                // Sixteen rows at a time go through the warp's 1 KB of shared memory, [row][n], and leave as
                // 16-byte stores, eight rows of 64 bytes per instruction, instead of 2-byte stores of one row.
                const bool y_vec = p.y_bf16 && ((p.ld | p.col0) & 7) == 0;
                unsigned char* stg = sEpi + (size_t)warp * kEpiStageBytes;
                const int ncol0 = (tile / p.m_tiles) * kTileN + q * 32 + (lane & 3) * 8;  // first of this thread's 8 columns on the way out
                auto store_rows = [&](const uint32_t* v, int c0, int cnt) {
                    if (y_vec) {  // (callers on this path pass sixteen rows)
                        __syncwarp();  // the previous sixteen rows have been read
#pragma unroll
                        for (int j = 0; j < 16; j += 2) {
                            const __nv_bfloat162 pr = __floats2bfloat162_rn(__uint_as_float(v[j]), __uint_as_float(v[j + 1]));
                            *reinterpret_cast<__nv_bfloat16*>(stg + j * 64 + lane * 2) = pr.x;
                            *reinterpret_cast<__nv_bfloat16*>(stg + (j + 1) * 64 + lane * 2) = pr.y;
                        }
                        __syncwarp();
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            const int row = i * 8 + (lane >> 2), m = c0 + row;
                            const uint4 val = *reinterpret_cast<const uint4*>(stg + row * 64 + (lane & 3) * 16);
                            if (m >= m_end || ncol0 >= p.N) continue;
                            const size_t idx = (size_t)(m0 + m) * p.ld + p.col0 + ncol0;
                            if (ncol0 + 8 <= p.N) {
                                for (int dst = 0; dst < p.world; dst++)
                                    *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(p.y_all[dst]) + idx) = val;
                            } else {  // the last columns of y: one by one
                                const uint32_t w4[4] = {val.x, val.y, val.z, val.w};
                                for (int dst = 0; dst < p.world; dst++) {
                                    uint16_t* yp = reinterpret_cast<uint16_t*>(p.y_all[dst]) + idx;
#pragma unroll
                                    for (int e = 0; e < 8; e++)
                                        if (ncol0 + e < p.N) yp[e] = (uint16_t)(w4[e >> 1] >> ((e & 1) * 16));
                                }
                            }
                        }
                        return;
                    }
                    if (n >= p.N) return;
                    // column-sharded layers: the tile goes into every rank's copy of y (peer stores over NVLink)
                    const size_t idx0 = (size_t)(m0 + c0) * p.ld + p.col0 + n;
                    for (int dst = 0; dst < p.world; dst++) {
                        if (p.y_bf16) {
                            __nv_bfloat16* yp = reinterpret_cast<__nv_bfloat16*>(p.y_all[dst]) + idx0;
#pragma unroll
                            for (int j = 0; j < 32; j++)
                                if (j < cnt && c0 + j < m_end) yp[(size_t)j * p.ld] = __float2bfloat16_rn(__uint_as_float(v[j]));
                        } else {
                            float* yp = reinterpret_cast<float*>(p.y_all[dst]) + idx0;
#pragma unroll
                            for (int j = 0; j < 32; j++)
                                if (j < cnt && c0 + j < m_end) yp[(size_t)j * p.ld] = __uint_as_float(v[j]);
                        }
                    }
                };
                if (EPI && parts == 0) {
                    finish_rows(p, tmem_base + ((uint32_t)(q * 32) << 16), blk_lo * 32, blk_hi * 32, m0, m_end, n, [&](uint32_t* v, int c0) {
                        if (y_vec) store_rows(v, c0, 16);
                        else put_direct(p, v, m0 + c0, m_end - c0, n);
                    });
                } else if (parts == 0 && y_vec) {
                    // (requesting the next sixteen columns before the current ones are stored was tried: 3 % slower)
                    for (int c0 = blk_lo * 32; c0 < blk_hi * 32; c0 += 16) {
                        uint32_t v[16];
                        __syncwarp();
                        tmem_ld16(tmem_base + ((uint32_t)(q * 32) << 16) + c0, v);
                        store_rows(v, c0, 16);
                    }
                } else if (parts == 0) {
                    for (int blk = blk_lo; blk < blk_hi; blk++) {
                        uint32_t v[32];
                        __syncwarp();
                        tmem_ld32(tmem_base + ((uint32_t)(q * 32) << 16) + blk * 32, v);
                        store_rows(v, blk * 32, 32);
                    }
                } else {
                    // 16 rows of x at a time (accumulator + one partial in registers); the partial is requested
                    // before the accumulator is read
                    for (int c0 = blk_lo * 32; c0 < blk_hi * 32; c0 += 16) {
                        uint32_t v[32];
                        float pv[16];
                        const float* ws = p.ws + (size_t)(blockIdx.x + 1) * (kTileN * kMaxBM) + (size_t)c0 * kTileN + nl;
#pragma unroll
                        for (int j = 0; j < 16; j++) pv[j] = __ldcg(ws + (size_t)j * kTileN);
                        __syncwarp();
                        tmem_ld16(tmem_base + ((uint32_t)(q * 32) << 16) + c0, reinterpret_cast<uint32_t(&)[16]>(v));
                        for (int pt = 1; pt <= parts; pt++) {
#pragma unroll
                            for (int j = 0; j < 16; j++) v[j] = __float_as_uint(__uint_as_float(v[j]) + pv[j]);
                            if (pt < parts) {
                                ws += (size_t)kTileN * kMaxBM;
#pragma unroll
                                for (int j = 0; j < 16; j++) pv[j] = __ldcg(ws + (size_t)j * kTileN);
                            }
                        }
                        if constexpr (EPI) {
                            uint32_t r[16];
                            load_residual(p, m0 + c0, m_end - c0, n, r);
                            finish(p, v, r, p.bias && n < p.N ? __ldg(p.bias + n) : 0.0f);
                        }
                        store_rows(v, c0, 16);
                    }
                }
                if (parts > 0) {
                    // every epilogue thread has read the partials: their flags go back to zero for the next launch
                    asm volatile("bar.sync %0, %1;" ::"n"(kEpiBar), "n"(kEpiWarps * 32) : "memory");
                    if (et < parts) p.ws_flags[blockIdx.x + 1 + et] = 0;
                }
            }
            tc_fence_before();
            mbar_arrive(&sl->tmem_empty);
        }
    }
    // ---------------- teardown ----------------
    tc_fence_before();
    __syncthreads();
    settle_after_abort(abort_flag);
    if (tid == 0 && sl->abort_flag) *p.error = 1;
    if (warp == kMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tmem_base, kTmemCols);
    }
}

// Whole tiles, round robin, as a kernel of its own: the same roles without the bookkeeping of split tiles.  (One
// body for both schedules ran this one 5 % slower, and so did every addition tried here -- 16-byte stores through
// shared memory in the epilogue, the look-ahead of the MMA issuer: the launch is sensitive to the amount of code
// its roles execute side by side.)
template <int BITS, bool EPI>
__global__ void __launch_bounds__(kNumThreads, 1)
qmm_tc_tiles_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w,
              const __grid_constant__ GemmParams p) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    unsigned char* sB = smem;  // [kStagesB][bm rows][128 B], swizzled (TMA)
    const uint32_t b_bytes = (uint32_t)p.bm * 128;
    unsigned char* sW = sB + (size_t)kStagesB * kSub * b_bytes;  // [kDqGroups][w_slots][128 rows][64 B], 64-byte swizzle (TMA)
    SmemLayout* sl = reinterpret_cast<SmemLayout*>(sW + (size_t)kDqGroups * p.w_slots * kWUnitBytes);
    volatile int* abort_flag = &sl->abort_flag;

    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // (uniform for the compiler too)
    const int nks = p.K / kBK;                  // 64-weight sub-blocks along K
    const int nst = (nks + kSub - 1) / kSub;    // pipeline stages per tile
    const int total_tiles = p.n_tiles * p.m_tiles;

    if (tid == 0) {
        for (int s = 0; s < kStagesB; s++) {
            mbar_init(&sl->full[s], 4 + 1);  // the owning group's four warps + the TMA producer (with its byte count)
            mbar_init(&sl->empty[s], 1);        // one tcgen05.commit
        }
        for (int g = 0; g < kDqGroups * kMaxWSlots; g++) {
            mbar_init(&sl->wfull[g], 1);   // the weight producer's expect_tx
            mbar_init(&sl->wempty[g], 4);  // the group's four warps have read their rows
        }
        mbar_init(&sl->tmem_full, 1);
        mbar_init(&sl->tmem_empty, kEpiWarps * 32);
        sl->abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMmaWarp) tmem_alloc(&sl->tmem_base, kTmemCols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = __shfl_sync(0xffffffffu, sl->tmem_base, 0);

    if (warp == kTmaWarp) {
        // ---------------- TMA producer: x tiles ----------------
        if (lane == 0) {
            asm volatile("prefetch.tensormap [%0];" ::"l"(&tmap_x) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"(&tmap_w) : "memory");
            uint32_t it = 0;
            bool ok = true;
            for (int tile = blockIdx.x; tile < total_tiles && ok; tile += gridDim.x) {
                const int m0 = (tile % p.m_tiles) * p.bm;
                for (int st = 0; st < nst; st++, it++) {
                    const int sb = it % kStagesB;
                    const uint32_t ph = (it / kStagesB) & 1;
                    const int nsub = min(kSub, nks - st * kSub);
                    if (!mbar_wait(&sl->empty[sb], ph ^ 1, abort_flag)) { ok = false; break; }
                    mbar_expect_tx(&sl->full[sb], b_bytes * nsub);
                    for (int u = 0; u < nsub; u++)
                        tma_load_2d(sB + (sb * kSub + u) * b_bytes, &tmap_x, (st * kSub + u) * kBK, m0, &sl->full[sb]);
                }
            }
        }
    } else if (warp == kMmaWarp) {
        // ---------------- MMA issuer (as above: the whole warp, one elected lane) ----------------
        {
            const uint32_t idesc = umma_idesc(kTileN, p.bm);
            uint32_t tile_i = 0, slot = 0, phase = 0;
            const uint64_t db0 = umma_desc_sw128(s32(sB));
            bool ok = true;
            for (int tile = blockIdx.x; tile < total_tiles && ok; tile += gridDim.x, tile_i++) {
                if (!mbar_wait_warp(&sl->tmem_empty, (tile_i & 1) ^ 1, abort_flag)) break;
                tc_fence_after();
                for (int st = 0; st < nst; st++) {
                    if (!mbar_wait_warp(&sl->full[slot], phase, abort_flag)) { ok = false; break; }
                    tc_fence_after();
                    const uint64_t db = db0 + (uint64_t)(slot * (kSub * b_bytes >> 4));
                    const uint32_t a_tmem = tmem_base + kAColBase + slot * kAColsPerSlot;
                    if (elect_one()) {
                        // 16 k per MMA = 8 TMEM columns of A, 32 bytes of each B row
#pragma unroll
                        for (int kk = 0; kk < kBK / 16; kk++) tc_mma_ts(tmem_base, a_tmem + 8 * kk, db + 2 * kk, idesc, (kk > 0 || st != 0) ? 1u : 0u);
                        if (st * kSub + 1 < nks) {  // (the last stage of an odd K has one sub-block)
#pragma unroll
                            for (int kk = 0; kk < kBK / 16; kk++)
                                tc_mma_ts(tmem_base, a_tmem + kAColsPerSub + 8 * kk, db + (b_bytes >> 4) + 2 * kk, idesc, 1u);
                        }
                        tc_commit(&sl->empty[slot]);  // arrives when the MMAs above have consumed their operands
                    }
                    __syncwarp();
                    if (++slot == kStagesB) { slot = 0; phase ^= 1; }
                }
                if (ok && elect_one()) tc_commit(&sl->tmem_full);
                __syncwarp();
            }
        }
    } else if (warp == kWWarp) {
        // ---------------- TMA producer: packed weights ----------------
        const TileIter seg{(int)blockIdx.x, (int)gridDim.x, total_tiles, nst};
        if (lane == 0) weight_producer<BITS>(p, seg, nks, sW, sl->wfull, sl->wempty, abort_flag, [&](const auto& s) { return make_int2((s.tile() / p.m_tiles) * kTileN, 0); },
                                              [&](void* dst, int x, int2 at, uint64_t* bar) { tma_load_2d(dst, &tmap_w, x, at.x, bar); });
    } else if (warp >= kEpiWarps) {
        // ---------------- dequantisers ----------------
        const int q = warp & 3, grp = (warp - kEpiWarps) >> 2;
        const TileIter seg{(int)blockIdx.x, (int)gridDim.x, total_tiles, nst};
        dequant_role<BITS>(p, seg, grp, q * 32 + lane, nks, sW + (size_t)grp * p.w_slots * kWUnitBytes, &sl->wfull[grp * kMaxWSlots],
                           &sl->wempty[grp * kMaxWSlots], &sl->empty[grp],
                           tmem_base + ((uint32_t)(q * 32) << 16) + kAColBase + grp * kAColsPerSlot, abort_flag,
                           [&](const auto& s, int r) { return min((s.tile() / p.m_tiles) * kTileN + r, p.N - 1); }, [&]() { mbar_arrive(&sl->full[grp]); });
    } else {
        // ---------------- epilogue: warp w reads TMEM lanes 32*(w%4).., half w/4 of the column blocks ----------------
        const int q = warp & 3, half = warp >> 2;
        const int nblk = (p.bm + 31) / 32, blk_lo = half ? (nblk + 1) / 2 : 0, blk_hi = half ? nblk : (nblk + 1) / 2;
        uint32_t tile_i = 0;
        for (int tile = blockIdx.x; tile < total_tiles; tile += gridDim.x, tile_i++) {
            const int n = (tile / p.m_tiles) * kTileN + q * 32 + lane;
            const int m0 = (tile % p.m_tiles) * p.bm;
            if (EPI) prefetch_residual(p, m0, min(p.bm, p.M - m0), (tile / p.m_tiles) * kTileN, tid);
            if (!mbar_wait_epi(&sl->tmem_full, tile_i & 1, abort_flag)) break;
            tc_fence_after();
            // this thread: column n of y, rows m0 + c (32 consecutive n per warp: 64-byte row segments)
            const int m_end = min(p.bm, p.M - m0);
            if (EPI)
                finish_rows(p, tmem_base + ((uint32_t)(q * 32) << 16), blk_lo * 32, blk_hi * 32, m0, m_end, n, [&](uint32_t* v, int c0) { put_direct(p, v, m0 + c0, m_end - c0, n); });
            for (int blk = blk_lo; !EPI && blk < blk_hi; blk++) {
                const int c0 = blk * 32;
                uint32_t v[32];
                __syncwarp();
                tmem_ld32(tmem_base + ((uint32_t)(q * 32) << 16) + c0, v);
                if (n < p.N) {
                    // column-sharded layers: the tile goes into every rank's copy of y (peer stores over NVLink)
                    const size_t idx0 = (size_t)(m0 + c0) * p.ld + p.col0 + n;
                    for (int dst = 0; dst < p.world; dst++) {
                        if (p.y_bf16) {
                            __nv_bfloat16* yp = reinterpret_cast<__nv_bfloat16*>(p.y_all[dst]) + idx0;
                            if (c0 + 32 <= m_end) {
#pragma unroll
                                for (int j = 0; j < 32; j++) yp[(size_t)j * p.ld] = __float2bfloat16_rn(__uint_as_float(v[j]));
                            } else {
#pragma unroll
                                for (int j = 0; j < 32; j++)
                                    if (c0 + j < m_end) yp[(size_t)j * p.ld] = __float2bfloat16_rn(__uint_as_float(v[j]));
                            }
                        } else {
                            float* yp = reinterpret_cast<float*>(p.y_all[dst]) + idx0;
#pragma unroll
                            for (int j = 0; j < 32; j++)
                                if (c0 + j < m_end) yp[(size_t)j * p.ld] = __uint_as_float(v[j]);
                        }
                    }
                }
            }
            tc_fence_before();
            mbar_arrive(&sl->tmem_empty);
        }
    }
    // ---------------- teardown ----------------
    tc_fence_before();
    __syncthreads();
    settle_after_abort(abort_flag);
    if (tid == 0 && sl->abort_flag) *p.error = 1;
    if (warp == kMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tmem_base, kTmemCols);
    }
}

// ---- CTA pairs (cta_group::2): two CTAs of a cluster share one MMA stream ------------------------------------
// The MMA is 256 rows of W (128 from each CTA's tensor memory) x bm rows of x, of which each CTA stages half in
// its shared memory; the thread that issues it (in CTA 0) issues for both tensor cores, so the instruction
// stream that bounds a stage is halved per SM, and x takes half the shared memory per stage.
constexpr int kPairEpiBar = 1 + kDqGroups;       // named barrier of the epilogue warps
static_assert(kDqGroups == kStagesP, "a group always owns the same slot");
static_assert(kAColBase + kStagesP * kAColsPerSlot <= kTmemCols, "A ring does not fit");
struct PairSmemLayout {
    uint64_t full[kStagesP], empty[kStagesP], wfull[kDqGroups * kMaxWSlots], wempty[kDqGroups * kMaxWSlots], tmem_full, tmem_empty;
    uint32_t tmem_base;
    int abort_flag;
};
static_assert(sizeof(SmemLayout) <= kGemmCtlBytes && sizeof(PairSmemLayout) <= kGemmCtlBytes, "the plan's share of shared memory");
// a finished tile of y from shared memory ([row of x][128 columns] bf16) to global memory; rows and columns past
// the ends of y are clipped by the copy engine
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, const void* src, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];"
                 ::"l"(map), "r"(x), "r"(y), "r"(s32(src)) : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
template <int BITS, bool EPI>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kNumThreads, 1)
qmm_tc_pair_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w,
                   const __grid_constant__ CUtensorMap tmap_y, const __grid_constant__ GemmParams p) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    unsigned char* sB = smem;  // [kStagesP][kSub][bm/2 rows][128 B], swizzled (TMA): this CTA's half of the x tile
    const uint32_t b_bytes = (uint32_t)(p.bm >> 1) * 128;
    unsigned char* sW = sB + (size_t)kStagesP * kSub * b_bytes;  // [kDqGroups][w_slots][128 rows][64 B], 64-byte swizzle (TMA)
    unsigned char* sY = sW + (size_t)kDqGroups * p.w_slots * kWUnitBytes;  // [bm rows of x][128 columns] bf16: a finished tile on its way out
    // (without the staging buffer the shared memory is that much smaller, and L1, which holds the rows' scales and
    // biases over a tile, that much larger: worth 4 % on this kernel)
    PairSmemLayout* sl = reinterpret_cast<PairSmemLayout*>(sY + (p.y_tma ? pair_y_bytes(p.bm) : 0));
    uint32_t rank;  // of this CTA in its pair: 0 issues the MMAs of both
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    const int cl = (int)(blockIdx.x >> 1), ncl = (int)(gridDim.x >> 1);
    volatile int* abort_flag = &sl->abort_flag;

    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // (uniform for the compiler too)
    const int nks = p.K / kBK;                  // 64-weight sub-blocks along K
    const int nst = (nks + kSub - 1) / kSub;    // pipeline stages per tile
    // A pair takes two neighbouring 128-row tiles of W (CTA `rank` the tile 2*np + rank) against the same rows of x;
    // with an odd number of W tiles the last pair's second CTA works on rows past N (zeros in, nothing out).
    const int total_tiles = ((p.n_tiles + 1) >> 1) * p.m_tiles;  // pair tiles
    auto n0_of = [&](int pt) { return ((pt / p.m_tiles) * 2 + (int)rank) * kTileN; };

    if (tid == 0) {
        for (int s = 0; s < kStagesP; s++) {
            // (used in CTA 0 only) the four warps of the owning group in either CTA + CTA 0's TMA producer, whose
            // byte count covers both CTAs' halves of x
            mbar_init(&sl->full[s], 4 + 4 + 1);
            mbar_init(&sl->empty[s], 1);  // one tcgen05.commit, multicast to both CTAs
        }
        for (int g = 0; g < kDqGroups * kMaxWSlots; g++) {
            mbar_init(&sl->wfull[g], 1);   // the weight producer's expect_tx
            mbar_init(&sl->wempty[g], 4);  // the group's four warps have read their rows
        }
        mbar_init(&sl->tmem_full, 1);
        mbar_init(&sl->tmem_empty, 2 * kEpiWarps);  // (used in CTA 0 only) the epilogue warps of both CTAs
        sl->abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMmaWarp) tmem_alloc_pair(&sl->tmem_base, kTmemCols);  // the same warp of both CTAs
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // the peer's barriers are initialised before anything arrives on them
    tc_fence_after();
    const uint32_t tmem_base = __shfl_sync(0xffffffffu, sl->tmem_base, 0);

    if (warp == kTmaWarp) {
        // ---------------- TMA producer: x tiles ----------------
        if (lane == 0) {
            asm volatile("prefetch.tensormap [%0];" ::"l"(&tmap_x) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"(&tmap_w) : "memory");
            uint32_t it = 0;
            bool ok = true;
            for (int tile = cl; tile < total_tiles && ok; tile += ncl) {
                const int m0 = (tile % p.m_tiles) * p.bm + (int)rank * (p.bm >> 1);  // this CTA's half of the rows of x
                for (int st = 0; st < nst; st++, it++) {
                    const int sb = it % kStagesP;
                    const uint32_t ph = (it / kStagesP) & 1;
                    const int nsub = min(kSub, nks - st * kSub);
                    if (!mbar_wait(&sl->empty[sb], ph ^ 1, abort_flag)) { ok = false; break; }
                    // both halves complete on CTA 0's barrier, which expects the bytes of both
                    if (rank == 0) mbar_expect_tx(&sl->full[sb], 2 * b_bytes * nsub);
                    for (int u = 0; u < nsub; u++)
                        tma_load_2d_pair(sB + (sb * kSub + u) * b_bytes, &tmap_x, (st * kSub + u) * kBK, m0, &sl->full[sb]);
                }
            }
        }
    } else if (warp == kMmaWarp) {
        // ---------------- MMA issuer (as above: the whole warp, one elected lane) ----------------
        if (rank == 0) {
            const uint32_t idesc = umma_idesc(2 * kTileN, p.bm);  // 256 rows of W over the two CTAs x bm rows of x
            uint32_t tile_i = 0, slot = 0, phase = 0;
            const uint64_t db0 = umma_desc_sw128(s32(sB));
            bool ok = true;
            for (int tile = cl; tile < total_tiles && ok; tile += ncl, tile_i++) {
                if (!mbar_wait_warp(&sl->tmem_empty, (tile_i & 1) ^ 1, abort_flag)) break;
                tc_fence_after();
                for (int st = 0; st < nst; st++) {
                    if (!mbar_wait_warp(&sl->full[slot], phase, abort_flag)) { ok = false; break; }
                    tc_fence_after();
                    const uint64_t db = db0 + (uint64_t)(slot * (kSub * b_bytes >> 4));
                    const uint32_t a_tmem = tmem_base + kAColBase + slot * kAColsPerSlot;
                    if (elect_one()) {
                        // 16 k per MMA = 8 TMEM columns of A, 32 bytes of each B row
#pragma unroll
                        for (int kk = 0; kk < kBK / 16; kk++) tc_mma_ts_pair(tmem_base, a_tmem + 8 * kk, db + 2 * kk, idesc, (kk > 0 || st != 0) ? 1u : 0u);
                        if (st * kSub + 1 < nks) {  // (the last stage of an odd K has one sub-block)
#pragma unroll
                            for (int kk = 0; kk < kBK / 16; kk++)
                                tc_mma_ts_pair(tmem_base, a_tmem + kAColsPerSub + 8 * kk, db + (b_bytes >> 4) + 2 * kk, idesc, 1u);
                        }
                        tc_commit_pair(&sl->empty[slot]);  // arrives, in both CTAs, when the MMAs above have consumed their operands
                    }
                    __syncwarp();
                    if (++slot == kStagesP) { slot = 0; phase ^= 1; }
                }
                if (ok && elect_one()) tc_commit_pair(&sl->tmem_full);
                __syncwarp();
            }
        }
    } else if (warp == kWWarp) {
        // ---------------- TMA producer: packed weights ----------------
        const TileIter seg{cl, ncl, total_tiles, nst};
        if (lane == 0) weight_producer<BITS>(p, seg, nks, sW, sl->wfull, sl->wempty, abort_flag, [&](const auto& s) { return make_int2(n0_of(s.tile()), 0); },
                                              [&](void* dst, int x, int2 at, uint64_t* bar) { tma_load_2d(dst, &tmap_w, x, at.x, bar); });
    } else if (warp >= kEpiWarps) {
        // ---------------- dequantisers ----------------
        const int q = warp & 3, grp = (warp - kEpiWarps) >> 2;
        const TileIter seg{cl, ncl, total_tiles, nst};
        dequant_role<BITS>(p, seg, grp, q * 32 + lane, nks, sW + (size_t)grp * p.w_slots * kWUnitBytes, &sl->wfull[grp * kMaxWSlots],
                           &sl->wempty[grp * kMaxWSlots], &sl->empty[grp],
                           tmem_base + ((uint32_t)(q * 32) << 16) + kAColBase + grp * kAColsPerSlot, abort_flag,
                           [&](const auto& s, int r) { return min(n0_of(s.tile()) + r, p.N - 1); }, [&]() { mbar_arrive_cta0(&sl->full[grp]); });
    } else {
        // ---------------- epilogue: warp w reads TMEM lanes 32*(w%4).., half w/4 of the column blocks ----------------
        const int q = warp & 3, half = warp >> 2;
        const int nblk = (p.bm + 31) / 32, blk_lo = half ? (nblk + 1) / 2 : 0, blk_hi = half ? nblk : (nblk + 1) / 2;
        uint32_t tile_i = 0;
        for (int tile = cl; tile < total_tiles; tile += ncl, tile_i++) {
            const int n = n0_of(tile) + q * 32 + lane;
            const int m0 = (tile % p.m_tiles) * p.bm;
            if (EPI) prefetch_residual(p, m0, min(p.bm, p.M - m0), n0_of(tile), tid);
            if (p.y_tma) {
                // the copy engine has finished reading the previous tile out of the staging buffer
                if (tid == 0 && tile_i > 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                if (!mbar_wait_epis<kPairEpiBar, kEpiWarps>(&sl->tmem_full, tile_i & 1, abort_flag)) break;
            } else if (!mbar_wait_epi(&sl->tmem_full, tile_i & 1, abort_flag)) {
                break;
            }
            tc_fence_after();
            if (p.y_tma) {
                // The accumulator goes to shared memory as bf16, [row of x][column], and is released at once; the
                // copy engine takes the tile to y while the next tile's MMAs run.
                if (EPI)
                    finish_rows(p, tmem_base + ((uint32_t)(q * 32) << 16), blk_lo * 32, blk_hi * 32, m0, min(p.bm, p.M - m0), n, [&](uint32_t* v, int c0) {
                        __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(sY + (size_t)c0 * 256) + q * 32 + lane;
#pragma unroll
                        for (int j = 0; j < 16; j++) dst[j * 128] = __float2bfloat16_rn(__uint_as_float(v[j]));
                    });
                for (int blk = blk_lo; !EPI && blk < blk_hi; blk++) {
                    const int c0 = blk * 32;
                    uint32_t v[32];
                    __syncwarp();
                    tmem_ld32(tmem_base + ((uint32_t)(q * 32) << 16) + c0, v);
                    __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(sY + (size_t)c0 * 256) + q * 32 + lane;
#pragma unroll
                    for (int j = 0; j < 32; j++) dst[j * 128] = __float2bfloat16_rn(__uint_as_float(v[j]));
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cta0(&sl->tmem_empty);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // these writes, then the copy engine's reads
                asm volatile("bar.sync %0, %1;" ::"n"(kPairEpiBar), "n"(kEpiWarps * 32) : "memory");
                if (p.y_tma == 1) {
                    if (tid == 0 && n0_of(tile) < p.N) tma_store_2d(&tmap_y, sY, n0_of(tile), m0);
                } else {
                    // column-sharded layers: the tile goes into every rank's copy of y, 16 bytes per store (plain
                    // stores: no TMA on a peer's memory), a row of the tile = 16 lanes
                    const int m_end = min(p.bm, p.M - m0);
                    const int ncol = n0_of(tile) + (tid & 15) * 8;
                    for (int row = tid >> 4; row < m_end; row += (kEpiWarps * 32) >> 4) {
                        const uint4 val = *reinterpret_cast<const uint4*>(sY + (size_t)row * 256 + (tid & 15) * 16);
                        if (ncol >= p.N) continue;
                        const size_t idx = (size_t)(m0 + row) * p.ld + p.col0 + ncol;
                        if (ncol + 8 <= p.N) {
                            for (int dst = 0; dst < p.world; dst++)
                                *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(p.y_all[dst]) + idx) = val;
                        } else {  // the last columns of y: one by one
                            const uint32_t w4[4] = {val.x, val.y, val.z, val.w};
                            for (int dst = 0; dst < p.world; dst++) {
                                uint16_t* yp = reinterpret_cast<uint16_t*>(p.y_all[dst]) + idx;
#pragma unroll
                                for (int e = 0; e < 8; e++)
                                    if (ncol + e < p.N) yp[e] = (uint16_t)(w4[e >> 1] >> ((e & 1) * 16));
                            }
                        }
                    }
                }
                continue;
            }
            // this thread: column n of y, rows m0 + c (32 consecutive n per warp: 64-byte row segments)
            const int m_end = min(p.bm, p.M - m0);
            if (EPI)
                finish_rows(p, tmem_base + ((uint32_t)(q * 32) << 16), blk_lo * 32, blk_hi * 32, m0, m_end, n, [&](uint32_t* v, int c0) { put_direct(p, v, m0 + c0, m_end - c0, n); });
            for (int blk = blk_lo; !EPI && blk < blk_hi; blk++) {
                const int c0 = blk * 32;
                uint32_t v[32];
                __syncwarp();
                tmem_ld32(tmem_base + ((uint32_t)(q * 32) << 16) + c0, v);
                if (n < p.N) {
                    // column-sharded layers: the tile goes into every rank's copy of y (peer stores over NVLink)
                    const size_t idx0 = (size_t)(m0 + c0) * p.ld + p.col0 + n;
                    for (int dst = 0; dst < p.world; dst++) {
                        if (p.y_bf16) {
                            __nv_bfloat16* yp = reinterpret_cast<__nv_bfloat16*>(p.y_all[dst]) + idx0;
                            if (c0 + 32 <= m_end) {
#pragma unroll
                                for (int j = 0; j < 32; j++) yp[(size_t)j * p.ld] = __float2bfloat16_rn(__uint_as_float(v[j]));
                            } else {
#pragma unroll
                                for (int j = 0; j < 32; j++)
                                    if (c0 + j < m_end) yp[(size_t)j * p.ld] = __float2bfloat16_rn(__uint_as_float(v[j]));
                            }
                        } else {
                            float* yp = reinterpret_cast<float*>(p.y_all[dst]) + idx0;
#pragma unroll
                            for (int j = 0; j < 32; j++)
                                if (c0 + j < m_end) yp[(size_t)j * p.ld] = __uint_as_float(v[j]);
                        }
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cta0(&sl->tmem_empty);
        }
    }
    // ---------------- teardown ----------------
    if (tid == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");  // the last tile has left
    tc_fence_before();
    __syncthreads();
    settle_after_abort(abort_flag);
    cluster_sync();  // neither CTA leaves (or frees tensor memory) while the other may still reach into it
    if (tid == 0 && sl->abort_flag) *p.error = 1;
    if (warp == kMmaWarp) {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, kTmemCols);
    }
}

// ---- host side -------------------------------------------------------------------
}  // namespace

EncodeTiledFn encode_tiled_fn() {
    static EncodeTiledFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeTiledFn>(p);
    }();
    return fn;
}

namespace {

int* g_error_host = nullptr;  // pinned + mapped: written by kernels that give up on a wait, read by the host
std::once_flag g_error_once;

int* error_word() {
    std::call_once(g_error_once, [] {
        void* p = nullptr;
        if (cudaHostAlloc(&p, sizeof(int), cudaHostAllocMapped | cudaHostAllocPortable) == cudaSuccess) {
            g_error_host = static_cast<int*>(p);
            *g_error_host = 0;
        } else {
            cudaGetLastError();
        }
    });
    return g_error_host;
}

bool make_gemm_plan(const QmmArgs& a, int sm_count, const ShardPush* push, GemmPlan* pl) {
    if (push && push->world <= 1) push = nullptr;
    if (a.x_dtype != LUX_DTYPE_BFLOAT16 || a.sb_dtype != LUX_DTYPE_BFLOAT16) return false;
    if (a.bits != 4 && a.bits != 8) return false;
    if (a.group != 32 && a.group != 64 && a.group != 128) return false;
    if (a.M <= 16 || a.N < 1 || a.K % kBK) return false;
    if (((uintptr_t)a.x | (uintptr_t)a.wq | (uintptr_t)a.scales | (uintptr_t)a.biases | (uintptr_t)a.y) & 15) return false;
    if ((long long)a.N * (a.K / a.group) > (1ll << 31) - 1) return false;
    // LUXCUDA_QMM_SCHEDULE = "streamk" | "tiles", LUXCUDA_QMM_PAIR = "0" | "1" (experiments)
    const char *schedule = getenv("LUXCUDA_QMM_SCHEDULE"), *pair = getenv("LUXCUDA_QMM_PAIR");
    GemmForce force;
    if (schedule) force.streamk = schedule[0] == 's';
    if (pair) force.pair = pair[0] == '1';
    const GemmShape shape{a.M, a.K, a.N, a.bits, a.group, a.y_dtype == LUX_DTYPE_BFLOAT16, push != nullptr, push ? push->ld : a.N, push ? push->col0 : 0, a.residual != nullptr};
    return choose_gemm_plan(shape, sm_count, force, getenv("LUXCUDA_QMM_NO_YTMA") != nullptr, pl) && encode_tiled_fn() != nullptr;
}

template <int BITS, bool EPI>
cudaError_t launch_gemm_pair_t(const CUtensorMap& tmap, const CUtensorMap& tmap_w, const CUtensorMap& tmap_y, const GemmParams& p, const GemmPlan& pl, int sm_count, cudaStream_t stream) {
    auto kern = qmm_tc_pair_kernel<BITS, EPI>;
    static std::atomic<bool> attr_set[64];
    if (cudaError_t e = allow_smem(kern, kGemmSmemLimit, attr_set)) return e;
    // one pair of CTAs per pair of SMs (the kernel carries its cluster shape), unless there are fewer pair tiles
    const int pairs = ((pl.n_tiles + 1) / 2) * pl.m_tiles;
    const int grid = 2 * std::min(sm_count / 2, pairs);
    kern<<<grid, kNumThreads, pl.smem, stream>>>(tmap, tmap_w, tmap_y, p);
    return cudaGetLastError();
}

// SK: stream-K, else whole tiles
template <int BITS, bool SK, bool EPI>
cudaError_t launch_gemm_t(const CUtensorMap& tmap, const CUtensorMap& tmap_w, const GemmParams& p, const GemmPlan& pl, int sm_count, cudaStream_t stream) {
    auto kern = SK ? qmm_tc_kernel<BITS, EPI> : qmm_tc_tiles_kernel<BITS, EPI>;
    static std::atomic<bool> attr_set[64];
    if (cudaError_t e = allow_smem(kern, kGemmSmemLimit, attr_set)) return e;
    // one CTA per SM, unless the launch has fewer units of work (tiles, or k-stages under stream-K) than that
    const long long units = (long long)pl.m_tiles * pl.n_tiles * (SK ? (p.K / kBK + kSub - 1) / kSub : 1);
    const int grid = (int)std::min<long long>(sm_count, units);
    kern<<<grid, kNumThreads, pl.smem, stream>>>(tmap, tmap_w, p);
    return cudaGetLastError();
}

}  // namespace

bool qmm_tc_supported(const QmmArgs& a, int sm_count) {
    GemmPlan pl;
    return make_gemm_plan(a, sm_count, nullptr, &pl);
}

// Scratch of a launch: one partial accumulator and one flag word per CTA (see SegIter).  The flags must be zero
// before the first launch; every launch leaves them zero.
size_t qmm_tc_workspace_bytes(int sm_count) { return kWsFlagBytes + (size_t)sm_count * kTileN * kMaxBM * sizeof(float); }

cudaError_t launch_qmm_tc(const QmmArgs& a, void* workspace, int sm_count, cudaStream_t stream, const char** name,
                          const ShardPush* push) {
    GemmPlan pl;
    if (!make_gemm_plan(a, sm_count, push, &pl) || !workspace || sm_count * sizeof(uint32_t) > kWsFlagBytes) return cudaErrorInvalidValue;
    int* err = a.error ? a.error : error_word();
    if (!err) return cudaErrorMemoryAllocation;
    // x as a 2-D tensor [M rows][K], boxes of 64 elements (128 bytes) x bm rows, 128-byte swizzle;
    // rows past M are filled with zeros by the copy engine
    CUtensorMap tmap;
    const cuuint64_t dims[2] = {(cuuint64_t)a.K, (cuuint64_t)a.M};
    const cuuint64_t strides[1] = {(cuuint64_t)a.K * 2};
    const cuuint32_t box[2] = {(cuuint32_t)kBK, (cuuint32_t)(pl.pair ? pl.bm / 2 : pl.bm)};  // (a CTA of a pair stages half the rows)
    const cuuint32_t estr[2] = {1, 1};
    CUresult r = encode_tiled_fn()(&tmap, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(a.x), dims, strides, box,
                                   estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        set_last_error("cuTensorMapEncodeTiled failed (%d)", (int)r);
        return cudaErrorInvalidValue;
    }
    // the packed weights as bytes, [N rows][K*bits/8], boxes of 64 bytes x 128 rows, 64-byte swizzle
    CUtensorMap tmap_w;
    {
        const cuuint64_t wdims[2] = {(cuuint64_t)a.K * a.bits / 8, (cuuint64_t)a.N};
        const cuuint64_t wstrides[1] = {(cuuint64_t)a.K * a.bits / 8};
        const cuuint32_t wbox[2] = {64u, (cuuint32_t)kTileN};
        r = encode_tiled_fn()(&tmap_w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint32_t*>(a.wq), wdims, wstrides, wbox,
                              estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        if (r != CUDA_SUCCESS) {
            set_last_error("cuTensorMapEncodeTiled (weights) failed (%d)", (int)r);
            return cudaErrorInvalidValue;
        }
    }
    GemmParams p;
    p.wq = a.wq;
    p.scales = (const __nv_bfloat16*)a.scales;
    p.biases = (const __nv_bfloat16*)a.biases;
    p.y = a.y;
    int* derr = nullptr;
    if (cudaHostGetDevicePointer((void**)&derr, err, 0) != cudaSuccess) return cudaGetLastError();
    p.error = derr;
    p.M = a.M; p.K = a.K; p.N = a.N;
    p.gshift = a.group == 32 ? 5 : (a.group == 64 ? 6 : 7);
    p.y_bf16 = a.y_dtype == LUX_DTYPE_BFLOAT16;
    p.world = 1; p.ld = a.N; p.col0 = 0;
    for (int r = 0; r < kMaxShardWorld; r++) p.y_all[r] = nullptr;
    p.y_all[0] = a.y;
    if (push && push->world > 1) {
        if (push->world > kMaxShardWorld) return cudaErrorInvalidValue;
        p.world = push->world; p.ld = push->ld; p.col0 = push->col0;
        // own copy first, then the peers
        int k = 0;
        p.y_all[k++] = push->y[push->me];
        for (int r = 0; r < push->world; r++)
            if (r != push->me) p.y_all[k++] = push->y[r];
    }
    p.bias = a.bias; p.residual = a.residual; p.act = a.act; p.r_bf16 = a.r_bf16;
    p.bm = pl.bm; p.w_slots = pl.w_slots; p.n_tiles = pl.n_tiles; p.m_tiles = pl.m_tiles;
    p.ws_flags = static_cast<uint32_t*>(workspace);
    p.ws = reinterpret_cast<float*>(static_cast<unsigned char*>(workspace) + kWsFlagBytes);
    p.y_tma = 0;
    if (pl.pair) {
        // y as a 2-D tensor [M rows][N] of bf16, boxes of 128 columns x bm rows, for the epilogue's TMA store
        CUtensorMap tmap_y = tmap;
        p.y_tma = pl.y_tma;
        if (p.y_tma == 1) {
            const cuuint64_t ydims[2] = {(cuuint64_t)a.N, (cuuint64_t)a.M};
            const cuuint64_t ystrides[1] = {(cuuint64_t)a.N * 2};
            const cuuint32_t ybox[2] = {(cuuint32_t)kTileN, (cuuint32_t)pl.bm};
            r = encode_tiled_fn()(&tmap_y, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.y, ydims, ystrides, ybox, estr,
                                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
            if (r != CUDA_SUCCESS) {
                set_last_error("cuTensorMapEncodeTiled (y) failed (%d)", (int)r);
                return cudaErrorInvalidValue;
            }
        }
        if (name) *name = a.bits == 4 ? "qmm_tc<4,pairs>" : "qmm_tc<8,pairs>";
        if (a.epi)
            return a.bits == 4 ? launch_gemm_pair_t<4, true>(tmap, tmap_w, tmap_y, p, pl, sm_count, stream)
                               : launch_gemm_pair_t<8, true>(tmap, tmap_w, tmap_y, p, pl, sm_count, stream);
        return a.bits == 4 ? launch_gemm_pair_t<4, false>(tmap, tmap_w, tmap_y, p, pl, sm_count, stream)
                           : launch_gemm_pair_t<8, false>(tmap, tmap_w, tmap_y, p, pl, sm_count, stream);
    }
    if (name) *name = a.bits == 4 ? (pl.streamk ? "qmm_tc<4,stream-k>" : "qmm_tc<4>") : (pl.streamk ? "qmm_tc<8,stream-k>" : "qmm_tc<8>");
    if (a.epi) {
        if (a.bits == 4) return pl.streamk ? launch_gemm_t<4, true, true>(tmap, tmap_w, p, pl, sm_count, stream) : launch_gemm_t<4, false, true>(tmap, tmap_w, p, pl, sm_count, stream);
        return pl.streamk ? launch_gemm_t<8, true, true>(tmap, tmap_w, p, pl, sm_count, stream) : launch_gemm_t<8, false, true>(tmap, tmap_w, p, pl, sm_count, stream);
    }
    if (a.bits == 4) return pl.streamk ? launch_gemm_t<4, true, false>(tmap, tmap_w, p, pl, sm_count, stream) : launch_gemm_t<4, false, false>(tmap, tmap_w, p, pl, sm_count, stream);
    return pl.streamk ? launch_gemm_t<8, true, false>(tmap, tmap_w, p, pl, sm_count, stream) : launch_gemm_t<8, false, false>(tmap, tmap_w, p, pl, sm_count, stream);
}

// Device-side address of the host-visible error word (the same on every GPU: portable mapped memory).
int* device_error_word() {
    int* err = error_word();
    int* derr = nullptr;
    if (!err || cudaHostGetDevicePointer((void**)&derr, err, 0) != cudaSuccess) {
        cudaGetLastError();
        return nullptr;
    }
    return derr;
}

int take_context_error(Context* c) {
    if (!c || !c->err_host) return 0;
    return __atomic_exchange_n(c->err_host, 0, __ATOMIC_ACQ_REL);
}

// Non-zero once a kernel has given up on a bounded wait; reading clears it.
int take_device_error() {
    if (!g_error_host || !*g_error_host) return 0;
    return __atomic_exchange_n(g_error_host, 0, __ATOMIC_ACQ_REL);
}

}  // namespace luxcuda
