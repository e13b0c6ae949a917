// What the prefill GEMMs (qmm_tc.cu, qmm_experts.cu) share: barriers, tensor memory, TMA, and the two roles that bring the weights, one that
// fetches packed words and one that dequantises them into tensor memory.  qmm_tc.cu says how the roles of a CTA work together.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>

#include "dequant.cuh"
#include "internal.h"
#include "qmm_plan.h"

namespace luxcuda {

constexpr int kDqWarps = 4 * kDqGroups;
static_assert(kDqGroups == kStagesB, "a group always owns the same slot (and its waits, by parity, cannot alias)");
constexpr int kTmaWarp = kEpiWarps + kDqWarps, kMmaWarp = kTmaWarp + 1, kWWarp = kMmaWarp + 1;
constexpr int kNumThreads = (kWWarp + 1) * 32;
constexpr uint32_t kTmemCols = 512, kAColBase = 256, kAColsPerSub = kBK / 2, kAColsPerSlot = kSub * kAColsPerSub;
constexpr uint32_t kWaitClocks = 4000000000u;

__device__ __forceinline__ uint32_t s32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint64_t* b, uint32_t n) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(s32(b)), "r"(n));
}
__device__ __forceinline__ void mbar_arrive(uint64_t* b) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(s32(b)) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* b, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(s32(b)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint64_t* b, uint32_t parity) {
    uint32_t ok;
    // (the hint, in ns, lets the hardware hold a waiting warp instead of having it poll: polls take issue slots)
    asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3; selp.u32 %0, 1, 0, p; }"
                 : "=r"(ok) : "r"(s32(b)), "r"(parity), "r"(20000u) : "memory");
    return ok != 0;
}
// Bounded wait, about two seconds of SM clock (a poll may itself last 20 us: counting polls would not bound it).  Returns
// false (and raises *abort_flag) when the barrier does not flip within the limit or another role has already given up.
__device__ __forceinline__ bool mbar_wait(uint64_t* b, uint32_t parity, volatile int* abort_flag) {
    if (mbar_try(b, parity)) return true;
    const uint32_t t0 = clock();
    uint32_t i = 0;
    do {
#pragma unroll 1
        for (uint32_t end = i + 64; i < end; i++) {
            if (i > 4) __nanosleep(40);  // waiting roles must not steal issue slots from the working ones
            if (mbar_try(b, parity)) return true;
        }
    } while (!*abort_flag && (uint32_t)clock() - t0 < kWaitClocks);
    *abort_flag = 1;
    return false;
}

// Same bound, no back-off, for the warp whose wake-up latency is on the tensor pipe's critical path.  Whole warp; the vote
// makes the answer, and with it the control flow behind it, uniform for the compiler.
__device__ __forceinline__ bool mbar_wait_warp(uint64_t* b, uint32_t parity, volatile int* abort_flag) {
    if (__all_sync(0xffffffffu, mbar_try(b, parity))) return true;
    const uint32_t t0 = clock();
    do {
#pragma unroll 1
        for (uint32_t i = 0; i < 64; i++)
            if (__all_sync(0xffffffffu, mbar_try(b, parity))) return true;
    } while (__all_sync(0xffffffffu, !*abort_flag && (uint32_t)clock() - t0 < kWaitClocks));
    *abort_flag = 1;
    return false;
}
// The epilogue warps' wait.  One answer for a warp, whose loads from tensor memory are collective: a lane may still have seen the barrier flip when
// others gave up.
__device__ __forceinline__ bool mbar_wait_epi(uint64_t* b, uint32_t parity, volatile int* abort_flag) {
    return __all_sync(0xffffffffu, mbar_wait(b, parity, abort_flag));
}
// ... and one for all WARPS warps where they meet at the named barrier BAR before they wait again (and they meet there now).
template <int BAR, int WARPS>
__device__ __forceinline__ bool mbar_wait_epis(uint64_t* b, uint32_t parity, volatile int* abort_flag) {
    uint32_t all;
    asm volatile("{ .reg .pred p, q; setp.ne.u32 q, %1, 0; bar.red.and.pred p, %2, %3, q; selp.u32 %0, 1, 0, p; }"
                 : "=r"(all) : "r"((uint32_t)mbar_wait(b, parity, abort_flag)), "n"(BAR), "n"(WARPS * 32) : "memory");
    return all != 0;
}
// After an abort nobody waits for the copies and MMAs in flight any more; before the CTA frees its tensor memory and ends
// they get two milliseconds, far more than they take.  Every thread, behind the barrier at which all roles have returned.
__device__ __forceinline__ void settle_after_abort(volatile int* abort_flag) {
    if (!*abort_flag) return;
    const uint32_t t0 = clock();
    while ((uint32_t)clock() - t0 < 4000000u) __nanosleep(1000);
}
__device__ __forceinline__ bool elect_one() {  // whole warp: true in one lane, always the same
    uint32_t r;
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(r));
    return r != 0;
}

// ---- tcgen05 / TMEM ------------------------------------------------------------
__device__ __forceinline__ void tmem_alloc(uint32_t* dst_smem, uint32_t ncols) {  // whole warp
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s32(dst_smem)), "r"(ncols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t taddr, uint32_t ncols) {  // whole warp
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(s32(bar)) : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem desc], bf16 inputs, fp32 accumulate
__device__ __forceinline__ void tc_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{ .reg .pred p; setp.ne.b32 p, %4, 0;\n"
        "  tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }"
        ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}
// 16 consecutive 32-bit columns of this thread's TMEM lane <- 16 registers
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
          "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// Shared-memory matrix descriptor: K-major tile, rows of 128 bytes, 128-byte swizzle,
// 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t umma_desc_sw128(uint32_t smem_addr) {
    uint64_t d = 0;
    d |= (uint64_t)((smem_addr & 0x3FFFFu) >> 4);   // start address, 16-byte units
    d |= (uint64_t)1 << 16;                          // leading-dimension byte offset (unused for swizzled K-major)
    d |= (uint64_t)(1024 >> 4) << 32;                // stride-dimension byte offset: 8 rows x 128 B
    d |= (uint64_t)1 << 46;                          // descriptor version (sm_100)
    d |= (uint64_t)2 << 61;                          // layout: SWIZZLE_128B
    return d;
}
// Instruction descriptor, kind::f16: D = F32, A = B = BF16, both K-major, M x N.
__host__ __device__ constexpr uint32_t umma_idesc(int M, int N) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

// ---- TMA -----------------------------------------------------------------------
__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
        ::"r"(s32(dst)), "l"(map), "r"(x), "r"(y), "r"(s32(bar)) : "memory");
}

// ---- pairs of CTAs (cta_group::2) --------------------------------------------------
constexpr uint32_t kPeerBitMask = 0xFEFFFFFFu;  // a shared::cluster address with this bit cleared is CTA 0's copy
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_alloc_pair(uint32_t* dst_smem, uint32_t ncols) {  // whole warp, the same warp in both CTAs
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s32(dst_smem)), "r"(ncols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
// arrive on CTA 0's copy of a barrier (from either CTA)
__device__ __forceinline__ void mbar_arrive_cta0(uint64_t* b) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(s32(b) & kPeerBitMask) : "memory");
}
// arrives once on the barrier at this offset in both CTAs when the MMAs issued so far have completed
__device__ __forceinline__ void tc_commit_pair(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(s32(bar)), "h"((uint16_t)3) : "memory");
}
__device__ __forceinline__ void tc_mma_ts_pair(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    const uint32_t z = 0;
    asm volatile(
        "{ .reg .pred p; setp.ne.b32 p, %4, 0;\n"
        "  tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5, %5, %5, %5, %5}, p; }"
        ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(z) : "memory");
}
// this CTA's half of an x tile into its own shared memory, completion counted on CTA 0's barrier (no multicast)
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
        ::"r"(s32(dst)), "l"(map), "r"(x), "r"(y), "r"(s32(bar) & kPeerBitMask) : "memory");
}


__device__ __forceinline__ uint32_t ldg_u16(const uint16_t* p) {  // zero-extended straight into a 32-bit register
    uint32_t v;
    asm volatile("ld.global.nc.u16 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}

// scale_fast_ok of two
__device__ __forceinline__ bool scales_fast_ok(uint32_t s) {
    const uint32_t u = (s & 0x7FFF7FFFu) - 0x00800080u;  // (a borrow leaves the low half's top bit)
    return ((u | (u + 0x43804380u)) & 0x80008000u) == 0;
}

// 32 weights of one row (one scale) -> 16 registers of bf16 pairs in natural k order.
// The matrix instruction wants neighbours in k side by side, which dequant.cuh's masks do not yield (they pair weights 4
// apart, and a byte permute per pair put them in order afterwards: 9 integer operations per 8 weights at 4 bit, 10 at 8
// bit).  Here a permute puts them there.  4 bit: the low codes of all bytes by one mask, the high ones by another; then byte i of
// the first into the low half, q_2i, and of the second into the high one, 16 * q_2i+1, whose scale is 2^-4 of the low one's, and
// above either the first's sign, zero: 6 operations.  8 bit: two bytes into the two halves, which is all: 4 operations.  The
// products are the same (see dequant.cuh for the 2^-133 form).
template <int BITS, bool FAST>
__device__ __forceinline__ void dequant_32(const uint32_t* w, uint32_t s, uint32_t b2, uint32_t (&out)[16]) {
    if (BITS == 4) {
        const uint32_t s2 = FAST ? s + 0x40804280u : s;  // FAST: (s * 2^133, s * 2^129)
#pragma unroll
        for (int c = 0; c < 4; c++) {
            if (FAST) {
                const uint32_t lo = w[c] & 0x0F0F0F0Fu, hi = w[c] & 0xF0F0F0F0u;
#pragma unroll
                for (int i = 0; i < 4; i++) out[4 * c + i] = fma_bf16x2(prmt(lo, hi, 0x8480u + 0x1111u * i), s2, b2);
            } else {
                uint32_t r[4];  // r[i] = (w^_i, w^_{i+4})
                dequant4_general(w[c], s2, b2, r);
                out[4 * c + 0] = prmt(r[0], r[1], 0x5410u);
                out[4 * c + 1] = prmt(r[2], r[3], 0x5410u);
                out[4 * c + 2] = prmt(r[0], r[1], 0x7632u);
                out[4 * c + 3] = prmt(r[2], r[3], 0x7632u);
            }
        }
    } else {
        const uint32_t s2 = FAST ? s + 0x42804280u : s;
#pragma unroll
        for (int c = 0; c < 8; c++) {
            if (FAST) {
                out[2 * c] = fma_bf16x2(prmt(w[c], 0u, 0x4140u), s2, b2);
                out[2 * c + 1] = fma_bf16x2(prmt(w[c], 0u, 0x4342u), s2, b2);
            } else {
                uint32_t r[2];  // (w^_0, w^_2), (w^_1, w^_3)
                dequant8_general(w[c], s2, b2, r);
                out[2 * c] = prmt(r[0], r[1], 0x5410u);
                out[2 * c + 1] = prmt(r[0], r[1], 0x7632u);
            }
        }
    }
}

// ---- roles common to the kernels ----
// Whole tiles, every `step`-th one from `tile` on (the interface of SegIter).
struct TileIter {
    int tile_, step, total, nst;
    __device__ __forceinline__ bool valid() const { return tile_ < total; }
    __device__ __forceinline__ int tile() const { return tile_; }
    __device__ __forceinline__ int s_lo() const { return 0; }
    __device__ __forceinline__ int s_hi() const { return nst; }
    __device__ __forceinline__ void next() { tile_ += step; }
};
// The CTA's stages are counted 0, 1, 2, ... along its sequence of segments, alike in every role; dequantising group g owns
// the counts = g (mod GROUPS).
//
// One thread: the packed weights, unit after unit into the ring of the group that owns the stage.  GROUPS stages at a time,
// one for each group: first units first, so that with a single slot per group no group waits for another's second unit
// (8 bit).  Every stage is UPS units, so that the rings advance alike; the odd sub-block's partner is announced without a load.
// at(seg): where the tile's weights lie (two ints, whatever they mean to load); load(dst, first byte of the rows, at, barrier).
template <int BITS, int GROUPS = kDqGroups, class Prm, class Seg, class At, class Load>
__device__ __forceinline__ void weight_producer(const Prm& p, Seg seg, int nks, unsigned char* ring, uint64_t* wfull, uint64_t* wempty,
                                                volatile int* abort_flag, const At& at, const Load& load) {
    constexpr int UPS = BITS == 8 ? 2 : 1;  // weight units (128 rows x 64 packed bytes) per pipeline stage
    int2 row[GROUPS];
    int stage[GROUPS], cnt = 0, slot = 0;
    uint32_t ph = 1;
    auto flush = [&]() {
#pragma unroll
        for (int u = 0; u < UPS; u++) {
#pragma unroll
            for (int g = 0; g < GROUPS; g++) {
                if (g >= cnt) break;
                const int i = g * kMaxWSlots + slot;
                if (!mbar_wait(wempty + i, ph, abort_flag)) return false;
                if (u == 0 || stage[g] * kSub + u < nks) {
                    mbar_expect_tx(wfull + i, kWUnitBytes);
                    load(ring + (g * p.w_slots + slot) * kWUnitBytes, stage[g] * (kSub * kBK * BITS / 8) + u * 64, row[g], wfull + i);
                } else {
                    mbar_arrive(wfull + i);
                }
            }
            if (++slot == p.w_slots) { slot = 0; ph ^= 1; }
        }
        cnt = 0;
        return true;
    };
    for (; seg.valid(); seg.next()) {
        const int2 n0 = at(seg);
        const int s_hi = seg.s_hi();
        for (int st = seg.s_lo(); st < s_hi; st++) {
#pragma unroll
            for (int g = 0; g < GROUPS; g++)
                if (g == cnt) { row[g] = n0; stage[g] = st; }
            if (++cnt == GROUPS && !flush()) return;
        }
    }
    flush();
}
// One warp (lane quarter of group grp; a warp may only touch its own quarter of the TMEM lanes): the thread owns row r of
// every tile.  There are as many stages in flight as groups, so a group always writes the same slot.
// What bounds it is its instructions, GROUPS such warps to a scheduler, and the instruction caches that all roles share;
// hence row pointers per tile (a division each), one copy of the code for both sub-blocks, one arrival per warp.
// A group always writes the same slot of the A ring: `empty` and a_tmem are its, arrive() says that it is full.
// row_of(seg, r): the row of wq, scales and biases that is row r of the tile.
template <int BITS, int GROUPS = kDqGroups, class Prm, class Seg, class RowOf, class Arrive>
__device__ __forceinline__ void dequant_role(const Prm& p, Seg seg, int grp, int r, int nks, const unsigned char* wring, uint64_t* wfull,
                                             uint64_t* wempty, uint64_t* empty, uint32_t a_tmem, volatile int* abort_flag,
                                             const RowOf& row_of, const Arrive& arrive) {
    constexpr int UB = 16 / BITS;           // blocks of 32 weights in a unit's 64 bytes of a row
    constexpr int UPS = BITS == 8 ? 2 : 1;  // weight units (128 rows x 64 packed bytes) per pipeline stage
    const int gpr = p.K >> p.gshift;
    const int ng_full = (kSub * kBK) >> p.gshift;  // scale groups per full stage: 4, 2 or 1
    const bool vec_ok = (gpr % ng_full) == 0;      // then a stage's scales of one row are one aligned vector
    // row r of a unit in shared memory is 64 bytes, its 16-byte chunk c sits at c ^ ((r >> 1) & 3)
    const uint32_t wsw = (uint32_t)(r >> 1) & 3u;
    const unsigned char* wrow0 = wring + r * 64;
    const uint16_t *srow = nullptr, *brow = nullptr;  // scales / biases of this thread's row of the tile
    int st, end;
    bool more = true;
    auto new_rows = [&]() {
        const size_t at = (size_t)row_of(seg, r) * gpr;
        srow = reinterpret_cast<const uint16_t*>(p.scales) + at;
        brow = reinterpret_cast<const uint16_t*>(p.biases) + at;
    };
    auto settle = [&]() {  // st lies past the segment's end: the stage as far into the segments after it
        do {
            const int over = st - end;
            seg.next();
            if (!seg.valid()) {
                more = false;
                return;
            }
            st = seg.s_lo() + over;
            end = seg.s_hi();
        } while (st >= end);
        new_rows();
    };
    uint32_t sp[2], bp[2];  // scales / biases of the next owned stage of this row, bf16 pairs in group order
    auto fetch_sb = [&]() {
        const int g0 = (st * kSub * kBK) >> p.gshift;
        const uint16_t *sr = srow + g0, *br = brow + g0;
        sp[1] = 0; bp[1] = 0;
        if (vec_ok && ng_full == 4) {
            asm volatile("ld.global.nc.v2.u32 {%0,%1}, [%2];" : "=r"(sp[0]), "=r"(sp[1]) : "l"(sr));
            asm volatile("ld.global.nc.v2.u32 {%0,%1}, [%2];" : "=r"(bp[0]), "=r"(bp[1]) : "l"(br));
        } else if (vec_ok && ng_full == 2) {
            asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(sp[0]) : "l"(sr));
            asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(bp[0]) : "l"(br));
        } else if (ng_full == 4 && (gpr & 1) == 0) {  // (a load is one line per lane: four of pairs, not eight)
            asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(sp[0]) : "l"(sr));
            asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(bp[0]) : "l"(br));
            if (gpr - g0 > 2) {
                asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(sp[1]) : "l"(sr + 2));
                asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(bp[1]) : "l"(br + 2));
            }
        } else {
            const int ng = min(gpr - g0, ng_full);
            sp[0] = ldg_u16(sr); bp[0] = ldg_u16(br);
            if (ng > 1) { sp[0] |= ldg_u16(sr + 1) << 16; bp[0] |= ldg_u16(br + 1) << 16; }
            if (ng > 2) { sp[1] = ldg_u16(sr + 2); bp[1] = ldg_u16(br + 2); }
            if (ng > 3) { sp[1] |= ldg_u16(sr + 3) << 16; bp[1] |= ldg_u16(br + 3) << 16; }
        }
    };
    if (!seg.valid()) return;
    st = seg.s_lo() + grp;
    end = seg.s_hi();
    if (st >= end) settle();
    else new_rows();
    if (more) fetch_sb();
    // where a block's scale is among the stage's four, twice over; and those of two neighbouring blocks
    const bool g32 = p.gshift == 5, g64 = p.gshift == 6;
    const uint32_t at1 = g32 ? 0x3232u : 0x1010u, at2 = g32 ? 0x5454u : g64 ? 0x3232u : 0x1010u, at3 = g32 ? 0x7676u : at2, two0 = g32 ? 0x3210u : 0x1010u, two2 = g32 ? 0x7654u : at2;
    int wslot = 0;
    uint32_t wphase = 0, phase = 1;
    while (more) {
        const int nsub = min(kSub, nks - st * kSub);
        const uint32_t s_lo = sp[0], b_lo = bp[0], s_hi = sp[1], b_hi = bp[1];
        st += GROUPS;
        if (st >= end) settle();
        // GROUPS stages ahead of its use.  At 4 bit behind the proxy fence, which would wait for these loads too (777 rows in
        // groups of 32: 30.9 against 33-40 us); at 8 bit, with a fence per sub-block, here (512 x 8192 x 28672: 204 against 257).
        if (UPS == 2 && more) fetch_sb();
        bool ok = true;
#pragma unroll 1
        for (int u = 0; u < UPS; u++) {
            ok = mbar_wait(wfull + wslot, wphase, abort_flag) && ok;
            uint32_t w[16];
            const unsigned char* wrow = wrow0 + wslot * kWUnitBytes;
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const uint4 v = *reinterpret_cast<const uint4*>(wrow + ((c ^ wsw) << 4));
                w[4 * c] = v.x; w[4 * c + 1] = v.y; w[4 * c + 2] = v.z; w[4 * c + 3] = v.w;
            }
            // The reads above are generic-proxy accesses, the refill is an async-proxy write: the proxy
            // fence orders the two (without it a read still in the load pipe could see the next unit).
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if ((r & 31) == 0) mbar_arrive(wempty + wslot);
            if (++wslot == p.w_slots) { wslot = 0; wphase ^= 1; }
            if (UPS == 1 && more) fetch_sb();
            if (u >= nsub) break;  // (8 bit: an odd sub-block's partner, with nothing in it)
            if (u == 0) {
                ok = __all_sync(0xFFFFFFFFu, mbar_wait(empty, phase, abort_flag) && ok);  // tcgen05.st below is warp-collective
                phase ^= 1;
                tc_fence_after();
                if (!ok) break;
            }
            // the unit's blocks of 32 weights, each in one group
            const int blocks = UPS == 1 ? 2 * nsub : 2;
            const uint32_t a_unit = a_tmem + u * kAColsPerSub;
            uint32_t sv[UB], bv[UB];
#pragma unroll
            for (int i = 0; i < UB; i++) {
                const uint32_t at = UPS == 1 ? (i == 0 ? 0x1010u : i == 1 ? at1 : i == 2 ? at2 : at3) : (u == 0 ? (i == 0 ? 0x1010u : at1) : (i == 0 ? at2 : at3));
                sv[i] = prmt(s_lo, s_hi, at);
                bv[i] = prmt(b_lo, b_hi, at);
            }
            bool fast = scales_fast_ok(prmt(s_lo, s_hi, UPS == 2 && u == 1 ? two2 : two0));
            if (UPS == 1) fast = fast && (blocks == 2 || scales_fast_ok(prmt(s_lo, s_hi, two2)));
            // Scales out of the fast form's range are rare: one vote per unit and a loop of one copy whose operands move up, out of the way.  (A
            // branch per block, both forms side by side, and scales by shifts: 2330 instructions a stage, not 1740; 64 experts x 8 rows, 4096 x 2816,
            // 153 us against 132, 256 x 4096 x 4096 20.6 against 18.6.)
            if (__all_sync(0xFFFFFFFFu, fast)) {
#pragma unroll
                for (int i = 0; i < UB; i++) {
                    if (i == 2 && blocks == 2) break;
                    uint32_t out[16];
                    dequant_32<BITS, true>(w + i * BITS, sv[i], bv[i], out);
                    tmem_st16(a_unit + i * 16, out);
                }
            } else {
#pragma unroll 1
                for (int i = 0; i < blocks; i++) {
                    uint32_t out[16];
                    dequant_32<BITS, false>(w, sv[0], bv[0], out);
                    __syncwarp();
                    tmem_st16(a_unit + i * 16, out);
#pragma unroll
                    for (int k = 0; k + BITS < 16; k++) w[k] = w[k + BITS];
#pragma unroll
                    for (int k = 0; k + 1 < UB; k++) { sv[k] = sv[k + 1]; bv[k] = bv[k + 1]; }
                }
            }
        }
        ok = __all_sync(0xFFFFFFFFu, ok);  // (8 bit: the second unit's wait)
        if (!ok) {
            *abort_flag = 1;
            break;
        }
        tmem_st_wait();  // once per stage: both sub-blocks are in tensor memory
        tc_fence_before();
        __syncwarp();
        if ((r & 31) == 0) arrive();
    }
}

}  // namespace luxcuda
