// How a product of microscaled operands with few rows of x (mx4_tile_kernel, mx4_gemm.cu) is cut, as plain host arithmetic.
#pragma once
#include <algorithm>
#include <cstdint>

namespace luxcuda {
namespace mx4_plan {

constexpr int kStageK = 256;              // codes along K per stage: 128 bytes of a row, one swizzle span
constexpr int kTileN = 128;               // rows of W per tile
constexpr int kTileM = 128;               // rows of x per tile, at most
constexpr int kMmaK = 64;                 // codes along K per MMA
constexpr int kMaxStages = 6;
constexpr int kMaxSplit = 8;              // CTAs of a cluster
constexpr int kScaleTile = 512;           // bytes of a scale tile (128 rows x 4 blocks)
constexpr int kScaleCols = 4;             // and its columns of tensor memory
constexpr int kABytes = kTileN * 128;
constexpr int kSmemMax = 227 * 1024;
constexpr int kSmemReserved = 1024;       // of every CTA, beside what it asks for
constexpr int kTmemCols = 512;            // of an SM

// How a launch is cut: parts of K (CTAs of a cluster) and stages per CTA.
// A part costs 0.22 us per stage of 256 codes, a cluster about half a microsecond each time its size doubles: parts of eight stages
// are the best of the two, shorter ones where there are hardly any CTAs.  All CTAs have to find room at once (in four fifths of the
// slots: a cluster's CTAs have to lie in one group of SMs), and the ring is as deep as leaves the next launch of a chain, which fills
// its own meanwhile, some two fifths of the machine's shared memory.  Measured one after another, x behind the wait, us, (parts, stages):
//   1 x 4096 x 4096     (1,6) 6.0  (2,6) 4.8  (4,4) 5.2  (8,3) 4.9        8 x 11008 x 4096   (4,6) 7.5  (6,5) 7.0  (8,3) 7.0
//   1 x 4096 x 11008    (1,6) 7.8  (2,4) 6.9  (2,6) 11.1 (4,2) 6.7        16 x 8192 x 28672  (1,4) 22.3 (1,6) 27.1 (2,4) 27.2
//   8 x 4096 x 22016    (1,4) 10.5 (2,3) 10.3 (2,4) 11.9 (4,3) 14.8       48 x 4096 x 11008  (1,6) 8.5  (2,4) 7.7  (4,3) 8.6
// CTAs of a cluster wait for one another, and a CTA waits for room in tensor memory: each of a cluster asks for as much of an SM's shared
// memory as it takes of the tensor memory, so that an SM never holds one for which there is no room.
struct TilePlan {
    int bm, m_tiles, split, stages, stage_bytes, per_sm;
    long long tiles;
    uint32_t sf_col, tmem_cols;
    int smem;  // what a CTA asks for
};
// st: scale tiles along K per stage
inline TilePlan plan_tile(int M, int K, int N, int st, int sm_count) {
    const int nst = (K + kStageK - 1) / kStageK;
    TilePlan t;
    int need = 0;  // shared memory that it uses
    t.bm = M >= kTileM ? kTileM : (M + 15) & ~15;
    t.m_tiles = (M - 1) / t.bm + 1;
    t.tiles = (long long)t.m_tiles * ((N - 1) / kTileN + 1);
    t.stage_bytes = (kABytes + t.bm * 128 + 2 * st * kScaleTile + 1023) & ~1023;
    t.sf_col = (t.bm + 31) & ~31;
    auto fit = [&](int stages) {
        t.stages = std::max(2, stages);
        while (t.stages * t.stage_bytes < kTileN * t.bm * 4) t.stages++;  // (the sums take the ring's place)
        need = t.stages * t.stage_bytes + 8 * (2 * kMaxStages + 1) + 1024;
        for (t.tmem_cols = 32; t.tmem_cols < t.sf_col + t.stages * 2 * st * kScaleCols; t.tmem_cols *= 2) {}
        const int by_tmem = (int)(kTmemCols / t.tmem_cols);
        t.per_sm = std::min(kSmemMax / (need + kSmemReserved), by_tmem);
        t.smem = t.split > 1 ? std::max(need, kSmemMax / by_tmem - kSmemReserved) : need;
    };
    auto resident = [&]() { return t.tiles * t.split <= (long long)sm_count * t.per_sm * 4 / 5; };
    t.split = (int)std::min<long long>(std::min(kMaxSplit, nst), std::max((nst + 7) / 8, (int)(48 / std::min(48ll, t.tiles))));
    for (;; t.split--) {
        fit(std::min(3, (nst + t.split - 1) / t.split));
        if (t.split == 1 || resident()) break;
    }
    for (int stages = std::min(kMaxStages, (nst + t.split - 1) / t.split); stages > 3; stages--) {
        fit(stages);
        if (resident() && t.tiles * t.split * need <= (long long)sm_count * kSmemMax * 5 / 8) return t;
    }
    fit(std::min(3, (nst + t.split - 1) / t.split));
    return t;
}

}  // namespace mx4_plan
}  // namespace luxcuda
