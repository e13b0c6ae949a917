// Which kernel takes a product grouped by expert, and the GEMM's tiles (qmm_experts.cu), as plain host arithmetic.
#pragma once
#include <algorithm>
#include <cmath>
#include <cstddef>

#include "qmm_plan.h"

namespace luxcuda {

struct ExpertsShape {
    size_t rows;  // of y: what the experts get together, at most
    int experts, K, N, bits;
    bool gather;  // rows of x are fetched by index
};
// Pairs of CTAs: from so many rows an expert on average, where single ones would have so many tiles each (64 experts x 256 rows, 4096 x 2816: pairs 372 us, single
// ones 410; 64 rows: 163 and 160; 150 shapes with 32 to 1000 rows an expert and mostly fewer tiles: 3 % lost all in all, by the rows alone 12).
constexpr int kPairMean = 80, kPairTiles = 3;
inline bool experts_in_pairs(const ExpertsShape& s, int sm_count) {
    const size_t mean = (s.rows + s.experts - 1) / s.experts, tiles = (size_t)s.experts * ((mean + 127) / 128) * ((s.N + 127) / 128);
    return sm_count % 2 == 0 && s.N > 128 && mean >= (size_t)kPairMean && tiles > (size_t)kPairTiles * sm_count;
}

// Estimates of the times in microseconds, for experts that share the rows evenly: the host does not know better.  Fitted to 170 shapes (2 to 128
// experts, K 512 to 4096, N 128 to 8192, 0.5 to 90 rows an expert, 4 and 8 bit; calls from a host, launches included): the faster of the two, or
// one within 5 % of it, is taken on 162 of them, all in all 0.8 % is lost, 37 % at worst; the times are off by a seventh on average.
//   few rows (qmv_stream.cu): the row tiles of all items of eight rows, dealt over the SMs, a tile at the rate of its packed bytes but
//   not below what starting one costs; x is loaded again for every item a CTA works on;
//   many (qmm_experts.cu): rounds of tiles, a k-stage of 128 bound by dequantisation until the tiles are high; gathered rows first.
inline void experts_estimates(const ExpertsShape& s, int sm_count, double* few, double* many) {
    const double mean = (double)s.rows / s.experts, active = s.experts * (1.0 - std::exp(-mean)), m = s.rows / active;
    const double row_tiles = (s.N + 15) / 16, items = active * std::max(1.0, m / 8 + 0.29), tiles = items * row_tiles / sm_count;
    const double tile = std::max(0.15 + 0.063 * (s.K * (double)s.bits / 1024), 0.49);
    *few = 5.9 + std::max(1.0, tiles) * tile + 0.07 * std::max(1.0, tiles / row_tiles);
    const bool pairs = experts_in_pairs(s, sm_count);
    const double n_tiles = (s.N + 127) / 128, G = pairs ? sm_count / 2 : sm_count, bm = std::min(pairs ? 256.0 : 128.0, std::max(32.0, 2 * mean));
    const double T = active * std::max(1.0, m / bm + 0.35) * (pairs ? std::ceil(n_tiles / 2) : n_tiles);
    const double high = std::max(0.0, std::min(m, bm) - 48), stage = pairs ? 0.44 + 0.0017 * high : (s.bits == 8 ? 0.53 : 0.33) + 0.0051 * high;
    *many = 5.5 + (s.gather ? 0.67 + s.rows * (double)s.K * 4 / 1.85e6 : 0.0) + std::ceil(T / G) * (std::ceil(s.K / 128.0) * stage + 1.2);
}
inline bool experts_have_many_rows(const ExpertsShape& s, int sm_count) {
    if (!s.rows) return false;
    double few, many;
    experts_estimates(s, sm_count, &few, &many);
    return many < few;
}

// The decode kernel's boxes (qmv_stream.cu) of the packed weights [expert][half][row][byte]: a tile is 16 rows, eight of either half where gated.
// What a box of whole 128-byte k-blocks holds behind a row's end is the start of the row after it, which must be there: so rows below 128 bytes end
// with themselves (the k-block is filled up with zeros), and the last tile of all takes single k-blocks of a map that ends with the rows, `end`.
struct ExpertsMap {
    unsigned long long dims[4], strides[3];
    unsigned box[4];
};
inline ExpertsMap experts_map(int experts, int K, int N, int bits, bool gated, int kbc) {
    const unsigned long long row = (unsigned long long)K * bits / 8, halves = gated ? 2 : 1, rows = N / halves;
    return {{row < 128 ? row : 128, rows, halves * experts, (row + 127) / 128}, {row, rows * row, 128}, {128, (unsigned)(16 / halves), (unsigned)halves, (unsigned)kbc}};
}
inline ExpertsMap experts_map_end(int experts, int K, int N, int bits, bool gated) {  // (three dimensions)
    ExpertsMap m = experts_map(experts, K, N, bits, gated, 1);
    m.dims[0] = m.strides[0];
    return m;
}
// of `tiles` tiles from tile0 on of expert e: those that take the first of the two maps
constexpr int experts_whole(bool k_tail, int e, int experts, int tile0, int tiles, int n_rt) { return k_tail && e + 1 == experts && tile0 + tiles == n_rt ? tiles - 1 : tiles; }

constexpr int kExpertStages = 4, kExpertGroups = 4, kExpertEpis = 4;  // of the GEMM (see qmm_experts.cu)
constexpr int kLowRows = 128;                                         // rows of x of a single CTA's tile, at most: half an accumulator's columns
constexpr int y_pitch(bool gated) { return gated ? kTileN + 16 : 2 * kTileN; }  // of a finished tile in shared memory, bytes a row of x (gated: off the banks)
struct ExpertsPlan {
    int bm, box, w_slots, n_tiles;  // box: rows of x per TMA box, a divisor of what a CTA fetches; n_tiles: of pairs two
    bool pair, y_staged;
    size_t smem;
};
// bm: an expert of twice the average still takes one tile, as far as there is room; lower tiles leave shared memory to L1, which holds the rows'
// scales.  Weight rings: a stage of each group's, one unit at 4 bit, two at 8 bit (one: 89 us against 70 at 8 x 32 rows, 4096 x 8192; more than a
// stage: the same).  y_pieces: y leaves in 16-byte pieces of its rows.
inline ExpertsPlan plan_experts(const ExpertsShape& s, bool gated, bool y_pieces, int sm_count, int force_pair = -1) {
    ExpertsPlan p;
    const size_t mean = (s.rows + s.experts - 1) / s.experts;
    const int n_tiles = (s.N + kTileN - 1) / kTileN;
    p.pair = force_pair >= 0 ? force_pair == 1 && sm_count % 2 == 0 : experts_in_pairs(s, sm_count);
    p.n_tiles = p.pair ? (n_tiles + 1) / 2 : n_tiles;
    p.y_staged = p.pair && y_pieces;
    p.w_slots = s.bits == 8 ? 2 : 1;
    const int step = p.pair ? 32 : 16;
    p.bm = (int)std::min<size_t>(p.pair ? kMaxBM : kLowRows, std::max<size_t>(32, (2 * mean + step - 1) / step * step));
    for (;; p.bm -= step) {  // (pairs without a gate: their finished tiles cost some rows, at 8 bit more)
        p.smem = 1024 + kGemmCtlBytes + (size_t)kExpertStages * kSub * (p.pair ? p.bm / 2 : p.bm) * 128 + (size_t)p.w_slots * kExpertGroups * kWUnitBytes +
                 (p.pair ? (size_t)(p.y_staged ? p.bm * y_pitch(gated) : 0) : (size_t)kExpertEpis * kEpiStageBytes) + (size_t)8 * (s.experts + 1);
        if (p.smem <= (size_t)kGemmSmemLimit) break;
    }
    const int half = p.pair ? p.bm / 2 : p.bm;  // rows a CTA fetches
    for (p.box = 64; half % p.box; p.box -= 16) {}
    return p;
}

}  // namespace luxcuda
