// How a low-rank product is cut up, by its sizes alone (plain C++: host code, and
// what a test compiles by itself).
#pragma once

#include <stdint.h>

namespace gdn {

constexpr int kLowRankBlocks = 8;      // blocks of columns a call takes
constexpr int kLowRankTile = 256;      // rows of a plan's large tiles
constexpr int kLowRankDownWaves = 8;   // waves a workgroup of the first product, which share out K
constexpr int kLowRankUpWaves = 4;     // of the second, 64 columns each
constexpr int kLowRankColumns = 64 * kLowRankUpWaves;

struct LowRankPlan {
    int ranks, down_rows;  // ranks and rows of a tile that a workgroup of the first product takes
    int steps;    // K in steps of 128 bytes of a row, shared out over the waves
    int up_rows;  // rows of a tile that a workgroup of the second product takes
    int held;     // 16-rank pieces of B that its waves keep in registers (0: none)
};

// Few tiles: the first product's ranks apart, 16 a workgroup, so that the reading of
// an adapter is spread; many: together, so that x is read once. The second takes as
// many rows of a tile as leave 4096 workgroups, since those share its
// reading of B.
inline LowRankPlan low_rank_plan(int tiles, int tile_rows, int rank_total, int rank_block, int K, int elem,
                                 int64_t column_groups) {
    LowRankPlan p;
    const int64_t parts = int64_t(tiles) * (tile_rows / 16);
    p.ranks = parts * (rank_total / 16) <= 256 || rank_total <= 16 ? 16 : rank_total <= 32 ? 32 : 64;
    p.down_rows = tile_rows > 16 && parts / 2 * ((rank_total + p.ranks - 1) / p.ranks) >= 256 ? 32 : 16;
    p.steps = int((int64_t(K) * elem + 127) / 128);
    p.up_rows = tile_rows;
    while (p.up_rows > 16 && tiles * (tile_rows / p.up_rows) * column_groups < 4096) p.up_rows /= 2;
    p.held = rank_block <= 16 ? 1 : rank_block <= 32 ? 2 : rank_block <= 64 ? 4 : 0;
    return p;
}

}  // namespace gdn
