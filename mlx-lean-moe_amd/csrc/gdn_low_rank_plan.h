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

constexpr int kLowRankSmallColumns = 64 * kLowRankDownWaves;  // of both in one launch

struct LowRankPlan {
    bool small;            // both products in one launch
    int ranks, down_rows;  // ranks and rows of a tile that a workgroup of the first product takes
    int steps;    // K in steps of 128 bytes of a row, shared out over the waves
    int up_rows;  // rows of a tile that a workgroup of the second product takes
    int held;     // 16-rank pieces of B that its waves keep in registers (0: none)
};

// Few tiles: the first product's ranks apart, 16 a workgroup, so that the reading of
// an adapter is spread; many: together, so that x is read once, and 32 rows share a
// reading of the adapter where that leaves a workgroup for each CU (8192 rows of rank
// 64 50.1 us in all, 52.6 with 16 rows). The second product takes as many rows of a
// tile as leave 4096 workgroups, since those share a reading of B (8192 x 4096, rank 64,
// and 4096 x 12288, rank 32: 54.5 and 53.2 us in all, with 512 workgroups 57 and 58).
//
// Both in one launch while that is one round of workgroups and what each reads of A is
// little (us, one launch and two, 2048 -> 8192 | 4096: 1 row of rank 16 4.4 and 6.5, of
// rank 64 6.6 and 6.8; 64 rows of 8 adapters 7.3 and 7.6; 64 rows of 27 adapters, three
// rounds, 12.3 and 11.1; 4096 -> 2048, 200 rows of rank up to 64, 512 KB each, 18.1 and
// 14.8).
inline LowRankPlan low_rank_plan(int tiles, int tile_rows, int rank_total, int rank_block, int K, int elem,
                                 int64_t column_groups, int64_t small_groups) {
    LowRankPlan p;
    const int64_t parts = int64_t(tiles) * (tile_rows / 16);
    p.ranks = parts * (rank_total / 16) <= 256 || rank_total <= 16 ? 16 : rank_total <= 32 ? 32 : 64;
    p.down_rows = tile_rows > 16 && parts / 2 * ((rank_total + p.ranks - 1) / p.ranks) >= 256 ? 32 : 16;
    p.steps = int((int64_t(K) * elem + 127) / 128);
    p.up_rows = tile_rows;
    while (p.up_rows > 16 && tiles * (tile_rows / p.up_rows) * column_groups < 4096) p.up_rows /= 2;
    p.held = rank_block <= 16 ? 1 : rank_block <= 32 ? 2 : rank_block <= 64 ? 4 : 0;
    p.small = p.held > 0 && parts * small_groups <= 256 && p.held * 16 * int64_t(K) * elem <= 1 << 18;
    return p;
}

}  // namespace gdn
