// How a low-rank product is cut up, by its sizes alone (plain C++: host code, and
// what a test compiles by itself).
#pragma once

#include <stdint.h>

namespace gdn {

constexpr int kLowRankBlocks = 8;      // blocks of columns a call takes
constexpr int kLowRankMostColumns = 1 << 30;  // of a block
constexpr int kLowRankTile = 256;      // rows of a plan's large tiles
constexpr int kLowRankDownWaves = 8;   // waves a workgroup of the first product, which share out K
constexpr int kLowRankUpWaves = 4;     // of the second, 64 columns each
constexpr int kLowRankColumns = 64 * kLowRankUpWaves;

// Columns of each block in groups of `columns`: how many, and where each block's end.
inline int64_t column_groups(const int* widths, int blocks, int columns, int* ends) {
    int64_t groups = 0;
    for (int j = 0; j < blocks; ++j) {
        groups += (int64_t(widths[j]) + columns - 1) / columns;
        if (ends) ends[j] = int(groups < INT32_MAX ? groups : INT32_MAX);
    }
    return groups;
}

struct LowRankPlan {
    int columns;           // of a block a workgroup takes, 16 rows of a tile, both products in one launch (0: two)
    int ranks, down_rows;  // two: ranks and rows of a tile that a workgroup of the first product takes
    int up_rows;           // and rows that one of the second does
    int steps;             // K in steps of 128 bytes of a row, shared out over the waves
    int held;              // 16-rank pieces of B that a wave keeps in registers (0: none)
};

// Two launches. Few tiles: the first product's ranks apart, 16 a workgroup, so that the
// reading of an adapter is spread; many: together, so that x is read once; between, 32
// (both launches, 64 columns, us, 16, 32 and 64 ranks a workgroup: 1024 rows of 2048, rank
// 64 8.9, 9.5, 11.0, float32 12.2, 14.5, 21.7; 2048 rows 11.5, 10.3, 11.3, float32 17.0,
// 15.5, 22.5; 4096 rows 15.9, 13.0, 12.5, float32 27.2, 23.5, 24.5; 2048 rows of 8
// adapters, rank 96 17.8, 14.7, 16.9, float32 27.4, 24.8, 37.1). 32 rows share a reading of
// the adapter where that leaves a workgroup for each CU (8192 rows of rank 64 53.8 us in
// all, 56.2 with 16 rows). The second product takes as many rows of a tile as leave 4096
// workgroups, since those share a reading of B (4096 packed rows of 6 adapters x 12288, rank
// 32: 68.4 us in all, with 2048 69.6, with 512 79.2; 8192 x 4096, rank 16 41.7, 44.1, 44.0);
// with four pieces of B to read as many as leave 512, up to 64 (rank 64, us, 16 rows, 32 and
// 64: 2048 x 4096 20.0, 18.8, 19.5, float16 23.1, 20.4, 19.3, float32 36.7, 35.0, 34.5; 1024
// x 4096 14.0, 13.7, 15.1, which 512 leaves at 32; 4096 x 8192 49.9, 44.5, 41.3, float16
// 65.0, 53.9, 48.7; 8192 x 4096, 32 rows, 64 and 128 51.8, 53.5, 54.2, float16 61.1 and 59.3
// with 32 and 64).
//
// One, where that is one round of workgroups of not many columns, and what each reads of
// A (its own adapter's rows, as every other workgroup of its block) is little. us, one
// launch and two, 2048 -> 8192 | 4096: rank 16, 1 row 4.5 and 6.4, 64 rows of 27 adapters
// 9.3 and 10.3 (4096 values a row: 11.2 and 11.5), 512 rows of one 11.9 and 13.9, 1024
// 17.1 and 18.4, 2048 (16 steps of columns) 31.7 and 27.0, 4096 54 and 54; rank 32, 1 row
// 5.5 and 6.6, 64 rows of 8 adapters 10.1 and 9.3, of 27 12.3 and 12.3, 512 rows of one
// 13.8 and 15.2; rank 64, 1 row 7.5 and 7.1, 8 rows 8.4 and 7.8, 512 19.0 and 16.2.
inline LowRankPlan low_rank_plan(int tiles, int tile_rows, int rank_total, int rank_block, int K, int elem,
                                 const int* widths, int blocks) {
    LowRankPlan p;
    const int64_t parts = int64_t(tiles) * (tile_rows / 16);
    p.ranks = 64;
    if (rank_total <= 32 || parts * ((rank_total + 31) / 32) <= 384) p.ranks = 32;
    if (rank_total <= 16 || parts * (rank_total / 16) <= 256) p.ranks = 16;
    p.down_rows = tile_rows > 16 && parts / 2 * ((rank_total + p.ranks - 1) / p.ranks) >= 256 ? 32 : 16;
    p.steps = int((int64_t(K) * elem + 127) / 128);
    p.held = rank_block <= 16 ? 1 : rank_block <= 32 ? 2 : rank_block <= 64 ? 4 : 0;
    const int64_t groups = column_groups(widths, blocks, kLowRankColumns, nullptr);
    p.up_rows = p.held == 4 && tile_rows > 64 ? 64 : tile_rows;
    while (p.up_rows > 16 && tiles * (tile_rows / p.up_rows) * groups < (p.held == 4 ? 512 : 4096)) p.up_rows /= 2;

    p.columns = 0;
    if ((p.held == 1 || p.held == 2) && p.held * 16 * int64_t(K) * elem <= 1 << 17)
        for (int columns = 512; columns <= 4096 && !p.columns; columns *= 2)
            if (parts * column_groups(widths, blocks, columns, nullptr) <= 256) p.columns = columns;
    return p;
}

}  // namespace gdn
