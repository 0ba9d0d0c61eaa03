// How a low-rank product is cut up, by its sizes alone (plain C++: host code, and
// what a test compiles by itself).
#pragma once

#include <stdint.h>

namespace gdn {

constexpr int kLowRankBlocks = 8;    // blocks of columns a call takes
constexpr int kLowRankWaves = 4;     // waves a workgroup, both kernels
constexpr int kLowRankColumns = 256; // columns a workgroup of the second product takes

// The first product's shares of K, in steps of 128 bytes of a row: as many as give
// each CU a workgroup, as long as every wave of each has a step.
struct LowRankPlan {
    int steps, per_wave, splits;
};

inline LowRankPlan low_rank_plan(int tiles, int rank_total, int K, int elem, int ranks_per_group) {
    LowRankPlan p;
    p.steps = int((int64_t(K) * elem + 127) / 128);
    const int64_t groups = int64_t(tiles) * ((rank_total + ranks_per_group - 1) / ranks_per_group);
    int64_t splits = groups >= 256 ? 1 : 256 / (groups > 0 ? groups : 1);
    const int most = (p.steps + kLowRankWaves - 1) / kLowRankWaves;
    if (splits > most) splits = most;
    if (splits > 8) splits = 8;
    p.per_wave = int((p.steps + splits * kLowRankWaves - 1) / (splits * kLowRankWaves));
    p.splits = (p.steps + p.per_wave * kLowRankWaves - 1) / (p.per_wave * kLowRankWaves);
    return p;
}

}  // namespace gdn
