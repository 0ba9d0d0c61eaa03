// How the selective scan cuts a call into workgroups and segments, by its sizes
// alone (plain C++: host code, and what a test compiles by itself).
#pragma once

#include <stdint.h>

namespace gdn {

// How a call is cut: what a workgroup covers, and the tokens of a segment.
//
// A workgroup takes two heads of a group, or up to 128 head_dim rows of one
// (wide), or one head's 64 rows (narrow): narrow ones walk a run faster where
// most CUs are idle, wide ones read B and C for twice the work. Segments add
// the pass that sums each of them (0.6 of the main one), the chain's way
// through memory (both ways, 5.3 TB/s) and each workgroup's start and end, and
// shorten the longest walk. The estimate below is the time of each choice from
// 64 tokens' time with one and two workgroups on a CU (64 rows of 128 states,
// bfloat16 and float32 kernels) and that start; it ranks them as measured (us, 64 heads):
//   41 tokens narrow 8.6, wide 11.8; 300 whole and narrow 25.5, wide 35.5, in
//   segments of 64 28.6; 1000 in 128s 39.6, whole 100; 4096 in 256s 82, 512s
//   95, 128s 107, whole 380; 8192 in 512s 129, 256s 151; 8 runs of 2000 whole
//   and narrow 169, wide 200, in 1024s 212; 16 runs of 0 to 4096 (11 k tokens)
//   in 512s 202, 1024s 220, whole 407.
// float32, 32 heads of 128: 256 tokens narrow in 64s 32.1, whole 43.9, wide in 64s
//   36.5; 1000 wide in 64s 66.6, 128s 67.1, narrow 73; 2500 wide in 128s 145, 256s
//   162; 8192 in 512s 314, 256s 326; 8 runs of 1000 to 2000, 64 heads
//   of 64: whole and narrow 422, wide 501, in 256s 513.
//
// The estimate knows the times of 128 states only, and 512 workgroups side by side;
// only the chain's bytes go by the state. Against the best choice for the call
// (64 heads of 64; 300, 1000 and 4096 tokens, 8 runs of 1000 to 2000) it took, in
// bfloat16 and float32: 16 states 1.00 to 1.27 and 1.01 to 1.19 times as long, 64
// states 1.00 to 1.42 and 1.01 to 1.09, 256 states 1.10 to 1.21 and 1.09 to 1.42.
struct ScanPlan {
    int heads, waves;  // of a workgroup (waves of 16 head_dim rows)
    int shift;
    int64_t slots, units;
    bool segmented;
    int64_t bytes;
};

inline ScanPlan scan_plan(bool bf16, int N, int64_t T, int64_t longest, int G, int H, int P, int S) {
    const int per = H / G;
    if (longest <= 0 || longest > T) longest = T;
    ScanPlan best{};
    double best_us = 1e30;
    for (int narrow = 0; narrow < 2; ++narrow) {
        ScanPlan p;
        p.heads = !narrow && P <= 64 && per % 2 == 0 ? 2 : 1;
        p.waves = !narrow && (P > 64 || (P > 32 && p.heads == 2)) ? 8 : 4;
        if (narrow && P <= 32 && per % 2 == 0) continue;  // (half of its rows would be empty)
        const int rows = 16 * p.waves / p.heads;
        p.units = int64_t(H / p.heads) * ((P + rows - 1) / rows);
        const double alone = bf16 ? (narrow ? 4.1 : 5.9) : (narrow ? 10.4 : 14.6);
        const double paired = bf16 ? (narrow ? 5.1 : 6.2) : (narrow ? 13.0 : 22.0), ends = 9.0;
        for (int shift = 6; shift <= 12; ++shift) {
            p.segmented = shift < 12 && longest > (int64_t(1) << shift);
            if (shift < 12 && !p.segmented) continue;  // the same as whole runs
            p.shift = p.segmented ? shift : 31;
            p.slots = (T >> p.shift) + N;
            const double slots = p.segmented ? double(T >> shift) + 0.5 * N : N, groups = slots * p.units;
            const double walk = double(((p.segmented ? int64_t(1) << shift : longest) + 63) / 64);
            const double chunk = groups <= 300 ? alone : paired, side_by_side = groups < 512 ? groups : 512;
            const double work = (T / 64.0 + 0.5 * slots) * p.units / side_by_side;
            const int64_t rounds = int64_t((groups + 511) / 512);
            double us = (walk > work ? walk : work) * chunk + ends * double(rounds);
            if (p.segmented) us = 1.6 * us + double(p.slots) * H * P * S * 8 / 5.3e6 + 4;
            p.bytes = p.segmented ? p.slots * H * (int64_t(P) * S + 4) * 4 : 0;
            if (us < best_us) best_us = us, best = p;
        }
    }
    return best;
}

}  // namespace gdn
