// Which kernel, tiles and shares of K a block-scaled 8-bit product takes, by its
// sizes alone (plain C++: host code, and what a test compiles by itself).
#pragma once

#include <stdint.h>

namespace gdn {

// Up to 16 rows of up to 384 groups of 128 values in all go in one launch (the
// measurements stand at its kernel).
constexpr int kSkinnyRows = 16, kSkinnyGroups = 384;

inline bool skinny(int M, int kb) { return M <= kSkinnyRows && int64_t(M) * kb <= kSkinnyGroups; }

// The tiles of a product and how many shares of K it is cut into.
//
// What a tile costs was measured over 1 to 4096 rows of 64 to 12352 outputs, K
// 1024 to 8192: a start and an end, and a time per block of K that grows with
// the workgroups on the CU (memory's latency for the small tiles, the matrix
// cores and LDS for the large ones). From that the time of each choice: rounds
// of 256 CUs with so many workgroups each; a split adds a second launch and
// its partial sums' way through memory. Figures (us, measured; 16-bit results,
// 2048 -> 12352): 65 rows 12.5 (64 x 64) against 31 (256 x 256), 512 rows 21.8
// (128 x 256), 28.0, 32.3; 1024 rows 34 (256 x 256), 39, 49; 4096 -> 2048 at
// 200 rows 17.5 (64 x 64), 14.0 split in two, 36 (128 x 256).
struct Fp8Tiles {
    int tn, tm, per_cu;
    float step1, more, ends;  // us a block of K at one workgroup a CU, for each further one, and apart from the blocks
};
constexpr Fp8Tiles kTiles16[] = {{64, 32, 6, .35f, .12f, 2.5f}, {64, 64, 4, .45f, .15f, 3.f}, {128, 256, 1, .87f, 0.f, 7.f},
                                 {256, 256, 1, 1.65f, 0.f, 8.f}};
constexpr Fp8Tiles kTilesExact[] = {{64, 32, 6, .43f, .12f, 2.5f}, {64, 64, 4, .53f, .27f, 3.f}, {128, 128, 2, 1.25f, .55f, 5.f}};
constexpr int kMaxSplits = 8;

struct Fp8Plan {
    int kind, splits, steps;
    int64_t part_bytes;
    float us;
};

inline Fp8Plan fp8_plan(bool exact, int M, int N, int kb) {
    Fp8Plan best{0, 1, kb, 0, 1e30f};
    const int kinds = exact ? 3 : 4;
    for (int k = 0; k < kinds; ++k) {
        const Fp8Tiles& t = exact ? kTilesExact[k] : kTiles16[k];
        const int64_t tiles = ((int64_t(N) + t.tn - 1) / t.tn) * ((int64_t(M) + t.tm - 1) / t.tm);
        if (k + 1 < kinds && tiles * 512 >= int64_t(1) << 32) continue;  // more threads than a grid dimension holds
        for (int splits = 1; splits <= kMaxSplits && splits * 2 <= kb + 1; splits *= 2) {
            const int steps = (kb + splits - 1) / splits;
            const int64_t load = (tiles * splits + 255) / 256, full = load / t.per_cu;
            const int rest = int(load % t.per_cu);
            const auto round_us = [&](int n) { return n ? steps * (t.step1 + t.more * (n - 1)) + t.ends : 0.f; };
            float us = full * round_us(t.per_cu) + round_us(rest);
            if (splits > 1) us += 2.5f + 8e-6f / 4 * splits * float(M) * float(N);
            if (us < best.us)
                best = {k, splits, steps, splits > 1 ? int64_t(splits) * M * ((int64_t(N) + 3) / 4 * 4) * 4 : 0, us};
        }
    }
    best.splits = (kb + best.steps - 1) / best.steps;  // (no share without a block)
    return best;
}

// A product's columns in one launch, or the first `n0` in one and the rest in
// another with tiles of its own, where few of the large tiles would take a last
// round of the CUs: 12352 columns are 48 tiles of 256 and 64 columns more, 4096
// rows of them three rounds of 256 tiles and 16 tiles more (2048 values a row:
// 143 us whole, 117 + 9 cut at 12288). Cuts that are looked at: the last whole
// tile, and the last whole round.
struct Fp8Cut {
    int n0;  // N: not cut
    Fp8Plan first, rest;
    int64_t part_bytes() const { return first.part_bytes > rest.part_bytes ? first.part_bytes : rest.part_bytes; }
};

inline Fp8Cut fp8_cut(bool exact, int M, int N, int kb) {
    constexpr int kTile = 256;
    Fp8Cut best{N, fp8_plan(exact, M, N, kb), {}};
    const int64_t down = (int64_t(M) + kTile - 1) / kTile, whole = N / kTile;
    const int64_t cuts[2] = {whole, (whole + 1) * down / 256 * 256 / down};
    float best_us = best.first.us;
    if (whole * down >= 256)
        for (const int64_t c : cuts) {
            const int n0 = int(c * kTile);
            if (n0 <= 0 || n0 >= N) continue;
            const Fp8Cut cut{n0, fp8_plan(exact, M, n0, kb), fp8_plan(exact, M, N - n0, kb)};
            const float us = cut.first.us + cut.rest.us;
            if (us < best_us) best_us = us, best = cut;
        }
    return best;
}

}  // namespace gdn
