"""What the selective scan and the block-scaled 8-bit product choose for given
sizes: the framework's own plan headers, compiled for the host."""

from __future__ import annotations

import os
import subprocess
import tempfile

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlx-lean-moe_amd", "csrc")

_PROGRAM = r"""
#include "gdn_fp8_plan.h"
#include "gdn_ssm_plan.h"
#include <cstdio>
int main() {
    char what;
    while (std::scanf(" %c", &what) == 1) {
        long long v[8];
        const int count = what == 's' ? 8 : 4;
        for (int i = 0; i < count; ++i)
            if (std::scanf("%lld", v + i) != 1) return 1;
        if (what == 's') {
            const gdn::ScanPlan p = gdn::scan_plan(v[0], int(v[1]), v[2], v[3], int(v[4]), int(v[5]), int(v[6]), int(v[7]));
            std::printf("%d %d %d %lld\n", p.heads, p.waves, p.segmented ? 1 << p.shift : 0, (long long)p.bytes);
        } else {
            const bool exact = v[0];
            const int M = int(v[1]), N = int(v[2]), kb = int((v[3] + 127) / 128);
            if (gdn::skinny(M, kb)) {
                std::printf("skinny\n");
                continue;
            }
            const gdn::Fp8Cut c = gdn::fp8_cut(exact, M, N, kb);
            const auto tile = [&](const gdn::Fp8Plan& p, int cols) {
                const gdn::Fp8Tiles& t = exact ? gdn::kTilesExact[p.kind] : gdn::kTiles16[p.kind];
                std::printf("%d:%dx%d/%d ", cols, t.tn, t.tm, p.splits);
            };
            tile(c.first, c.n0);
            if (c.n0 < N) tile(c.rest, N - c.n0);
            std::printf("\n");
        }
    }
}
"""


def _ask(lines):
    with tempfile.TemporaryDirectory() as tmp:
        src, exe = os.path.join(tmp, "plan.cpp"), os.path.join(tmp, "plan")
        with open(src, "w") as f:
            f.write(_PROGRAM)
        subprocess.run(["g++", "-std=c++17", "-O1", "-I", CSRC, src, "-o", exe], check=True)
        out = subprocess.run([exe], input="\n".join(lines), text=True, capture_output=True, check=True).stdout
    return out.splitlines()


def scan_plans(calls):
    """``(bf16, lens, (H, P, G, N))`` each -> (heads and waves of a workgroup,
    tokens of a segment or 0)."""
    ask = [f"s {int(bf16)} {len(lens)} {sum(lens)} {max(lens)} {G} {H} {P} {N}" for bf16, lens, (H, P, G, N) in calls]
    return [tuple(map(int, line.split()[:3])) for line in _ask(ask)]


def fp8_plans(calls):
    """``(float32 results, M, N, K)`` each -> the launches' "columns:tile/splits"
    (a tile's columns of y by its rows), or "skinny"."""
    return [line.split() for line in _ask([f"f {int(exact)} {M} {N} {K}" for exact, M, N, K in calls])]


# (bfloat16 kernel, lens, (H, P, G, N), (heads, waves, tokens of a segment)): every
# workgroup shape, whole and in segments of more than one chunk, states of 16 to
# 256, head dimensions that fill no tile, more runs than a wave has lanes
_MANY = [900, 1, 0] + [1] * 35 + [0, 0, 899] + [1] * 34
SCAN_LAYOUTS = [
    (True, [500] * 8, (64, 64, 8, 128), (1, 4, 0)),
    (True, [2000, 3, 0, 1000], (64, 64, 8, 128), (2, 8, 256)),
    (True, _MANY, (64, 64, 8, 128), (2, 8, 0)),
    (True, _MANY, (64, 32, 2, 16), (2, 4, 256)),
    (True, [2000, 3, 0, 1000], (64, 32, 2, 16), (2, 4, 256)),
    (True, [2000, 3, 0, 1000], (32, 128, 2, 128), (1, 8, 256)),
    (True, [1300], (40, 96, 2, 64), (1, 8, 128)),
    (True, [1999], (24, 200, 3, 128), (1, 8, 256)),
    (True, [2000, 3, 0, 1000], (32, 64, 2, 256), (2, 8, 128)),
    (True, [1300], (32, 64, 2, 256), (1, 4, 128)),
    (True, [64, 65, 63] * 10, (32, 64, 2, 256), (2, 8, 0)),
    (True, [1300], (30, 128, 1, 256), (1, 8, 128)),
    (True, [2501], (66, 64, 2, 64), (1, 4, 512)),
    (True, [2501], (64, 56, 2, 64), (2, 8, 256)),
    (True, [2501], (64, 64, 2, 24), (2, 8, 256)),
    (True, [1300], (20, 64, 20, 32), (1, 4, 64)),
    (False, [500] * 8, (64, 64, 8, 128), (1, 4, 0)),
    (False, [2000, 3, 0, 1000], (64, 64, 8, 128), (2, 8, 256)),
    (False, _MANY, (64, 64, 8, 128), (2, 8, 256)),
    (False, [64, 65, 63] * 10, (64, 64, 8, 128), (2, 8, 0)),
    (False, _MANY, (64, 32, 2, 16), (2, 4, 128)),
    (False, [2000, 3, 0, 1000], (32, 128, 2, 128), (1, 8, 256)),
    (False, [64, 65, 63] * 10, (32, 128, 2, 128), (1, 8, 0)),
    (False, [4000], (40, 96, 2, 64), (1, 8, 512)),
    (False, [1300], (24, 200, 3, 128), (1, 8, 128)),
    (False, [1300], (32, 64, 2, 256), (1, 4, 128)),
    (False, _MANY, (32, 64, 2, 256), (2, 8, 128)),
    (False, [4000], (30, 128, 1, 256), (1, 8, 256)),
    (False, [2501], (64, 64, 2, 24), (2, 8, 128)),
    (False, [1300], (20, 64, 20, 32), (1, 4, 64)),
]

# (float32 results, M, N, K, launches): every tile with an odd number of blocks of
# K and more than the two that LDS holds at once, rows and columns that end inside
# a tile and inside a piece, K that ends inside a block
FP8_LAYOUTS = [
    (False, 512, 12352, 656, ["12352:128x256/1"]),
    (False, 1500, 4001, 1408, ["4001:128x256/1"]),
    (False, 1021, 6002, 640, ["6002:128x256/1"]),
    (False, 700, 12353, 1296, ["12353:256x256/1"]),
    (False, 1800, 7940, 1168, ["7940:256x256/1"]),
    (False, 2100, 8261, 656, ["7168:256x256/1", "1093:64x32/1"]),
    (False, 4096, 6001, 656, ["4096:256x256/1", "1905:128x256/1"]),
    (False, 513, 6401, 656, ["6401:64x64/1"]),
    (False, 301, 8001, 640, ["8001:64x32/1"]),
    (False, 130, 1030, 4112, ["1030:64x32/7"]),
    (True, 1500, 4001, 1408, ["4001:128x128/1"]),
    (True, 1021, 6002, 640, ["6002:128x128/1"]),
    (True, 2100, 8261, 656, ["7168:128x128/1", "1093:64x32/1"]),
    (True, 513, 6401, 656, ["6401:64x64/1"]),
    (True, 301, 8001, 640, ["8001:64x32/1"]),
    (True, 130, 1030, 4112, ["1030:64x32/7"]),
]
