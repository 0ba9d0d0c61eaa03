"""The cuts that the low-rank product takes at the sizes of the GPU tests and of serving
(its plan header, compiled for the host; no GPU)."""

from __future__ import annotations

import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlx-lean-moe_amd", "csrc")

_PROGRAM = r"""
#include "gdn_low_rank_plan.h"
#include <cstdio>
int main() {
    int tiles, rows, total, block, K, elem, n, w[8];
    while (std::scanf("%d %d %d %d %d %d %d", &tiles, &rows, &total, &block, &K, &elem, &n) == 7) {
        for (int i = 0; i < n; ++i)
            if (std::scanf("%d", w + i) != 1) return 1;
        const gdn::LowRankPlan p = gdn::low_rank_plan(tiles, rows, total, block, K, elem, w, n);
        std::printf("%d %d %d %d %d %d\n", p.columns, p.ranks, p.down_rows, p.up_rows, p.steps, p.held);
    }
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    at = tmp_path_factory.mktemp("plan")
    (at / "plan.cpp").write_text(_PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", CSRC, str(at / "plan.cpp"), "-o", str(at / "plan")], check=True)

    def ask(tiles, tile_rows, rank_total, rank_block, K, elem, widths):
        line = " ".join(map(str, (tiles, tile_rows, rank_total, rank_block, K, elem, len(widths), *widths)))
        out = subprocess.run([str(at / "plan")], input=line, text=True, capture_output=True, check=True).stdout
        return dict(zip(("columns", "ranks", "down_rows", "up_rows", "steps", "held"), map(int, out.split())))

    return ask


def test_one_launch_for_few_rows(plan):
    wide = (8192, 4096)
    assert plan(1, 16, 32, 16, 2048, 2, wide)["columns"] == 512
    assert plan(27, 16, 32, 16, 2048, 2, wide)["columns"] == 2048
    assert plan(4, 256, 16, 16, 1024, 4, (1231,))["columns"] == 512
    # ranks of more than two pieces, much of A a workgroup, more than one round: two
    for call in ((1, 16, 128, 64, 2048, 2, wide), (1, 16, 16, 16, 8192, 2, wide), (200, 16, 32, 16, 2048, 2, wide),
                 (1, 16, 64, 64, 512, 2, (64,)), (1, 16, 112, 112, 64, 2, (64,))):
        assert plan(*call)["columns"] == 0, call


def test_ranks_apart_for_few_rows(plan):
    for parts, total, ranks in ((64, 64, 16), (65, 64, 32), (128, 64, 32), (192, 64, 32), (193, 64, 64), (128, 96, 32), (129, 96, 64),
                                (128, 32, 16), (129, 32, 32), (5000, 32, 32), (5000, 16, 16), (1, 65536, 64)):
        assert plan(parts, 16, total, min(total, 64), 2048, 2, (4096,))["ranks"] == ranks, (parts, total)


def test_every_kernel_is_reached(plan):
    """By the calls of the GPU tests: (M as tiles, ranks, K, outputs)."""
    one, two = set(), set()
    for elem in (2, 4):
        for call in ((1, 16, 16, 16, 8, elem, (1,)), (3, 16, 32, 32, 256, elem, (300,)), (3, 32, 64, 64, 2048, elem, (512,)),
                     (3, 16, 112, 112, 2050, elem, (130,)), (33, 256, 16, 16, 104, elem, (70,)), (33, 256, 32, 32, 104, elem, (70,)),
                     (34, 256, 64, 64, 104, elem, (70,)), (33, 256, 112, 112, 104, elem, (70,)),
                     (36, 256, 128, 64, 1100, elem, (600, 70)), (140, 16, 80, 64, 512, elem, (320, 77))):
            p = plan(*call)
            if p["columns"]:
                one.add((elem, p["held"]))
            else:
                two.add((elem, "down", p["ranks"], p["down_rows"]))
                two.add((elem, "up", p["held"]))
    for elem in (2, 4):
        assert {(elem, 1), (elem, 2)} <= one
        assert {(elem, "up", h) for h in (0, 1, 2, 4)} <= two
        assert {(elem, "down", r, 32) for r in (16, 32, 64)} <= two and (elem, "down", 16, 16) in two


def test_cuts_fit_the_tiles(plan):
    for tiles in (1, 5, 100, 5000):
        for tile_rows in (16, 32, 64, 128, 256):
            for rank in (16, 32, 48, 64, 80, 1024):
                for widths in ((1,), (64, 8192), (12352,), (4096,) * 8):
                    p = plan(tiles, tile_rows, rank * len(widths), rank, 2048, 2, widths)
                    assert p["down_rows"] in (16, 32) and tile_rows % p["down_rows"] == 0
                    assert tile_rows % p["up_rows"] == 0 and 16 <= p["up_rows"] <= 256 and p["steps"] == 32
                    assert p["held"] * 16 >= rank if p["held"] else rank > 64
                    if p["columns"]:
                        assert p["held"] in (1, 2) and p["columns"] % 512 == 0
                        assert tiles * tile_rows // 16 * sum(-(-n // p["columns"]) for n in widths) <= 256
