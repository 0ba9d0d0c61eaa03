"""What the plan takes for the calls of the GPU test of add_low_rank's loops (no GPU)."""

from __future__ import annotations

import numpy as np

import mlx_lean_moe_amd as gdn

from .low_rank_cases import CASES, index_of
from .test_low_rank_plan_host import plan  # noqa: F401  (the compiled plan)


def test_every_loop_turns_over(plan):  # noqa: F811
    steps, first = {}, set()
    for name, runs, ranks, K, widths in CASES:
        rows = gdn.AdapterRows(index_of(runs), len(ranks[0]), device="cpu")
        assert len(ranks) == len(widths), name
        padded = -(-np.array(ranks) // 16) * 16  # (projections, adapters)
        for elem in (2, 4):
            p = plan(rows.tiles, rows.tile_rows, int(padded.sum(0).max()), int(padded.max()), K, elem, widths)
            if p["columns"]:
                assert name.startswith(("one", "decode")), name
                turns = p["columns"] // 512  # of 64 columns, by each of eight waves
                kind = (elem, "one", p["held"])
            else:
                assert not name.startswith(("one", "decode")), name
                turns = p["up_rows"] // 16
                kind = (elem, "two", p["held"])
                first.add((elem, p["ranks"], p["down_rows"]))
            steps.setdefault(kind, set()).add(turns)
    for elem in (2, 4):
        for kind in ([("two", held) for held in (0, 1, 2, 4)] + [("one", held) for held in (1, 2)]):
            assert max(steps[(elem, *kind)]) > 2, (elem, kind, steps)
        assert {(elem, ranks, rows) for ranks in (16, 32, 64) for rows in (16, 32)} <= first, sorted(first)
