"""Calls of add_low_rank that go round every loop of its kernels several times, for the
GPU test that makes them and the host test that asks the plan what each takes: name,
[(adapter, rows), ...] of the batch (-1: none), each projection's ranks by adapter, K,
the projections' outputs. Rows of an adapter fill neither 16 nor a tile, the outputs
no wave's 64 columns."""

from __future__ import annotations

import numpy as np

CASES = [
    # two launches: 64 rows a workgroup of the second product and more, so that its row stream turns over
    ("two_16", [(0, 9001), (-1, 7), (1, 7350), (2, 33)], [[16, 9, 3]], 72, [4097]),
    ("two_30", [(0, 9001), (-1, 7), (1, 7350), (2, 33)], [[30, 17, 16]], 72, [4097]),
    ("two_64", [(0, 1741), (-1, 7), (1, 1250), (2, 33)], [[64, 33, 5]], 72, [4097]),
    ("two_100", [(0, 9001), (-1, 7), (1, 7350), (2, 33)], [[100, 70, 16]], 72, [4097]),
    # packed prompts over two stacked projections
    ("packed", [(0, 501), (2, 700), (-1, 90), (1, 1333), (3, 17), (0, 1451)], [[32, 8, 20, 30], [16, 32, 0, 5]], 200, [8190, 4097]),
    # the first product with 16 rows and 16, 32 or 64 ranks a workgroup
    ("down_16", [(0, 1), (1, 17)], [[64, 40]], 1000, [300]),
    ("down_32", [(0, 2050), (1, 31)], [[32, 20]], 200, [8200]),
    ("down_64", [(0, 2050), (1, 31)], [[64, 40], [50, 64]], 200, [130, 70]),
    # one launch: 1024 to 4096 columns a workgroup, two to eight steps a wave
    ("one_16_1024", [(0, 800), (1, 45)], [[16, 5], [3, 12]], 136, [2113, 65]),
    ("one_16_2048", [(0, 1570), (1, 30)], [[16, 5]], 136, [2113]),
    ("one_30_2048", [(0, 1570), (1, 30)], [[30, 5]], 136, [2113]),
    ("one_16_4096", [(0, 1570), (-1, 3), (1, 30)], [[16, 5]], 136, [4161]),
    ("one_30_4096", [(0, 1570), (-1, 3), (1, 30)], [[30, 17]], 136, [4161]),
    # serving: a decode batch in which most requests have an adapter of their own
    ("decode", [(a, 1 + a % 3) for a in range(27)], [[16] * 27, [9] * 27], 136, [8192, 4096]),
]


def index_of(runs) -> list[int]:
    """The batch's adapters, its rows in no order."""
    index = np.repeat([a for a, _ in runs], [n for _, n in runs])
    return np.random.default_rng(len(index)).permutation(index).tolist()
