"""AdapterRows' plans, and the refusals of the low-rank entry points, without a GPU."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import mlx_lean_moe_amd as gdn
from mlx_lean_moe_amd import _lib

P = lambda i: ctypes.c_void_p((1 << 32) + (i << 28))  # distinct, aligned, never dereferenced


def _tiles(rows):
    plan = rows._plan.numpy()
    return plan[:rows.rows], plan[rows.rows:].reshape(-1, 3)


@pytest.mark.parametrize("M,S,without", [(0, 1, 0), (1, 1, 0), (1, 3, 1), (17, 1, 0), (40, 40, 0.5), (64, 32, 0), (500, 3, 0.1),
                                         (4096, 6, 0.0), (1000, 900, 0.2)])
def test_every_row_with_an_adapter_is_in_one_tile(M, S, without):
    rng = np.random.default_rng(M + S)
    index = np.where(rng.random(M) < without, -1, rng.integers(0, S, M))
    assert gdn.AdapterRows(index, S, device="cpu").tiles <= (rows := gdn.AdapterRows(index, S, device="cpu", distinct=S)).tiles
    for _ in range(2):
        order, tiles = _tiles(rows)
        seen = []
        for adapter, start, count in tiles:
            assert 0 <= count <= rows.tile_rows
            part = order[start:start + count]
            assert (index[part] == adapter).all()
            seen += part.tolist()
        assert sorted(seen) == np.flatnonzero(index >= 0).tolist()
        assert len(tiles) == rows.tiles
        # any other batch of the same rows fits as well
        index = rng.integers(-1, S, M)
        rows.assign(index)


def test_tiles_have_about_as_many_rows_as_adapters():
    for rows, adapters, want in ((1, 1, 16), (16, 1, 16), (17, 1, 32), (31, 2, 16), (64, 1, 64), (65, 1, 128), (5000, 1, 256),
                                 (5000, 100, 64), (0, 1, 16)):
        assert gdn.AdapterRows([i % adapters for i in range(rows)], adapters, device="cpu").tile_rows == want


def test_numbers_that_are_none_are_refused():
    for index, count in (([0, 2], 2), ([-2], 2), ([0.0], 2), ([[0]], 2), ([True], 2), ([0], 0)):
        with pytest.raises(ValueError):
            gdn.AdapterRows(index, count, device="cpu")
    with pytest.raises(ValueError, match="room"):
        gdn.AdapterRows([0, 0], 2, device="cpu").assign([0, 1])
    gdn.AdapterRows([0, 0], 2, device="cpu", distinct=2).assign([0, 1])
    rows = gdn.AdapterRows([0, 1], 2, device="cpu")
    for index in ([0], [0, 2], [0, 1, 1]):
        with pytest.raises(ValueError):
            rows.assign(index)
    runs = gdn.PackedRuns([0, 3, 5], device="cpu")
    with pytest.raises(ValueError, match="runs"):
        gdn.AdapterRows.of_runs(runs, [0], 2)
    got = gdn.AdapterRows.of_runs(runs, [1, -1], 2)
    assert got.rows == 5 and _tiles(got)[0][:3].tolist() == [0, 1, 2]


def test_argument_checks():
    lib = _lib.load()
    err = lambda: lib.gdn_last_error().decode()
    size = lib.gdn_add_low_rank_workspace_size
    wide = (ctypes.c_int * 2)(100, 64)
    need = size(1, 2, 32, 16, wide, 200, 16, 2048)  # more than one round of workgroups: two launches
    assert need == 200 * 16 * 32 * 4 and size(1, 2, 32, 16, wide, 4, 16, 2048) == 0
    for bad in ((9, 2, 32, 16, wide, 200, 16, 2048), (1, 2, 33, 16, wide, 200, 16, 2048), (1, 9, 32, 16, wide, 200, 16, 2048),
                (1, 2, 32, 16, wide, 200, 48, 2048), (1, 2, 32, 16, wide, 200, 512, 2048), (1, 2, 32, 16, None, 200, 16, 2048), (1, 2, 32, 16, wide, -1, 16, 2048)):
        assert size(*bad) == 0

    def call(widths=(100, 64), outs=(P(0), P(1)), strides=(164, 164), **over):
        a = dict(x=P(2), xs=2048, dt=1, A=P(3), B=P(4), table=P(5), S=3, blocks=len(widths), rt=32, rb=16)
        b = dict(order=P(6), tiles=P(7), nt=200, tr=16, M=40, K=2048, ws=P(8), wsb=need)
        a.update({k: v for k, v in over.items() if k in a})
        b.update({k: v for k, v in over.items() if k in b})
        n = len(widths)
        return lib.gdn_add_low_rank(*a.values(), (ctypes.c_void_p * n)(*[getattr(o, "value", o) for o in outs]),
                                    (ctypes.c_int64 * n)(*strides), (ctypes.c_int * n)(*widths), *b.values(), None)

    assert call(M=0) == 0 and call(nt=0) == 0
    assert call(widths=(0, 0), outs=(None, None)) == 0
    for over, what in [(dict(K=0), "sizes"), (dict(tr=48), "sizes"), (dict(rt=20), "sizes"), (dict(rb=48), "sizes"), (dict(rb=0), "sizes"), (dict(S=0), "sizes"),
                       (dict(dt=5), "dtype"), (dict(x=None), "null"), (dict(tiles=None), "null"), (dict(xs=2047), "width"),
                       (dict(wsb=need - 1), "workspace"), (dict(ws=None), "workspace"), (dict(A=ctypes.c_void_p(8)), "aligned"),
                       (dict(widths=(100, -1)), "block 1"), (dict(strides=(99, 164)), "block 0"),
                       (dict(outs=(P(0), None)), "block 1"),
                       (dict(widths=(1,) * 9, outs=(P(0),) * 9, strides=(9,) * 9), "blocks"),
                       (dict(widths=(1 << 30, 1 << 30), strides=(1 << 30, 1 << 30)), "too many")]:
        assert call(**over) == _lib.GDN_EINVAL and what in err(), (over, err())


def test_adapters_on_the_cpu_are_refused():
    with pytest.raises(RuntimeError, match="ROCm"):
        gdn.LowRankAdapters([[(torch.zeros(4, 8), torch.zeros(8, 4), 1.0)]])
