"""add_low_rank round every loop of its kernels, against float64."""

from __future__ import annotations

import pytest
import torch

import mlx_lean_moe_amd as gdn

from .low_rank_cases import CASES, index_of
from .test_gpu_low_rank import _index, _Maker, _pairs, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: c[0])
def test_against_float64(gpu, act, case):
    _, runs, ranks, K, widths = case
    _run(gpu, act, index_of(runs), ranks, K, widths, seed=K)
    torch.cuda.empty_cache()


@pytest.mark.parametrize("act", ["bf16", "f16"])
def test_two_launches_on_two_streams(gpu, act):
    """The first product's results of one stream are not the other's."""
    m = _Maker(gpu, act)
    adapters = gdn.LowRankAdapters([_pairs(m, [64] * 8, 2048, 2048)])
    rows = gdn.AdapterRows(_index(64, 8), 8, device=gpu)
    assert adapters._workspace(rows.tiles, rows.tile_rows) > 0
    xs, y = [m(64, 2048) for _ in range(2)], m(64, 2048)
    want = [gdn.add_low_rank(y.clone(), x, adapters, rows) for x in xs]
    assert not torch.equal(*want)
    streams, got = [torch.cuda.Stream() for _ in xs], []
    torch.cuda.synchronize()
    for i in range(16):
        with torch.cuda.stream(streams[i % 2]):
            got.append(gdn.add_low_rank(y.clone(), xs[i % 2], adapters, rows))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i % 2]) for i, g in enumerate(got))
