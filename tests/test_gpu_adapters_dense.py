"""quantized_linear with adapters beside dense weights as the checkpoint reader gives
them: bfloat16 ones widened to float32, whose product would be float32."""

from __future__ import annotations

import pytest
import torch

import mlx_lean_moe_amd as gdn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act,stored", [(torch.bfloat16, torch.float32), (torch.float16, torch.float32),
                                        (torch.bfloat16, torch.float16), (torch.float32, torch.bfloat16),
                                        (torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("wrapped", [False, True])
def test_adapters_beside_widened_weights(gpu, act, stored, wrapped):
    g = torch.Generator(device=gpu)
    g.manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, device=gpu)
    K, N = 256, 130
    w = (r(N, K) * K ** -0.5).bfloat16().to(stored)
    adapters = gdn.LowRankAdapters([[((r(8, K) * K ** -0.5).to(act), r(N, 8).to(act), 0.5)] * 2])
    index = [0, -1, 1, 1, 0, -1]
    rows = gdn.AdapterRows(index, 2, device=gpu)
    x, res = r(2, 3, K).to(act), r(2, 3, N).to(act)
    weights = gdn.LinearWeights(w, None) if wrapped else w
    for residual in (None, res):
        # the weights are values of x's dtype in all these cases but bfloat16 rows beside float16
        # weights, where both sides round them: the same product, and the adapters on top
        want = gdn.quantized_linear(x, w.to(act), residual=residual)
        assert want.dtype == act
        gdn.add_low_rank(want.view(6, N), x.view(6, K), adapters, rows)
        got = gdn.quantized_linear(x, weights, residual=residual, adapters=adapters, adapter_rows=rows)
        assert got.dtype == act and torch.equal(got, want)
