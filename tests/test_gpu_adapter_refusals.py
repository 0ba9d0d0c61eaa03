"""Refusals that have to come before a state changes: what follows autograd in
out_proj's product."""

from __future__ import annotations

import pytest
import torch

import mlx_lean_moe_amd as gdn

from .test_gpu_layer_adapters import D, HIDDEN, HV, _adapters, _layer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,what", [("dense", "weight"), ("dense", "residual"), ("affine4", "residual")])
def test_a_step_that_would_need_a_gradient_leaves_the_states_alone(gpu, kind, what):
    layer, _, _, _ = _layer(gpu, kind)
    layer.set_adapters(**_adapters(gpu, torch.bfloat16, names=("out_proj",)))
    x = torch.randn(3, HIDDEN, device=gpu).bfloat16()
    rows = gdn.AdapterRows([0, 1, 2], 3, device=gpu)
    pool = gdn.RecurrentStatePool(4, 4, D.conv_dim, HV, 128, 128, dtype=torch.bfloat16, device=gpu)
    cache = layer.new_cache(torch.bfloat16)
    residual = torch.randn(3, HIDDEN, device=gpu).bfloat16()
    layer.decode_batch(x, pool, slots=[3, 0, 1], residual=residual, adapter_rows=rows)
    layer(x, cache, residual=residual, adapter_rows=rows)
    kept = [t.clone() for t in (pool.ssm_state, pool.conv_buf, pool.conv_half_dev, pool.size, cache.ssm_state, cache.conv_state)]
    if what == "weight":
        layer.out_proj = layer.out_proj.clone().requires_grad_()
    else:
        residual.requires_grad_()
    for call in (lambda: layer.decode_batch(x, pool, slots=[3, 0, 1], residual=residual, adapter_rows=rows),
                 lambda: layer(x, cache, residual=residual, adapter_rows=rows)):
        with pytest.raises(RuntimeError, match="no gradient"):
            call()
    now = (pool.ssm_state, pool.conv_buf, pool.conv_half_dev, pool.size, cache.ssm_state, cache.conv_state)
    assert all(torch.equal(a, b) for a, b in zip(kept, now))
    with torch.no_grad():
        layer.decode_batch(x, pool, slots=[3, 0, 1], residual=residual, adapter_rows=rows)
        layer(x, cache, residual=residual, adapter_rows=rows)
    assert not torch.equal(pool.ssm_state, kept[0]) and not torch.equal(cache.ssm_state, kept[4])
