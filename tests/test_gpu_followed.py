"""The state-space operators and fp8_block products refuse what they take no
part in: gradients, forward mode, function transforms."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import mlx_lean_moe_amd as gdn

pytestmark = pytest.mark.gpu

FP8 = gdn.QuantScheme(8, 128, "fp8_block")


def _calls(gpu):
    """name -> (call of its operands, their number)"""
    r = lambda *s: torch.randn(*s, device=gpu)
    d = gdn.StateSpaceDims(1, 2, 16, 8, 4)
    conv = [r(5, 24), r(1, 3, 24), r(24, 4), r(24)]
    scan = [r(1, 5, 2, 8), r(1, 5, 2), r(1, 5, 1, 16), r(1, 5, 1, 16), r(2), r(2), r(2), r(1, 2, 8, 16)]
    step = [r(3, 48), r(3, 2), r(3, 3, 48), r(3, 2, 8, 16), r(48, 4), r(48), r(2), r(2), r(2)]
    w = (r(130, 144) * 60).to(torch.float8_e4m3fn)
    linear = [r(4, 144), r(2, 2).abs(), r(4, 130)]
    return {"conv": (lambda *a: gdn.conv_silu(*a)[0], conv), "scan": (lambda *a: gdn.selective_scan(*a)[0], scan),
            "step": (lambda *a: gdn.selective_step(*a, d)[0], step),
            "linear": (lambda x, s, res: gdn.quantized_linear(x, {"weight": w, "scales": s}, FP8, residual=res), linear)}


@pytest.mark.parametrize("name", ["conv", "scan", "step", "linear"])
def test_followed_calls_are_refused(gpu, name):
    call, args = _calls(gpu)[name]
    want = call(*args)
    for i, a in enumerate(args):
        other = lambda t: args[:i] + [t] + args[i + 1:]
        with pytest.raises(RuntimeError, match="no gradient"):
            call(*other(a.clone().requires_grad_()))
        with torch.no_grad():
            assert torch.equal(call(*other(a.clone().requires_grad_())), want)
        with forward_ad.dual_level():
            with pytest.raises(RuntimeError, match="forward mode"):
                call(*other(forward_ad.make_dual(a, torch.ones_like(a))))
            assert torch.equal(call(*args), want)
        with pytest.raises(RuntimeError):
            torch.vmap(lambda t: call(*other(t)))(torch.stack([a, a]))
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda t: call(*other(t)).sum())(a)
    assert torch.equal(call(*args), want)
