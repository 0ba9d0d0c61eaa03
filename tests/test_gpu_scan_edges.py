"""The selective scan where single tokens differ widely from their neighbours:
steps that forget everything, and values that are not finite.

Tolerances as in test_gpu_state_space.py, but for the state of bfloat16 inputs:
its update takes x' = d exp(..) x in three bfloat16 pieces, all 24 bits of it, so
its bound is the float32 one."""

from __future__ import annotations

import pytest
import torch

import mlx_lean_moe_amd as gdn
from .scan64 import scan64

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
U = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}


def _case(gpu, act, lens, dims, seed):
    H, P, G, N = dims
    g = torch.Generator(device=gpu)
    g.manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=gpu)
    T = sum(lens)
    return dict(x=r(T, H, P).to(DT[act]), dt=r(T, H).to(DT[act]), B=r(T, G, N).to(DT[act]), C=r(T, G, N).to(DT[act]),
                A_log=torch.linspace(-1.0, 2.7, H, device=gpu), dt_bias=r(H) * 1.5 - 2.0, D=r(H), state=r(len(lens), H, P, N))


def _offsets(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


def _within(got, ref, tol, what):
    worst = ((got.double() - ref).abs() / tol).nan_to_num(nan=float("inf")).max().item()
    assert worst <= 1, f"{what}: worst ratio {worst:.3g}"


@pytest.mark.parametrize("act", ["bf16", "f32"])
@pytest.mark.parametrize("lens", [[150], [700, 0, 70]])
def test_steps_that_forget_everything_among_small_ones(gpu, act, lens):
    """A few tokens per tile of 16 take steps so large that nothing before them
    is left (their exponents reach 1e8), the others small ones: a decay between
    two of these is as exact as ever, whatever stands before them in the sum.

    Tolerance: a tile's exponents are held to 24 bits of at most 16 x 256 (powers
    of two), 2^-13 each, so a decay within it to 2 x 2^-13 ln 2 < 2^-12; whole
    and longer ones, and float32 inputs, to the float32 bound."""
    case = _case(gpu, act, lens, (4, 64, 2, 128), 40)
    T = sum(lens)
    case["A_log"] = torch.tensor([9.0, 4.0, 1.0, 9.0], device=gpu)
    case["dt_bias"] = torch.zeros(4, device=gpu)
    g = torch.Generator(device=gpu)
    g.manual_seed(41)
    big = torch.rand(T, 4, generator=g, device=gpu) < 0.15
    small = torch.tensor([-12.0, -7.0, -4.0, -12.0], device=gpu) + torch.randn(T, 4, generator=g, device=gpu) * 0.5
    case["dt"] = torch.where(big, torch.exp(torch.rand(T, 4, generator=g, device=gpu) * 5 + 4), small).to(DT[act])
    y, S = gdn.selective_scan(**case, cu_seqlens=_offsets(lens))
    ref, state, ya, sa = scan64(**case, lens=lens)
    e = (max(lens) + 128 + 128) * 2.0 ** -24 + 2.0 ** -18
    if act == "bf16":
        _within(y, ref, U[act] * ref.abs() + (U[act] * 1.01 + 2.0 ** -12 + e) * ya, "y")
    else:
        _within(y, ref, U[act] * ref.abs() + e * ya + 2.0 ** -48, "y")
    _within(S, state, e * sa + 1e-30, "state")
