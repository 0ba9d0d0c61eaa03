"""The block-scaled 8-bit product in each of its tiles, at ragged sizes.

Tolerances as in test_gpu_fp8.py: float32 results pass the 128 sums of a block,
a product and a sum per block; 16-bit ones are rounded once (twice with a
residual) from sums that keep 2^-11 of a block's absolute sum."""

from __future__ import annotations

import pytest
import torch

import mlx_lean_moe_amd as gdn
from . import plans

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
U = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}
# float16 values below 2^-14 lie 2^-24 apart: half of that is what rounding takes
LEAST = {"bf16": 1e-30, "f16": 2.0 ** -25, "f32": 1e-30}
FP8 = gdn.QuantScheme(8, 128, "fp8_block")


def _case(gpu, M, N, K, act, seed):
    g = torch.Generator(device=gpu)
    g.manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=gpu)
    w = (r(N, K) * 60).clamp(-440, 440).to(torch.float8_e4m3fn)
    s = torch.rand(-(-N // 128), -(-K // 128), generator=g, device=gpu) * 0.02 + 1e-3
    return (r(M, K) * torch.exp(r(M, 1))).to(DT[act]), {"weight": w, "scales": s}, r(M, N).to(DT[act])


def _reference(x, W):
    """(y, sum of |terms|) in float64, on the GPU; codes and scales of x by
    their definition (float32 quotients)."""
    M, K = x.shape
    N = W["weight"].shape[0]
    kb = -(-K // 128)
    rows = torch.zeros(M, kb * 128, device=x.device)
    rows[:, :K] = x.float()
    rows = rows.reshape(M, kb, 128)
    # (tensors on both sides: torch multiplies by the reciprocal of a number)
    s = (rows.abs().amax(-1, keepdim=True) / torch.full((1,), 448.0, device=x.device)).clamp(min=2.0 ** -126)
    q = ((rows / s).to(torch.float8_e4m3fn).double() * s.double()).reshape(M, kb * 128)[:, :K].contiguous()
    w = W["weight"].double() * W["scales"].double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    return q @ w.T.contiguous(), q.abs() @ w.abs().T.contiguous()


def _check(y, x, W, act, residual=None):
    K = x.shape[1]
    ref, mag = _reference(x, W)
    tol = mag * ((128 + K / 128 + 8) * 2.0 ** -24 if act == "f32" else 2.0 ** -11)
    tol = tol + U[act] * (ref.abs() + tol) + LEAST[act]
    if residual is not None:
        ref = ref + residual.double()
        tol = tol + U[act] * (ref.abs() + tol)
    assert y.shape == ref.shape and y.dtype == DT[act] and torch.isfinite(y).all()
    worst = ((y.double() - ref).abs() / tol).max().item()
    assert worst <= 1, f"worst ratio {worst:.3g}"


@pytest.mark.parametrize("act", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("M,N,K", [(2100, 8261, 256), (2100, 8258, 144), (4100, 4100, 128)])
def test_columns_in_two_launches_of_rows_that_start_anywhere(gpu, act, M, N, K):
    """The first launch's columns are whole tiles, its rows of y N apart: odd, or
    no multiple of a piece."""
    x, W, res = _case(gpu, M, N, K, act, M + N)
    _check(gdn.quantized_linear(x, W, FP8), x, W, act)
    _check(gdn.quantized_linear(x, W, FP8, residual=res), x, W, act, res)


@pytest.mark.parametrize("exact,M,N,K,launches", plans.FP8_LAYOUTS, ids=lambda v: "+".join(v) if isinstance(v, list) else None)
def test_each_tile(gpu, exact, M, N, K, launches):
    """Which sizes take which tiles is held by test_plans_host.py."""
    for act in ("f32",) if exact else ("bf16", "f16"):
        x, W, res = _case(gpu, M, N, K, act, M + K)
        _check(gdn.quantized_linear(x, W, FP8), x, W, act)
        _check(gdn.quantized_linear(x, W, FP8, residual=res), x, W, act, res)


@pytest.mark.parametrize("exact,M,N,K,launches", [c for c in plans.FP8_LAYOUTS if c[1] > 1000][::2],
                         ids=lambda v: "+".join(v) if isinstance(v, list) else None)
def test_rows_that_are_not_finite_stay_their_own_in_large_tiles(gpu, exact, M, N, K, launches):
    act = "f32" if exact else "bf16"
    x, W, _ = _case(gpu, M, N, K, act, 3)
    clean = gdn.quantized_linear(x, W, FP8)
    rows = [0, 255, 700, M - 1]
    for i, m in enumerate(rows):
        x[m, (131 * i + K - 1) % K] = float("nan") if i % 2 else float("-inf")
    y = gdn.quantized_linear(x, W, FP8)
    assert torch.isnan(y[rows]).all()
    keep = torch.ones(M, dtype=torch.bool, device=gpu)
    keep[rows] = False
    assert torch.equal(y[keep], clean[keep])
