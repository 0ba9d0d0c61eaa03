"""The selective scan in each of its layouts (which sizes take which is held by
test_plans_host.py), against float64.

Tolerances count roundings of half a step against the sum of the absolute
terms: a term passes N products, a sum per token, and its decay (three roundings
of an exponent L, L e^-L of them, with the chunks' products within 2^-18). y of
bfloat16 inputs passes one bfloat16 copy on the way and one at its end; the state
is float32 in every kernel: its update takes x' = d exp(..) x in full."""

from __future__ import annotations

import pytest
import torch

import mlx_lean_moe_amd as gdn
from . import plans
from .scan64 import scan64

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
U = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}
# float16 values below 2^-14 lie 2^-24 apart: rounding takes up to half of that,
# whatever the value (the other types' least steps are far below 1e-30)
LEAST = {"bf16": 1e-30, "f16": 2.0 ** -25, "f32": 1e-30}
E = 2.0 ** -24


def _case(gpu, act, lens, dims, seed):
    """x, B and C side by side in one row, as the conv leaves them."""
    H, P, G, N = dims
    g = torch.Generator(device=gpu)
    g.manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=gpu)
    T = sum(lens)
    x, B, C = r(T, H * P + 2 * G * N).to(DT[act]).split([H * P, G * N, G * N], dim=1)
    return dict(x=x.view(T, H, P), dt=r(T, H).to(DT[act]), B=B.view(T, G, N), C=C.view(T, G, N),
                A_log=torch.linspace(-1.0, 2.7, H, device=gpu), dt_bias=r(H) * 1.5 - 2.0, D=r(H), state=r(len(lens), H, P, N))


def _offsets(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


def _within(got, ref, tol, what):
    worst = ((got.double() - ref).abs() / tol).nan_to_num(nan=float("inf")).max().item()
    assert worst <= 1, f"{what}: worst ratio {worst:.3g}"


def _name(case):
    bf16, lens, dims, plan = case
    return "-".join(["bf16" if bf16 else "f32", f"{len(lens)}x{max(lens)}", "x".join(map(str, dims)), "x".join(map(str, plan))])


@pytest.mark.parametrize("bf16,lens,dims,plan", plans.SCAN_LAYOUTS, ids=map(_name, plans.SCAN_LAYOUTS))
def test_layouts(gpu, bf16, lens, dims, plan):
    case = _case(gpu, "bf16" if bf16 else "f32", lens, dims, 60)
    runs = gdn.PackedRuns(_offsets(lens), gpu)
    ref, state, ya, sa = scan64(**case, lens=lens)
    e = (max(lens) + dims[3] + 128) * E + 2.0 ** -18
    # float16 values are float32 ones too: the same kernel, with either output
    for act in ("bf16",) if bf16 else ("f32", "f16"):
        if act == "f16":
            case = {k: v.half() if k in ("x", "dt", "B", "C") else v for k, v in case.items()}
            ref, state, ya, sa = scan64(**case, lens=lens)
        y, S = gdn.selective_scan(**case, cu_seqlens=runs)
        u = U[act]
        _within(y, ref, u * ref.abs() + ((u * 1.01 if bf16 else 0) + e) * ya + LEAST[act], "y")
        _within(S, state, e * sa + 1e-30, "state")
        for r, n in enumerate(lens):
            if n == 0:
                assert torch.equal(S[r], case["state"][r])
        again = dict(case, state=case["state"].clone())
        y2, S2 = gdn.selective_scan(**again, cu_seqlens=runs, state_out=again["state"])
        assert torch.equal(y, y2) and torch.equal(S, S2)


@pytest.mark.parametrize("bf16,lens,dims,plan", [c for c in plans.SCAN_LAYOUTS if c[3][1] == 8 and max(c[1]) > 600][::2],
                         ids=map(_name, [c for c in plans.SCAN_LAYOUTS if c[3][1] == 8 and max(c[1]) > 600][::2]))
def test_values_that_are_not_finite_in_wide_layouts(gpu, bf16, lens, dims, plan):
    case = _case(gpu, "bf16" if bf16 else "f32", lens, dims, 61)
    runs = gdn.PackedRuns(_offsets(lens), gpu)
    H, P = dims[:2]
    y0, S0 = gdn.selective_scan(**case, cu_seqlens=runs)
    long = max(range(len(lens)), key=lambda r: lens[r])
    first, end = runs.offsets[long], runs.offsets[long + 1]
    for n, t in enumerate((first, first + 45, first + 63, first + 130, first + 511, end - 1)):
        h, p = (7 * n + 1) % H, (29 * n + 3) % P
        x = case["x"].clone()
        x[t, h, p] = float("nan") if n % 2 else float("inf")
        y, S = gdn.selective_scan(**dict(case, x=x), cu_seqlens=runs)
        assert not torch.isfinite(y[t:end, h, p]).any() and not torch.isfinite(S[long, h, p]).any(), (t, h, p)
        y[t:end, h, p], S[long, h, p] = y0[t:end, h, p], S0[long, h, p]
        assert torch.equal(y, y0) and torch.equal(S, S0), (t, h, p)


@pytest.mark.parametrize("act", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dims", [(64, 64, 8, 128), (3, 40, 1, 16), (32, 128, 2, 256)])
def test_the_state_holds_x_in_full(gpu, act, dims):
    """One token of each of many runs, from no state: S = d x B^T. d carries the
    roundings of its argument (|v| < 8 of them) and some 8 of softplus, x' two, each
    of three pieces' products with B and their sums at most six more, the update's
    decays two: under 32 E of the value. x' cut to two bfloat16 pieces, 16 bits,
    is off by up to 2^-15, and the bound has to tell: 2^-17 is 4 times it."""
    H, P, G, N = dims
    case = _case(gpu, act, [1] * 40, dims, 62)
    case.update(state=None, dt=case["dt"].clamp(-2, 2), dt_bias=case["dt_bias"].clamp(-5, 2))
    _, S = gdn.selective_scan(**case, cu_seqlens=list(range(41)))
    _, state, _, sa = scan64(**case, lens=[1] * 40)
    _within(S, state, 32 * E * sa + 1e-30, "state")
    # the check itself: two pieces in the float64 result fall outside
    v = (case["dt"].double() + case["dt_bias"].double())
    step = v.clamp(min=0) + torch.log1p(torch.exp(-v.abs()))
    xs = (case["x"].double() * step[..., None]).float()
    one = (xs.view(torch.int32) & -65536).view(torch.float32)
    two = ((xs - one).view(torch.int32) & -65536).view(torch.float32)
    cut = (one.double() + two.double())[..., None] * case["B"].double().repeat_interleave(H // G, 1)[:, :, None]
    assert ((cut - state).abs() / (32 * E * sa + 1e-30)).max() > 4
