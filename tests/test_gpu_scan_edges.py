"""The selective scan where single tokens differ widely from their neighbours:
steps that forget everything, and values that are not finite.

Tolerances as in test_gpu_state_space.py, but for the state of bfloat16 inputs:
its update takes x' = d exp(..) x in three bfloat16 pieces, all 24 bits of it, so
its bound is the float32 one."""

from __future__ import annotations

import pytest
import torch

import mlx_lean_moe_amd as gdn
from mlx_lean_moe_amd import _lib
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


@pytest.mark.parametrize("act,y_act", [("bf16", "bf16"), ("f32", "f32"), ("f16", "f16"), ("bf16", "f32")])
@pytest.mark.parametrize("lens,dims", [([100, 0, 41], (4, 64, 2, 128)), ([300], (3, 40, 1, 64)), ([130, 64], (2, 128, 2, 256)),
                                       ([20, 90], (32, 96, 1, 16))])
def test_values_that_are_not_finite_reach_no_earlier_token(gpu, act, y_act, lens, dims):
    """One bad value of x at a time: the tokens before it, the other heads and the
    other rows of its head hold the bits that they hold without it; its own row of
    y and of the state, from its token to the end of its run, holds what the
    recurrence gives, no number."""
    H, P, G, N = dims
    case = _case(gpu, act, lens, dims, 50)
    cu = _offsets(lens)
    call = lambda **k: gdn.selective_scan(**dict(case, **k), cu_seqlens=cu, y_dtype=DT[y_act])
    y0, S0 = call()
    assert torch.isfinite(y0).all() and torch.isfinite(S0).all()
    for n, t in enumerate((0, 7, 15, 16, 31, 32, 33, 47, 62, 63, 64, 77, 95, 99)):
        run = max(r for r in range(len(lens)) if cu[r] <= t)
        end = cu[run + 1]
        h, p = (5 * n + 1) % H, (13 * n + 2) % P
        x = case["x"].clone()
        x[t, h, p] = (float("nan"), float("inf"), float("-inf"))[n % 3]
        y, S = call(x=x)
        assert not torch.isfinite(y[t:end, h, p]).any() and not torch.isfinite(S[run, h, p]).any(), (t, h, p)
        y[t:end, h, p], S[run, h, p] = y0[t:end, h, p], S0[run, h, p]
        assert torch.equal(y, y0) and torch.equal(S, S0), (t, h, p)


@pytest.mark.parametrize("act", ["bf16", "f32"])
def test_gates_and_states_that_are_not_finite_reach_no_earlier_token(gpu, act):
    """The same of dt, B and C: a step spoils its head, a row of B its group's
    heads, both from their token on, a row of C its group's heads at its token."""
    lens, (H, P, G, N) = [150, 30], (4, 64, 2, 128)
    case = _case(gpu, act, lens, (H, P, G, N), 51)
    call = lambda **k: gdn.selective_scan(**dict(case, **k), cu_seqlens=[0, 150, 180])
    y0, S0 = call()
    for t in (0, 9, 16, 40, 63, 64, 100, 149):
        for name in ("dt", "B", "C"):
            v = case[name].clone()
            v[(t, 2) if name == "dt" else (t, 1, t % N)] = float("nan")
            heads = slice(2, 3) if name == "dt" else slice(2, 4)
            y, S = call(**{name: v})
            at = slice(t, t + 1) if name == "C" else slice(t, 150)
            assert torch.isnan(y[at, heads]).all(), (name, t)
            y[at, heads] = y0[at, heads]
            if name != "C":
                assert torch.isnan(S[0, heads]).any()
                S[0, heads] = S0[0, heads]
            assert torch.equal(y, y0) and torch.equal(S, S0), (name, t)


@pytest.mark.parametrize("act", ["bf16", "f32"])
def test_whole_tokens_that_are_not_finite(gpu, act):
    """Every value of a token bad, and later tokens bad again (padding that was
    never written): what stands before them is as without them."""
    lens, dims = [170], (4, 64, 2, 128)
    case = _case(gpu, act, lens, dims, 52)
    for end in (1, 20, 64, 101):
        alone = {k: v[:end] if k in ("x", "dt", "B", "C") else v for k, v in case.items()}
        bad = dict(case)
        for k in ("x", "B", "C"):
            bad[k] = case[k].clone()
            bad[k][end:] = float("nan")
        y, _ = gdn.selective_scan(**bad, cu_seqlens=[0, 170])
        ref, _, ya, _ = scan64(**alone, lens=[end])
        u = U[act]
        e = (170 + 128 + 128) * 2.0 ** -24 + 2.0 ** -18
        _within(y[:end], ref, u * ref.abs() + ((u * 1.01 if act == "bf16" else 0) + e) * ya + 2.0 ** -48, "y")
        assert torch.isnan(y[end:]).all()


@pytest.mark.parametrize("act", ["bf16", "f32"])
@pytest.mark.parametrize("lens,tail", [([40, 0, 9], 30), ([700, 64, 1], 200), ([3, 1500], 1)])
def test_rows_behind_the_last_run_stay_at_the_c_boundary(gpu, act, lens, tail):
    """The offsets may end before the arrays, and the longest run may be given,
    left out or given too short: rows behind the last run are neither read nor
    written, and how the call is cut changes the sums' order only."""
    H, P, G, N = dims = (4, 64, 2, 128)
    case = _case(gpu, act, lens, dims, 70)
    ref, state, ya, sa = scan64(**case, lens=lens)
    end, T, R = sum(lens), sum(lens) + tail, len(lens)
    bad = lambda t: torch.cat([t, torch.full((tail, *t.shape[1:]), float("nan"), device=gpu, dtype=t.dtype)])
    x, dt, B, C = (bad(case[k]) for k in ("x", "dt", "B", "C"))
    cu = torch.tensor(_offsets(lens), dtype=torch.int32, device=gpu)
    code, lib = _lib.dtype_code(DT[act]), _lib.load()
    e, u = (T + 128 + 128) * 2.0 ** -24 + 2.0 ** -18, U[act]
    for longest in (max(lens), 0, 1, 65):
        y = torch.full((T, H, P), 7.0, device=gpu, dtype=DT[act])
        S = torch.empty(R, H, P, N, device=gpu)
        size = lib.gdn_selective_scan_workspace_size(code, code, R, T, longest, G, H, P, N)
        ws = torch.empty(max(size, 1), dtype=torch.uint8, device=gpu)
        _lib.call_on(gpu, "gdn_selective_scan", x.data_ptr(), H * P, B.data_ptr(), G * N, C.data_ptr(), G * N, code,
                     dt.data_ptr(), H, code, case["A_log"].data_ptr(), case["dt_bias"].data_ptr(), case["D"].data_ptr(),
                     case["state"].data_ptr(), S.data_ptr(), y.data_ptr(), code, cu.data_ptr(), R, T, longest, G, H, P, N,
                     ws.data_ptr(), size, _lib.stream_ptr(gpu))
        assert (y[end:] == 7).all()
        _within(y[:end], ref, u * ref.abs() + ((u * 1.01 if act == "bf16" else 0) + e) * ya + 1e-30, "y")
        _within(S, state, e * sa + 1e-30, "state")
