"""GPU parity of the state-space operators with their float64 definitions.

Tolerances count roundings (half a step: ``u`` = 2^-8 for bfloat16, 2^-11 for
float16, 2^-24 for float32) against the sum of the absolute terms:

* conv: K + 1 float32 roundings of the sum (SiLU's slope is at most 1.1), SiLU
  itself within (8 + 4 |u|) roundings (its exponent's argument is rounded), one
  rounding to the output.
* scan in float32: a term passes N products and sums, a few roundings per token
  it decays over, and its decay, whose exponent L carries three roundings: L e^-L
  times that, under 2^-18 for the lengths and rates here.
* scan in bfloat16: a term enters y through one bfloat16 copy, of its decayed
  score or of the state it lies in, and y is rounded; the state takes x in two
  bfloat16 pieces (u^2).
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

import mlx_lean_moe_amd as gdn
from mlx_lean_moe_amd import _lib
from oracle import state_space_ref as R

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
U = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}
E = 2.0 ** -24


def _np(t):
    return t.detach().double().cpu().numpy()


def _close(got, ref, tol):
    got = _np(got)
    assert got.shape == ref.shape
    assert np.isfinite(got).all()
    bad = np.abs(got - ref) > tol
    assert not bad.any(), (f"{int(bad.sum())} of {bad.size} outside; worst ratio "
                           f"{(np.abs(got - ref) / np.maximum(tol, 1e-300)).max():.3g}")


def _rng(seed, gpu):
    g = torch.Generator(device=gpu)
    g.manual_seed(seed)
    return lambda *s, scale=1.0, dtype=torch.float32: (torch.randn(*s, generator=g, device=gpu) * scale).to(dtype)


# ---------------------------------------------------------------------------
# conv
# ---------------------------------------------------------------------------


def _conv_case(gpu, act, lens, C, K, bias, pad=0, seed=0):
    r = _rng(seed, gpu)
    T, N = sum(lens), len(lens)
    x = r(T, C + pad, scale=2.0, dtype=DT[act])[:, pad // 2:pad // 2 + C]
    return (x, r(N, K - 1, C, dtype=DT[act]), r(C, K, scale=0.5), r(C) if bias else None,
            np.concatenate([[0], np.cumsum(lens)]).tolist())


def _check_conv(out, new, x, st, w, b, lens, act):
    ref, state, mag, u = R.conv_silu(_np(x), _np(st), _np(w), None if b is None else _np(b), lens)
    tol = U[act] * np.abs(ref) + E * (1.1 * (w.shape[1] + 1) * mag + (8 + 4 * np.abs(u)) * np.abs(ref)) + 2.0 ** -24 * U[act]
    _close(out, ref, tol)
    assert np.array_equal(_np(new), state)


@pytest.mark.parametrize("act", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("lens,C,K", [([1], 8, 4), ([3], 64, 4), ([33, 0, 1, 2, 15, 16, 17], 24, 4),
                                      ([100, 5], 2176, 3), ([0, 0, 40], 10, 2), ([7, 90], 5, 4), ([0], 16, 4)])
def test_conv_silu(gpu, act, lens, C, K):
    x, st, w, b, cu = _conv_case(gpu, act, lens, C, K, bias=C != 24)
    out, new = gdn.conv_silu(x, st, w, b, cu)
    assert out.dtype == new.dtype == DT[act]
    _check_conv(out, new, x, st, w, b, lens, act)


@pytest.mark.parametrize("act", ["bf16", "f16"])
def test_conv_silu_of_many_tokens(gpu, act):
    lens = [2100, 1, 0, 90, 2205]
    x, st, w, b, cu = _conv_case(gpu, act, lens, 4104, 4, True, pad=8, seed=3)
    out, new = gdn.conv_silu(x, st, w, b, cu)
    _check_conv(out, new, x, st, w, b, lens, act)


@pytest.mark.parametrize("T,C", [(60, 24), (4600, 4096)])
def test_rows_behind_the_last_run_stay(gpu, T, C):
    """At the C boundary the offsets may end before the arrays: what lies behind
    the last run is neither read nor written."""
    lens = [T // 2, T // 4 + 3]
    end = sum(lens)
    x, st, w, b, cu = _conv_case(gpu, "bf16", lens, C, 4, True, seed=4)
    x = torch.cat([x, torch.full((T - end, C), float("nan"), device=gpu, dtype=x.dtype)])
    out, new = torch.full_like(x, 7.0), torch.empty_like(st)
    cu = torch.tensor(cu, dtype=torch.int32, device=gpu)
    _lib.call_on(x.device, "gdn_conv_silu", x.data_ptr(), C, st.data_ptr(), new.data_ptr(), w.data_ptr(), b.data_ptr(),
                 cu.data_ptr(), 2, T, out.data_ptr(), C, 4, _lib.dtype_code(x.dtype), _lib.stream_ptr(x.device))
    assert (out[end:] == 7).all()
    _check_conv(out[:end], new, x[:end], st, w, b, lens, "bf16")


@pytest.mark.parametrize("pad", [16, 6, 1])
def test_conv_silu_reads_strided_rows_and_equal_runs(gpu, pad):
    lens = [50, 50, 50]
    x, st, w, b, _ = _conv_case(gpu, "bf16", lens, 48, 4, True, pad=pad, seed=1)
    out, new = gdn.conv_silu(x, st, w[:, :, None], b)
    _check_conv(out, new, x, st, w, b, lens, "bf16")


def test_conv_silu_of_large_and_special_values(gpu):
    """Far arguments of SiLU, both signs, and non-finite ones: only the windows
    of four rows that hold them are touched, a tap of zero among them (0 times
    NaN or infinity is NaN)."""
    x = torch.zeros(12, 8, device=gpu)
    x[:, 0] = torch.tensor([-200., -100, -90, -88, -50, -20, 20, 100, 1e30, -1e30, 0, 0], device=gpu)
    x[5, 1], x[5, 2] = float("nan"), float("inf")
    w = torch.zeros(8, 4, device=gpu)
    w[:, 3] = 1.0
    w[1:3, 2] = 1.0
    for act in ("f32", "bf16"):
        xa = x.to(DT[act])
        out, _ = gdn.conv_silu(xa, torch.zeros(1, 3, 8, device=gpu, dtype=DT[act]), w)
        ref = R.silu(_np(xa)[:, 0])
        tol = U[act] * np.abs(ref) + E * (8 + 4 * np.abs(_np(xa)[:, 0])) * np.abs(ref) + 2.0 ** -126
        _close(out[:, 0], ref, tol)
        assert torch.isfinite(out[:5]).all() and torch.isfinite(out[9:]).all()
        assert torch.isnan(out[5:9, 1]).all() and torch.isfinite(out[5:9, 3:]).all()


def test_conv_silu_in_pieces_is_one_prompt(gpu):
    x, st, w, b, _ = _conv_case(gpu, "bf16", [70], 40, 4, True, seed=2)
    whole, end = gdn.conv_silu(x, st, w, b)
    parts, state = [], st
    for a, z in ((0, 1), (1, 3), (3, 3), (3, 64), (64, 70)):
        o, state = gdn.conv_silu(x[a:z], state, w, b, [0, z - a])
        parts.append(o)
    assert torch.equal(torch.cat(parts), whole) and torch.equal(state, end)


# ---------------------------------------------------------------------------
# scan
# ---------------------------------------------------------------------------


def _scan_case(gpu, act, lens, dims, state=True, skip=True, seed=0):
    H, P, G, N = dims
    r = _rng(seed, gpu)
    T = sum(lens)
    u = r(T, H * P + 2 * G * N, dtype=DT[act])  # x, B, C side by side, as the conv leaves them
    x, B, C = torch.split(u, [H * P, G * N, G * N], dim=1)
    A_log = torch.linspace(-1.0, 2.7, H, device=gpu)
    dt_bias = r(H, scale=1.5) - 2.0
    return dict(x=x.view(T, H, P), dt=r(T, H, dtype=DT[act]), B=B.view(T, G, N), C=C.view(T, G, N), A_log=A_log,
                dt_bias=dt_bias, D=r(H) if skip else None, state=r(len(lens), H, P, N) if state else None)


def _check_scan(got, case, lens, act, y_act):
    y, S = got
    ref, state, ya, sa = R.scan(**{k: None if v is None else _np(v) for k, v in case.items()}, lens=lens)
    N, T = case["B"].shape[-1], max(lens, default=0)
    e = (T + N + 128) * E + 2.0 ** -18
    if act == y_act == "bf16":
        _close(y, ref, U["bf16"] * np.abs(ref) + (U["bf16"] * 1.01 + e) * ya)
        _close(S, state, (2.0 ** -16 + e) * sa + 1e-30)
    else:
        _close(y, ref, U[y_act] * np.abs(ref) + e * ya + 2.0 ** -24 * U[y_act])
        _close(S, state, e * sa + 1e-30)


DIMS = [(2, 8, 1, 8), (4, 64, 2, 128), (3, 64, 3, 16), (4, 40, 2, 32), (2, 128, 1, 256), (6, 96, 3, 64), (4, 32, 1, 128),
        (8, 64, 1, 64), (1, 200, 1, 40)]


@pytest.mark.parametrize("act,y_act", [("bf16", "bf16"), ("f32", "f32"), ("f16", "f16"), ("bf16", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("dims", DIMS)
def test_scan_over_packed_runs(gpu, act, y_act, dims):
    lens = [0, 1, 63, 64, 0, 65, 130, 2, 0]
    case = _scan_case(gpu, act, lens, dims, seed=dims[0])
    cu = np.concatenate([[0], np.cumsum(lens)]).tolist()
    got = gdn.selective_scan(**case, cu_seqlens=cu, y_dtype=DT[y_act])
    assert got[0].dtype == DT[y_act] and got[1].dtype == torch.float32
    _check_scan(got, case, lens, act, y_act)
    for r, n in enumerate(lens):
        if n == 0:
            assert torch.equal(got[1][r], case["state"][r])


@pytest.mark.parametrize("act", ["bf16", "f32", "f16"])
@pytest.mark.parametrize("lens,dims", [([700], (2, 64, 1, 128)), ([257, 0, 1030, 3], (4, 32, 2, 64)),
                                       ([1500, 255, 256], (1, 128, 1, 16))])
def test_scan_of_long_runs_cut_into_segments(gpu, act, lens, dims):
    case = _scan_case(gpu, act, lens, dims, seed=3)
    runs = gdn.PackedRuns(np.concatenate([[0], np.cumsum(lens)]).tolist())
    _check_scan(gdn.selective_scan(**case, cu_seqlens=runs), case, lens, act, act)


@pytest.mark.parametrize("act", ["bf16", "f32"])
def test_scan_batch_first_without_state_or_skip(gpu, act):
    lens = [77, 77, 77]
    case = _scan_case(gpu, act, lens, (4, 64, 2, 128), state=False, skip=False, seed=4)
    batch = {k: v.reshape(3, 77, *v.shape[1:]) if k in ("x", "dt", "B", "C") else v for k, v in case.items()}
    y, S = gdn.selective_scan(**batch)
    assert y.shape == (3, 77, 4, 64)
    _check_scan((y.reshape(231, 4, 64), S), case, lens, act, act)


@pytest.mark.parametrize("act", ["bf16", "f32"])
@pytest.mark.parametrize("lens", [[300], [20, 500]])
def test_scan_updates_the_state_in_place(gpu, act, lens):
    case = _scan_case(gpu, act, lens, (4, 64, 2, 128), seed=5)
    cu = np.concatenate([[0], np.cumsum(lens)]).tolist()
    want = gdn.selective_scan(**case, cu_seqlens=cu)
    case["state"] = case["state"].clone()
    y, S = gdn.selective_scan(**case, cu_seqlens=cu, state_out=case["state"])
    assert S is case["state"] and torch.equal(S, want[1]) and torch.equal(y, want[0])


@pytest.mark.parametrize("act", ["bf16", "f32"])
def test_scan_decays_from_none_to_all(gpu, act):
    """Rates from e^-30 (nothing is forgotten) to e^9 (all of it, at once) and
    steps from 1e-9 to 80: no overflow on either side of the diagonal."""
    lens = [200]
    case = _scan_case(gpu, act, lens, (4, 64, 1, 128), seed=6)
    case["A_log"] = torch.tensor([-30.0, 9.0, 2.0, 0.0], device=gpu)
    case["dt_bias"] = torch.tensor([-1.0, 3.0, 80.0, -20.0], device=gpu)
    _check_scan(gdn.selective_scan(**case, cu_seqlens=[0, 200]), case, lens, act, act)


@pytest.mark.parametrize("act", ["bf16", "f32"])
def test_scan_keeps_other_runs_and_rows_out(gpu, act):
    """Neighbouring runs full of NaN and rows of y behind the last run: a run
    sees its own tokens only."""
    lens = [70, 30, 90]
    case = _scan_case(gpu, act, lens, (4, 64, 2, 128), seed=7)
    for k in ("x", "B", "C", "dt"):
        case[k] = case[k].clone()
        case[k][:70] = float("nan")
        case[k][100:] = float("inf")
    y, S = gdn.selective_scan(**case, cu_seqlens=[0, 70, 100, 190])
    alone = {k: v[70:100] if k in ("x", "dt", "B", "C") else v[1:2] if k == "state" else v for k, v in case.items()}
    _check_scan((y[70:100], S[1:2]), alone, [30], act, act)


def test_scan_inputs_that_no_kernel_reads_in_place(gpu):
    """Odd row strides and offsets, expanded B and C, a transposed x."""
    lens, (H, P, G, N) = [50, 37], (2, 24, 1, 40)
    case = _scan_case(gpu, "bf16", lens, (H, P, G, N), seed=8)
    wide = torch.empty(87, H * P + 3, dtype=torch.bfloat16, device=gpu)
    wide[:, 1:1 + H * P] = case["x"].reshape(87, -1)
    odd = dict(case, x=wide[:, 1:1 + H * P].unflatten(1, (H, P)), dt=case["dt"].T.contiguous().T,
               C=case["C"].permute(2, 1, 0).contiguous().permute(2, 1, 0))
    odd["state"] = torch.empty(2 * H * P * N + 1, device=gpu)[1:].view(2, H, P, N).copy_(case["state"])
    want = gdn.selective_scan(**case, cu_seqlens=[0, 50, 87])
    got = gdn.selective_scan(**odd, cu_seqlens=[0, 50, 87])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    case["B"] = case["B"][:1].expand(87, G, N)
    _check_scan(gdn.selective_scan(**case, cu_seqlens=[0, 50, 87]), case, lens, "bf16", "bf16")


def test_scan_of_rows_far_apart(gpu):
    """Rows further apart than the kernels address in place."""
    case = _scan_case(gpu, "bf16", [3], (2, 8, 1, 16), seed=9)
    far = torch.empty(3, (1 << 22) + 8, dtype=torch.bfloat16, device=gpu)
    far[:, :16] = case["x"].reshape(3, 16)
    want = gdn.selective_scan(**case, cu_seqlens=[0, 3])
    got = gdn.selective_scan(**dict(case, x=far[:, :16].unflatten(1, (2, 8))), cu_seqlens=[0, 3])
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_scan_of_no_tokens(gpu):
    case = _scan_case(gpu, "bf16", [0, 0], (2, 64, 1, 128), seed=9)
    y, S = gdn.selective_scan(**case, cu_seqlens=[0, 0, 0])
    assert y.shape == (0, 2, 64) and torch.equal(S, case["state"])
    case["state"] = None
    assert not gdn.selective_scan(**case, cu_seqlens=[0, 0, 0])[1].any()


# ---------------------------------------------------------------------------
# step
# ---------------------------------------------------------------------------


def _step_case(gpu, act, B, dims, K=4, seed=0, pool=None):
    H, P, G, N = dims
    r = _rng(seed, gpu)
    d = gdn.StateSpaceDims(G, H, N, P, K)
    C = d.conv_dim
    rows = B if pool is None else pool
    return d, dict(xbc=r(B, C, dtype=DT[act]), dt=r(B, H, dtype=DT[act]), conv_state=r(rows, K - 1, C, dtype=DT[act]),
                   ssm_state=r(rows, H, P, N), conv_weight=r(C, K, scale=0.5), conv_bias=r(C),
                   A_log=torch.linspace(-1.0, 2.7, H, device=gpu), dt_bias=r(H) - 1.0, D=r(H))


def _step_ref(d, c, conv, ssm):
    """(y, new conv, new ssm, tolerances' yardsticks) in float64."""
    B, H, P, G, N = c["xbc"].shape[0], d.num_heads, d.head_dim, d.num_groups, d.state_dim
    bias = None if c["conv_bias"] is None else _np(c["conv_bias"])
    u, new, mag, arg = R.conv_silu(_np(c["xbc"]), _np(conv), _np(c["conv_weight"]), bias, [1] * B)
    D = None if c["D"] is None else _np(c["D"])
    args = (u[:, :H * P].reshape(B, H, P), _np(c["dt"]), u[:, H * P:H * P + G * N].reshape(B, G, N),
            u[:, H * P + G * N:].reshape(B, G, N), _np(c["A_log"]), _np(c["dt_bias"]), D, _np(ssm), [1] * B)
    y, S, ya, sa = R.scan(*args)
    # what the conv's float32 errors (relative to |u|, at most du) amount to
    du = E * (1.1 * (d.conv_kernel_dim + 1) * mag + (8 + 4 * np.abs(arg)) * np.abs(u)) + 1e-30
    a = np.abs(u) + du
    big = R.scan(a[:, :H * P].reshape(B, H, P), args[1], a[:, H * P:H * P + G * N].reshape(B, G, N),
                 a[:, H * P + G * N:].reshape(B, G, N), args[4], args[5], None if D is None else np.abs(D),
                 np.abs(args[7]), [1] * B)
    return y, new, S, (big[0] - ya) + (N + 40) * E * ya, (big[1] - sa) + 40 * E * sa


def _check_step(got, d, c, conv, ssm, act):
    y, new, S, ty, ts = _step_ref(d, c, conv, ssm)
    _close(got[0], y, U[act] * np.abs(y) + ty + 2.0 ** -24 * U[act])
    _close(got[2], S, ts)
    assert np.array_equal(_np(got[1]), new)


@pytest.mark.parametrize("act", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("B,dims,K", [(1, (4, 64, 2, 128), 4), (3, (2, 8, 1, 8), 4), (5, (3, 17, 1, 16), 3),
                                      (2, (6, 96, 3, 64), 2), (2, (2, 256, 2, 256), 4), (40, (16, 40, 4, 24), 4),
                                      (1, (1, 129, 1, 128), 4), (130, (5, 64, 5, 32), 4)])
def test_step(gpu, act, B, dims, K):
    d, c = _step_case(gpu, act, B, dims, K)
    if B == 3:
        c["conv_bias"] = c["D"] = None
    conv, ssm = c["conv_state"].clone(), c["ssm_state"].clone()
    got = gdn.selective_step(**c, dims=d)
    _check_step(got, d, c, conv, ssm, act)
    assert torch.equal(c["conv_state"], conv) and torch.equal(c["ssm_state"], ssm)
    again = gdn.selective_step(**c, dims=d, state_out=c["ssm_state"])
    assert again[2] is c["ssm_state"] and all(torch.equal(a, b) for a, b in zip(again, got))


@pytest.mark.parametrize("heads", [3, 8, 24])
def test_step_over_a_pool(gpu, heads):
    """Steps at scattered slots roll each slot's conv state between its halves
    and leave the other slots alone, for any number of heads."""
    d = gdn.StateSpaceDims(1, heads, 128, 64, 4)
    pool = gdn.RecurrentStatePool(9, 4, d.conv_dim, heads, 64, 128, dtype=torch.bfloat16, device=gpu)
    _, c = _step_case(gpu, "bf16", 9, (heads, 64, 1, 128), seed=1)
    pool.conv_buf[:9], pool.ssm_state[:] = c["conv_state"], c["ssm_state"]
    for slots in ([7, 0, 4], [4, 7], [8, 7, 1, 0]):
        slot_t = pool.device_slots(slots)
        _, s = _step_case(gpu, "bf16", len(slots), (heads, 64, 1, 128), seed=10 + len(slots))
        s.update(conv_state=pool.conv_buf, ssm_state=pool.ssm_state)
        before = pool.conv_state, pool.ssm_state.clone()
        y, _, _ = gdn.selective_step(**s, dims=d, slots=slot_t, conv_half=pool.conv_half_dev,
                                     conv_arrivals=pool.conv_arrivals)
        pool.advance(slots, slot_t, device_flipped=True)
        assert torch.equal(pool.device_halves().cpu().long(), pool.conv_half)
        assert not bool((pool.conv_arrivals & 0xFFFF).any())
        conv, ssm = pool.conv_state, pool.ssm_state
        _check_step((y, conv[slots], ssm[slots]), d, s, before[0][slots], before[1][slots], "bf16")
        rest = [i for i in range(9) if i not in slots]
        assert torch.equal(conv[rest], before[0][rest]) and torch.equal(ssm[rest], before[1][rest])


def test_step_halves_without_counters(gpu):
    d, c = _step_case(gpu, "f32", 2, (4, 64, 2, 128), pool=5, seed=2)
    conv2 = torch.cat([c["conv_state"], torch.zeros_like(c["conv_state"])])
    slots = torch.tensor([3, 1], dtype=torch.int32, device=gpu)
    half = torch.zeros(5, dtype=torch.int32, device=gpu)
    ssm = c["ssm_state"].clone()
    c.update(conv_state=conv2)
    y, _, _ = gdn.selective_step(**c, dims=d, slots=slots, conv_half=half)
    _check_step((y, conv2[[8, 6]], c["ssm_state"][[3, 1]]), d, c, conv2[[3, 1]], ssm[[3, 1]], "f32")
    assert not half.any()


def test_step_refuses_slots_outside_the_pool(gpu):
    d, c = _step_case(gpu, "bf16", 4, (4, 64, 2, 128), pool=6, seed=3)
    conv2 = torch.cat([c["conv_state"]] * 2)
    c.update(conv_state=conv2)
    ssm, conv = c["ssm_state"].clone(), conv2.clone()
    slots = torch.tensor([2, 6, -1, 5], dtype=torch.int32, device=gpu)
    half, arr = (torch.zeros(6, dtype=torch.int32, device=gpu) for _ in range(2))
    y, _, _ = gdn.selective_step(**c, dims=d, slots=slots, conv_half=half, conv_arrivals=arr)
    assert torch.isnan(y[1:3]).all() and torch.isfinite(y[[0, 3]]).all()
    assert arr.tolist() == [0, 0, 65536, 0, 0, 65536]
    keep = [0, 1, 3, 4]
    assert torch.equal(c["ssm_state"][keep], ssm[keep]) and torch.equal(conv2[:6], conv[:6])
    assert torch.equal(conv2[[6, 7, 9, 10]], conv[[6, 7, 9, 10]])


def test_steps_continue_a_prompt(gpu):
    """A prompt and then single tokens give what one longer prompt gives."""
    d, c = _step_case(gpu, "f32", 1, (4, 64, 2, 128), seed=4)
    r = _rng(5, gpu)
    T, n = 150, 9
    rows, dt = r(T + n, d.conv_dim), r(T + n, 4)

    def prompt(a, b, conv, ssm):
        u, conv = gdn.conv_silu(rows[a:b], conv, c["conv_weight"], c["conv_bias"], [0, b - a])
        x, B, C = torch.split(u, [256, 256, 256], dim=1)
        y, ssm = gdn.selective_scan(x.view(-1, 4, 64), dt[a:b], B.view(-1, 2, 128), C.view(-1, 2, 128), c["A_log"],
                                    c["dt_bias"], c["D"], ssm, cu_seqlens=[0, b - a])
        return y, conv, ssm

    conv0, ssm0 = c["conv_state"], c["ssm_state"]
    whole, conv_end, ssm_end = prompt(0, T + n, conv0, ssm0)
    y, conv, ssm = prompt(0, T, conv0, ssm0)
    ys = [y]
    for t in range(T, T + n):
        args = dict(c, xbc=rows[t:t + 1], dt=dt[t:t + 1], conv_state=conv, ssm_state=ssm)
        y, conv, ssm = gdn.selective_step(**args, dims=d)
        ys.append(y)
    got = torch.cat(ys)
    assert torch.equal(conv, conv_end)
    # two float32 evaluations of sums of terms up to about 100 in all
    assert (got - whole).abs().max() < 2e-3 and (ssm - ssm_end).abs().max() < 1e-4
    assert ((got - whole).norm() / whole.norm()) < 1e-5


# ---------------------------------------------------------------------------
# streams and graphs
# ---------------------------------------------------------------------------


def test_calls_on_two_streams_at_once(gpu):
    cases = [_scan_case(gpu, "bf16", [700, 40], (8, 64, 1, 128), seed=20 + i) for i in range(2)]
    runs = gdn.PackedRuns([0, 700, 740])
    want = [gdn.selective_scan(**c, cu_seqlens=runs) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(5):
        for i, (s, c) in enumerate(zip(streams, cases)):
            with torch.cuda.stream(s):
                got[i].append(gdn.selective_scan(**c, cu_seqlens=runs))
    torch.cuda.synchronize()
    for i in range(2):
        for y, S in got[i]:
            assert torch.equal(y, want[i][0]) and torch.equal(S, want[i][1])


def test_prompt_and_step_replay_from_graphs(gpu):
    """Captured once, replayed with other inputs and eager calls between."""
    lens, dims = [300, 0, 41], (4, 64, 2, 128)
    d = gdn.StateSpaceDims(2, 4, 128, 64, 4)
    runs = gdn.PackedRuns([0, 300, 300, 341])
    conv = _conv_case(gpu, "bf16", lens, d.conv_dim, 4, True, seed=30)[:4]
    scan = _scan_case(gpu, "bf16", lens, dims, seed=31)
    _, step = _step_case(gpu, "bf16", 3, dims, seed=32)

    def prompt(x, state):
        u, new = gdn.conv_silu(x, *conv[1:], runs)
        xs, B, C = torch.split(u, [256, 256, 256], dim=1)
        y, S = gdn.selective_scan(**dict(scan, x=xs.view(-1, 4, 64), B=B.view(-1, 2, 128), C=C.view(-1, 2, 128),
                                         state=state), cu_seqlens=runs)
        z, cs, ss = gdn.selective_step(**dict(step, conv_state=new, ssm_state=S), dims=d)
        return u, new, y, S, z, cs, ss

    x, state = conv[0].contiguous().clone(), scan["state"].clone()
    prompt(x, state)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = prompt(x, state)
    r = _rng(33, gpu)
    for _ in range(4):
        x.copy_(r(341, d.conv_dim, dtype=torch.bfloat16))
        state.copy_(r(*state.shape))
        want = prompt(x, state)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
