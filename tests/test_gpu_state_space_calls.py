"""Calls that the documentation allows beside the usual ones: very many runs,
operands of mixed types, row strides of every operand, two captured graphs at
once. Tolerances as in test_gpu_state_space.py."""

from __future__ import annotations

import pytest
import torch

import mlx_lean_moe_amd as gdn
from .scan64 import scan64

pytestmark = pytest.mark.gpu

E = 2.0 ** -24


def _rng(gpu, seed):
    g = torch.Generator(device=gpu)
    g.manual_seed(seed)
    return lambda *s: torch.randn(*s, generator=g, device=gpu)


def _within(got, ref, tol, what):
    worst = ((got.double() - ref).abs() / tol).nan_to_num(nan=float("inf")).max().item()
    assert worst <= 1, f"{what}: worst ratio {worst:.3g}"


def _offsets(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


@pytest.mark.parametrize("act", [torch.bfloat16, torch.float32])
def test_more_runs_than_a_grid_dimension(gpu, act):
    """70 000 runs, most of one token, some empty, two of hundreds: whole and (with
    few heads and a long run) in segments, each from its own state."""
    r = _rng(gpu, 0)
    H, P, G, N = 2, 8, 1, 8
    lens = [1] * 70000
    lens[5], lens[69990] = 300, 500
    for i in range(100, 70000, 97):
        lens[i] = 0
    T, R = sum(lens), len(lens)
    case = dict(x=r(T, H, P).to(act), dt=r(T, H).to(act), B=r(T, G, N).to(act), C=r(T, G, N).to(act), A_log=r(H),
                dt_bias=r(H) - 1, D=r(H), state=r(R, H, P, N))
    runs = gdn.PackedRuns(_offsets(lens), gpu)
    y, S = gdn.selective_scan(**case, cu_seqlens=runs)
    u = 2.0 ** -8 if act == torch.bfloat16 else E
    e = (512 + 128) * E + 2.0 ** -18
    at = 0
    for lo, hi in ((0, 40), (33000, 33200), (65500, 65600), (69950, 70000)):
        some = lens[lo:hi]
        a, z = runs.offsets[lo], runs.offsets[hi]
        sub = {k: v[a:z] if k in ("x", "dt", "B", "C") else v[lo:hi] if k == "state" else v for k, v in case.items()}
        ref, state, ya, sa = scan64(**sub, lens=some)
        _within(y[a:z], ref, u * ref.abs() + ((u * 1.01 if act == torch.bfloat16 else 0) + e) * ya + 1e-30, f"y {lo}")
        _within(S[lo:hi], state, e * sa + 1e-30, f"state {lo}")
    empty = torch.tensor([i for i, n in enumerate(lens) if n == 0], device=gpu)
    assert torch.equal(S[empty], case["state"][empty]) and torch.isfinite(y).all()
    # the conv over the same runs: a run's own state before its first token
    x, st, w = r(T, 24).to(act), r(R, 3, 24).to(act), r(24, 4)
    out, new = gdn.conv_silu(x, st, w, None, runs)
    for lo, hi in ((0, 40), (65500, 65600), (69950, 70000)):
        a, z = runs.offsets[lo], runs.offsets[hi]
        o2, n2 = gdn.conv_silu(x[a:z], st[lo:hi], w, None, [c - a for c in runs.offsets[lo:hi + 1]])
        assert torch.equal(out[a:z], o2) and torch.equal(new[lo:hi], n2)


@pytest.mark.parametrize("act", [torch.bfloat16, torch.float16, torch.float32])
def test_operands_of_mixed_types(gpu, act):
    """dt, the parameters and the state in types of their own: dt is read as it is,
    the others as float32, as if handed over so."""
    r = _rng(gpu, 1)
    H, P, G, N, T = 4, 64, 2, 128, 200
    x, B, C = r(T, H, P).to(act), r(T, G, N).to(act), r(T, G, N).to(act)
    half = lambda t: t.half()
    b16 = lambda t: t.bfloat16()
    A_log, dt_bias, D, state = r(H), r(H) - 2, r(H), r(1, H, P, N)
    for dt in (r(T, H), b16(r(T, H)), half(r(T, H))):
        got = gdn.selective_scan(x, dt, B, C, b16(A_log), half(dt_bias), b16(D), half(state), cu_seqlens=[0, T])
        want = gdn.selective_scan(x, dt.float(), B, C, b16(A_log).float(), half(dt_bias).float(), b16(D).float(),
                                  half(state).float(), cu_seqlens=[0, T])
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    # x, B and C of different types meet in their promotion
    got = gdn.selective_scan(b16(x), dt, B.float(), C, A_log, dt_bias, D, state, cu_seqlens=[0, T], y_dtype=torch.float32)
    want = gdn.selective_scan(b16(x).float(), dt, B.float(), C.float(), A_log, dt_bias, D, state, cu_seqlens=[0, T])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = gdn.selective_scan(b16(x), dt, B.float(), C, A_log, dt_bias, D, state, cu_seqlens=[0, T])
    assert torch.equal(got[0], b16(want[0])) and torch.equal(got[1], want[1])
    u = gdn.conv_silu(x.flatten(1), half(r(1, 3, H * P)), b16(r(H * P, 4)), half(r(H * P)))[0]
    assert u.dtype == act and torch.isfinite(u).all()


def test_rows_at_strides(gpu):
    """Steps over column slices, every other row and reversed slots give the bits
    of packed operands."""
    r = _rng(gpu, 2)
    d = gdn.StateSpaceDims(2, 6, 64, 40, 4)
    B = 7
    wide = r(2 * B, d.conv_dim + d.num_heads + 5).bfloat16()
    xbc, dt = wide[::2, 3:3 + d.conv_dim], wide[::2, 3 + d.conv_dim:3 + d.conv_dim + d.num_heads]
    conv, ssm = r(B, 3, d.conv_dim).bfloat16(), r(B, d.num_heads, d.head_dim, d.state_dim)
    w, bias, A_log, dt_bias, D = r(d.conv_dim, 4), r(d.conv_dim), r(d.num_heads), r(d.num_heads), r(d.num_heads)
    want = gdn.selective_step(xbc.contiguous(), dt.contiguous(), conv, ssm, w, bias, A_log, dt_bias, D, d)
    got = gdn.selective_step(xbc, dt, conv.transpose(1, 2).contiguous().transpose(1, 2), ssm, w.T.contiguous().T,
                             torch.stack([bias, bias], 1)[:, 0], A_log, dt_bias, D, d)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    back = torch.arange(B - 1, -1, -1, dtype=torch.int32, device=gpu)
    pool_conv, pool_ssm = conv.flip(0).contiguous(), ssm.flip(0).contiguous()
    y, new, _ = gdn.selective_step(xbc, dt, pool_conv, pool_ssm, w, bias, A_log, dt_bias, D, d, slots=back)
    assert torch.equal(y, want[0]) and torch.equal(new, want[1]) and torch.equal(pool_ssm.flip(0), want[2])


def test_two_graphs_of_segmented_scans_replayed_at_once(gpu):
    """Each graph has its own workspace: replays on two streams at a time, with eager
    calls of the same scan between, hold their bits."""
    r = _rng(gpu, 3)
    H, P, G, N = 32, 64, 2, 128
    runs = gdn.PackedRuns([0, 2000, 2003, 3003], gpu)
    T = runs.tokens
    cases = []
    for _ in range(2):
        u = r(T, H * P + 2 * G * N).bfloat16()
        x, B, C = u.split([H * P, G * N, G * N], dim=1)
        cases.append(dict(x=x.view(T, H, P), dt=r(T, H).bfloat16(), B=B.view(T, G, N), C=C.view(T, G, N), A_log=r(H),
                          dt_bias=r(H) - 2, D=r(H), state=r(3, H, P, N)))
    call = lambda c: gdn.selective_scan(**c, cu_seqlens=runs)
    want = [call(c) for c in cases]
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in cases], []
    for g, c in zip(graphs, cases):
        with torch.cuda.graph(g):
            outs.append(call(c))
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(4):
        for o in outs:
            o[0].zero_(), o[1].zero_()
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        again = call(cases[0])
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o[0], w[0]) and torch.equal(o[1], w[1])
        assert torch.equal(again[0], want[0][0])


@pytest.mark.parametrize("act", [torch.bfloat16, torch.float16])
def test_a_stack_in_pieces_is_one_prompt(gpu, act):
    """A long prompt in chunks of uneven lengths, each from the state that the one
    before left, against float64 over the whole."""
    r = _rng(gpu, 4)
    H, P, G, N, T = 16, 64, 1, 128, 1500
    case = dict(x=r(T, H, P).to(act), dt=r(T, H).to(act), B=r(T, G, N).to(act), C=r(T, G, N).to(act),
                A_log=torch.linspace(-1, 2, H, device=gpu), dt_bias=r(H) - 2, D=r(H))
    ref, state, ya, sa = scan64(**case, state=None, lens=[T])
    S, ys = None, []
    for a, z in ((0, 1), (1, 64), (64, 65), (65, 700), (700, 700), (700, 1499), (1499, 1500)):
        y, S = gdn.selective_scan(**{k: v[a:z] if k in ("x", "dt", "B", "C") else v for k, v in case.items()}, state=S,
                                  cu_seqlens=[0, z - a])
        ys.append(y)
    u = 2.0 ** -8 if act == torch.bfloat16 else 2.0 ** -11
    e = (T + N + 128) * E + 2.0 ** -18
    # (float16 values below 2^-14 lie 2^-24 apart)
    _within(torch.cat(ys), ref, u * ref.abs() + ((u * 1.01 if act == torch.bfloat16 else 0) + e) * ya + 2.0 ** -25, "y")
    _within(S, state, e * sa + 1e-30, "state")
