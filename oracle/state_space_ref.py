"""NumPy float64 restatement of the state-space operators and of the
block-scaled 8-bit product, straight from their definitions (test
infrastructure only). ``conv_silu``, ``scan`` and ``fp8_block_matmul`` also return
what the same sums give with every term's absolute value: the yardstick of
rounding errors."""

from __future__ import annotations

import numpy as np


def silu(x):
    x = np.asarray(x, np.float64)
    with np.errstate(over="ignore"):
        return x / (1.0 + np.exp(-x))


def softplus(x):
    return np.maximum(x, 0.0) + np.log1p(np.exp(-np.abs(x)))


def conv_silu(x, conv_state, weight, bias, lens):
    """Rows ``x (T, C)`` of runs of ``lens`` tokens -> (out, new state, sum of
    |terms|, the argument of SiLU)."""
    x, st, w = (np.asarray(v, np.float64) for v in (x, conv_state, weight))
    b = np.zeros(x.shape[1]) if bias is None else np.asarray(bias, np.float64)
    K = w.shape[1]
    us, mags, states, at = [], [], [], 0
    for i, n in enumerate(lens):
        rows = np.concatenate([st[i], x[at:at + n]])
        us.append(b + sum(rows[j:j + n] * w[:, j] for j in range(K)))
        mags.append(np.abs(b) + sum(np.abs(rows[j:j + n] * w[:, j]) for j in range(K)))
        states.append(rows[n:])
        at += n
    u = np.concatenate(us)
    return silu(u), np.stack(states), np.concatenate(mags), u


def scan(x, dt, B, C, A_log, dt_bias, D, state, lens):
    """``x (T, H, P), dt (T, H), B, C (T, G, N)``, runs of ``lens`` tokens ->
    (y, state, y of the absolute values, state of the absolute values)."""
    x, dt, B, C, A_log, dt_bias = (np.asarray(v, np.float64) for v in (x, dt, B, C, A_log, dt_bias))
    T, H, P = x.shape
    G, N = B.shape[1:]
    R = len(lens)
    S0 = np.zeros((R, H, P, N)) if state is None else np.asarray(state, np.float64)
    skip = np.zeros(H) if D is None else np.asarray(D, np.float64)
    step = softplus(dt + dt_bias)
    decay = np.exp(-np.exp(A_log) * step)
    Bh, Ch = np.repeat(B, H // G, axis=1), np.repeat(C, H // G, axis=1)
    y, ya = np.zeros((T, H, P)), np.zeros((T, H, P))
    out, outa, t = np.zeros((R, H, P, N)), np.zeros((R, H, P, N)), 0
    for r, n in enumerate(lens):
        S, Sa = S0[r].copy(), np.abs(S0[r])
        for _ in range(n):
            add = (step[t][:, None] * x[t])[..., None] * Bh[t][:, None]
            S = decay[t][:, None, None] * S + add
            Sa = decay[t][:, None, None] * Sa + np.abs(add)
            y[t] = (S * Ch[t][:, None]).sum(-1) + skip[:, None] * x[t]
            ya[t] = (Sa * np.abs(Ch[t])[:, None]).sum(-1) + np.abs(skip[:, None] * x[t])
            t += 1
        out[r], outa[r] = S, Sa
    return y, out, ya, outa


def e4m3(r):
    """The nearest e4m3 value, ties to even, of finite values up to 464."""
    r = np.asarray(r, np.float64)
    unit = 2.0 ** (np.floor(np.log2(np.maximum(np.abs(r), 2.0 ** -6))) - 3)
    return np.clip(np.round(r / unit) * unit, -448.0, 448.0)


def quantize_rows(x):
    """(values of the codes, scales): float32 scale and quotient by
    definition. ``x (M, K)``, groups of 128 columns, the last maybe short."""
    x = np.asarray(x, np.float32)
    M, K = x.shape
    kb = -(-K // 128)
    q, s = np.zeros((M, K)), np.zeros((M, kb), np.float32)
    for b in range(kb):
        part = x[:, b * 128:(b + 1) * 128]
        s[:, b] = np.maximum(np.abs(part).max(axis=1) / np.float32(448), np.float32(2.0 ** -126))
        q[:, b * 128:(b + 1) * 128] = e4m3(part / s[:, b:b + 1])
    return q, s


def fp8_block_matmul(x, codes, scales):
    """``codes`` the values of the weight's codes (N, K), ``scales`` (N / 128,
    K / 128) -> (y, sum of |terms|)."""
    q, s = quantize_rows(x)
    K, N = q.shape[1], codes.shape[0]
    xd = q * np.repeat(s.astype(np.float64), 128, axis=1)[:, :K]
    wd = np.asarray(codes, np.float64) * np.repeat(np.repeat(np.asarray(scales, np.float64), 128, 0)[:N], 128, 1)[:, :K]
    return xd @ wd.T, np.abs(xd) @ np.abs(wd).T
