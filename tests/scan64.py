"""The selective scan token by token in float64, in torch on any device: what
`oracle.state_space_ref.scan` computes, for prompts that NumPy takes too long
for. Returns the same sums of absolute values as yardsticks too."""

from __future__ import annotations

import torch


def scan64(x, dt, B, C, A_log, dt_bias, D, state, lens):
    """``x (T, H, P), dt (T, H), B, C (T, G, N)``, runs of ``lens`` tokens ->
    (y, state, y of the absolute values, state of the absolute values)."""
    T, H, P = x.shape
    G, N = B.shape[1:]
    R, f64 = len(lens), dict(dtype=torch.float64, device=x.device)
    x, dt, B, C = x.double(), dt.double(), B.double(), C.double()
    v = dt + dt_bias.double()
    step = torch.clamp(v, min=0) + torch.log1p(torch.exp(-v.abs()))
    decay = torch.exp(-torch.exp(A_log.double()) * step)
    first = [sum(lens[:r]) for r in range(R)]
    order = sorted(range(R), key=lambda r: -lens[r])
    at0 = torch.tensor([first[r] for r in order], device=x.device)
    S = torch.zeros(R, H, P, N, **f64) if state is None else state.double()[order].clone()
    Sa = S.abs()
    y, ya = torch.zeros(T, H, P, **f64), torch.zeros(T, H, P, **f64)
    for t in range(max(lens, default=0)):
        n = sum(k > t for k in lens)
        at = at0[:n] + t
        Bt, Ct = B[at].repeat_interleave(H // G, 1), C[at].repeat_interleave(H // G, 1)
        add = (x[at] * step[at][..., None])[..., None] * Bt[:, :, None]
        g = decay[at][..., None, None]
        S[:n] = S[:n] * g + add
        Sa[:n] = Sa[:n] * g + add.abs()
        y[at] = (S[:n] * Ct[:, :, None]).sum(-1)
        ya[at] = (Sa[:n] * Ct[:, :, None].abs()).sum(-1)
    if D is not None:
        y += D.double()[:, None] * x
        ya += (D.double()[:, None] * x).abs()
    back = torch.empty_like(S), torch.empty_like(S)
    back[0][order], back[1][order] = S, Sa
    return y, back[0], ya, back[1]
