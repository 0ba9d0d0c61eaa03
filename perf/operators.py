"""The state-space operators and the block-scaled 8-bit projections as timed
cases: the conv with SiLU over prompts, the selective scan over prompts, one
token for a batch of sequences, and ``quantized_linear`` on e4m3 weights with
a scale for each block of 128 x 128.

``listed()`` holds the cases, ``draw()`` gives further ones of the same
ranges; ``prepare`` / ``run`` make and run one, ``work`` is what a pass
cannot do without, and ``exact`` gives the outputs in float64. ``run``
computes the operators from elementary torch operations, or, with ``own``
set, through the package's entry points.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
CONV_K = 4
CHUNK = 64
BLOCK = 128
E4M3_MAX = 448.0
ACT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------


def listed() -> list[dict]:
    return [
        # the conv over one long prompt: 64 heads of 64, 8 groups of 128 states
        dict(name="conv_4096", kind="conv", runs=1, shortest=4096, longest=4096, lens_seed=0, channels=6144,
             act="bf16", bias=True),
        # the conv over packed prompts, float32, a channel count of no round size
        dict(name="conv_packed_7_f32", kind="conv", runs=7, shortest=1, longest=611, lens_seed=2, channels=2180,
             act="f32", bias=False),
        # a draft being verified, a short prompt's tail
        dict(name="scan_41", kind="scan", runs=1, shortest=41, longest=41, lens_seed=0, heads=32, head_dim=64,
             groups=1, state_dim=128, act="bf16", state=True, skip=True),
        # one long prompt from an empty state
        dict(name="scan_4096", kind="scan", runs=1, shortest=4096, longest=4096, lens_seed=0, heads=64, head_dim=64,
             groups=8, state_dim=128, act="bf16", state=False, skip=True),
        # a batch of prompts of mixed length packed into one stream, each
        # continuing from a state, one of them empty
        dict(name="scan_packed_16", kind="scan", runs=16, shortest=0, longest=4096, lens_seed=3, heads=64, head_dim=64,
             groups=1, state_dim=128, act="bf16", state=True, skip=True),
        # a prompt of an odd length in float32 at the gated-delta layer's heads
        dict(name="scan_f32_1531", kind="scan", runs=1, shortest=1531, longest=1531, lens_seed=0, heads=32,
             head_dim=128, groups=16, state_dim=128, act="f32", state=True, skip=False),
        # one sequence's token
        dict(name="step_1", kind="step", batch=1, pool=4, heads=64, head_dim=64, groups=8, state_dim=128, act="bf16"),
        # a serving step over part of a pool, float32, sequences at scattered slots
        dict(name="step_48_of_100_f32", kind="step", batch=48, pool=100, heads=32, head_dim=128, groups=16,
             state_dim=128, act="f32"),
        # the largest decode batch: 0.5 GB of state
        dict(name="step_256", kind="step", batch=256, pool=256, heads=64, head_dim=64, groups=1, state_dim=128,
             act="bf16"),
        # one sequence's input projection
        dict(name="linear_1", kind="linear", rows=1, out=12352, hidden=2048, act="bf16", residual=False),
        # the output projection of a decode batch or a short prompt, with the layer's residual
        dict(name="linear_200", kind="linear", rows=200, out=2048, hidden=4096, act="bf16", residual=True),
        # a prompt's input projection
        dict(name="linear_4096", kind="linear", rows=4096, out=12352, hidden=2048, act="bf16", residual=False),
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(("conv", "scan", "scan", "step", "linear", "linear"))
    act = rng.choice(("bf16", "bf16", "f32", "f16"))
    if kind in ("conv", "scan"):
        runs = rng.choice((1, 1, _log_int(rng, 2, 24)))
        longest = max(1, min(_log_int(rng, 1, 6000), 16384 // runs))
        shortest = longest if runs == 1 else rng.choice((longest, 0, 1, max(1, longest // rng.randint(2, 16))))
        case = dict(kind=kind, runs=runs, shortest=shortest, longest=longest, lens_seed=rng.randrange(1000))
        if kind == "conv":
            case.update(channels=rng.choice((6144, 4352, 8192, 2 * _log_int(rng, 64, 3000), _log_int(rng, 100, 3000))),
                        act=act, bias=rng.random() < 0.5)
        else:
            heads, groups = rng.choice(((64, 8), (64, 1), (32, 16), (24, 1), (24, 2), (9, 3), (5, 5), (80, 8)))
            case.update(heads=heads, groups=groups, head_dim=rng.choice((64, 64, 128, 96, 40)),
                        state_dim=rng.choice((128, 128, 64, 256, 16)), act=act, state=rng.random() < 0.7,
                        skip=rng.random() < 0.7)
            if case["head_dim"] * case["state_dim"] > 8192:  # no more state than the largest listed case
                case.update(heads=min(heads, 32) // groups * groups)
        return case
    if kind == "step":
        batch = _log_int(rng, 1, 256)
        heads, groups = rng.choice(((64, 8), (64, 1), (32, 16), (32, 4), (24, 2)))
        head_dim, state_dim = rng.choice(((64, 128), (64, 128), (128, 128), (64, 64), (64, 256), (48, 16)))
        if head_dim * state_dim * heads > 64 * 64 * 128:
            batch = min(batch, 100)
        return dict(kind=kind, batch=batch, pool=batch + rng.choice((0, 1, _log_int(rng, 1, 100))), heads=heads,
                    groups=groups, head_dim=head_dim, state_dim=state_dim, act=act)
    hidden = rng.choice((1024, 2048, 2048, 4096, 16 * _log_int(rng, 4, 200)))
    out = rng.choice((12352, 8192, 2048, 64, _log_int(rng, 1, 6000)))
    return dict(kind=kind, rows=_log_int(rng, 1, 2048 if hidden * out > 12352 * 2048 else 4096), out=out, hidden=hidden,
                act=act, residual=rng.random() < 0.3)


def _lengths(case: dict) -> list[int]:
    """The runs' lengths: spread over [shortest, longest], one at each end,
    in an order of their own."""
    runs, lo, hi = case["runs"], case["shortest"], case["longest"]
    if lo == hi:
        return [hi] * runs
    rng = random.Random(case["lens_seed"])
    lens = [lo, hi] + [min(hi, max(lo, round(math.exp(rng.uniform(math.log(max(1, lo)), math.log(hi))))))
                       for _ in range(runs - 2)]
    rng.shuffle(lens)
    return lens


def _offsets(lens) -> list[int]:
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


class _Maker:
    def __init__(self, seed: int):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(1_000_003 * (seed + 1))

    def normal(self, *shape, scale=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=self.g, device=DEV) * scale).to(dtype)

    def uniform(self, *shape, lo=0.0, hi=1.0):
        return torch.rand(*shape, generator=self.g, device=DEV) * (hi - lo) + lo


def _gate_params(m: _Maker, heads: int):
    """Decay rates of 1 to 16 and steps of 0.001 to 0.1 before the input's
    share, log-uniform, the usual start of such layers."""
    A_log = torch.log(m.uniform(heads, lo=1.0, hi=16.0))
    step = torch.exp(m.uniform(heads, lo=math.log(1e-3), hi=math.log(1e-1)))
    return A_log, torch.log(torch.expm1(step))


def prepare(case: dict, seed: int) -> dict:
    m = _Maker(seed)
    s = dict(case=case)
    if case["kind"] in ("conv", "scan"):
        lens = _lengths(case)
        s["offsets"] = _offsets(lens)
        s["cu"] = torch.tensor(s["offsets"], dtype=torch.int32, device=DEV)
        s["longest"] = max(lens)
    if case["kind"] == "conv":
        act, C, T, R = ACT[case["act"]], case["channels"], s["offsets"][-1], case["runs"]
        s.update(x=m.normal(T, C, dtype=act), conv_state=m.normal(R, CONV_K - 1, C, dtype=act),
                 weight=m.normal(C, CONV_K, scale=0.3), bias=m.normal(C, scale=0.1) if case["bias"] else None)
    elif case["kind"] == "scan":
        act, T, R = ACT[case["act"]], s["offsets"][-1], case["runs"]
        H, P, G, N = case["heads"], case["head_dim"], case["groups"], case["state_dim"]
        # what the conv hands over: x, B and C side by side in one row
        u = m.normal(T, H * P + 2 * G * N)
        u = (u * torch.sigmoid(u)).to(act)
        A_log, dt_bias = _gate_params(m, H)
        s.update(u=u, dt=m.normal(T, H, dtype=act), A_log=A_log, dt_bias=dt_bias,
                 D=m.uniform(H, lo=0.5, hi=1.5) if case["skip"] else None,
                 state=m.normal(R, H, P, N, scale=0.1) if case["state"] else None)
    elif case["kind"] == "step":
        act, B, pool = ACT[case["act"]], case["batch"], case["pool"]
        H, P, G, N = case["heads"], case["head_dim"], case["groups"], case["state_dim"]
        C = H * P + 2 * G * N
        A_log, dt_bias = _gate_params(m, H)
        slots = torch.randperm(pool, generator=torch.Generator().manual_seed(seed))[:B]
        s.update(u=m.normal(B, C, dtype=act), dt=m.normal(B, H, dtype=act), A_log=A_log, dt_bias=dt_bias,
                 D=m.uniform(H, lo=0.5, hi=1.5), weight=m.normal(C, CONV_K, scale=0.3), bias=m.normal(C, scale=0.1),
                 conv=m.normal(2 * pool, CONV_K - 1, C, dtype=act), ssm=m.normal(pool, H, P, N, scale=0.1),
                 slots=slots.to(DEV, torch.int32), half=(m.uniform(pool) < 0.5).to(torch.int32),
                 arrivals=torch.zeros(pool, dtype=torch.int32, device=DEV))
    else:
        act, M, N, K = ACT[case["act"]], case["rows"], case["out"], case["hidden"]
        nb, kb = -(-N // BLOCK), -(-K // BLOCK)
        w = torch.zeros(nb * BLOCK, kb * BLOCK, device=DEV)
        w[:N, :K] = m.normal(N, K, scale=K ** -0.5)
        blocks = w.reshape(nb, BLOCK, kb, BLOCK)
        scales = blocks.abs().amax(dim=(1, 3)) / E4M3_MAX
        codes = (blocks / scales[:, None, :, None]).reshape(nb * BLOCK, kb * BLOCK)[:N, :K]
        # activations of a residual stream: rows of different size, some large channels
        x = m.normal(M, K) * torch.exp(m.normal(M, 1, scale=0.5)) * (1 + 20 * (m.uniform(K) < 0.01))
        s.update(x=x.to(act), weight=codes.contiguous().to(torch.float8_e4m3fn), scales=scales,
                 residual=m.normal(M, N, dtype=act) if case["residual"] else None)
    if own:
        import mlx_lean_moe_amd as gdn

        if case["kind"] in ("conv", "scan"):
            s["runs"] = gdn.PackedRuns(s["offsets"], device=DEV)
        elif case["kind"] == "step":
            s["dims"] = gdn.StateSpaceDims(case["groups"], case["heads"], case["state_dim"], case["head_dim"], CONV_K)
        else:
            s["weights"] = gdn.LinearWeights({"weight": s["weight"], "scales": s["scales"]},
                                             gdn.QuantScheme(8, BLOCK, "fp8_block"))
    return s


# ---------------------------------------------------------------------------
# the operators from elementary operations, 32 bits
# ---------------------------------------------------------------------------


def _conv(x, conv_state, weight, bias, cu):
    """Taps t-3 .. t of each token, those before its run from the run's
    state; the new state is the last rows of state and run together."""
    T, C = x.shape
    K1 = conv_state.shape[1]
    token = torch.arange(T, device=x.device)
    run = torch.searchsorted(cu.long(), token, right=True) - 1
    back = torch.arange(-K1, 1, device=x.device)
    at = (token - cu[run])[:, None] + back  # place of each tap in its run
    rows = torch.cat([conv_state.flatten(0, 1), x])
    base = conv_state.shape[0] * K1
    src = torch.where(at < 0, run[:, None] * K1 + K1 + at, base + token[:, None] + back)
    u = (rows[src].float() * weight.T).sum(dim=1)
    if bias is not None:
        u = u + bias
    lens = (cu[1:] - cu[:-1]).long()
    at = lens[:, None] + torch.arange(-K1, 0, device=x.device)
    src = torch.where(at < 0, torch.arange(len(lens), device=x.device)[:, None] * K1 + K1 + at,
                      base + cu[:-1].long()[:, None] + at)
    return (u * torch.sigmoid(u)).to(x.dtype), rows[src]


def _softplus(x):
    return torch.clamp(x, min=0) + torch.log1p(torch.exp(-torch.abs(x)))


def _scan(u, dt, A_log, dt_bias, D, state, cu, longest, heads, head_dim, groups, state_dim):
    """The scan chunk by chunk: within a chunk the pairs of tokens with the
    decay between them, across chunks the states with the decay between
    theirs."""
    H, P, G, N, R, T = heads, head_dim, groups, state_dim, len(cu) - 1, u.shape[0]
    chunks = max(1, -(-longest // CHUNK))
    place = torch.arange(chunks * CHUNK, device=u.device)
    lens = (cu[1:] - cu[:-1]).long()
    valid = place < lens[:, None]
    rows = (cu[:-1].long()[:, None] + place).clamp(max=max(T - 1, 0))
    tok = torch.where(valid[..., None], u[rows].float(), 0.0).reshape(R, chunks, CHUNK, -1)
    x = tok[..., :H * P].reshape(R, chunks, CHUNK, H, P).permute(0, 3, 1, 2, 4)
    B, C = (t.reshape(R, chunks, CHUNK, G, N).permute(0, 3, 1, 2, 4).repeat_interleave(H // G, dim=1)
            for t in (tok[..., H * P:H * P + G * N], tok[..., H * P + G * N:]))
    step = torch.where(valid[..., None], _softplus(dt[rows].float() + dt_bias), 0.0)
    step = step.reshape(R, chunks, CHUNK, H).permute(0, 3, 1, 2)
    # sums of decays in 64 bits: their differences are what counts
    total = torch.cumsum(-torch.exp(A_log.double())[:, None, None] * step.double(), dim=-1)
    end = torch.cumsum(total[..., -1], dim=-1)
    begin = end - total[..., -1]
    order = torch.arange(CHUNK, device=u.device)
    decay = (total[..., :, None] - total[..., None, :]).masked_fill(order[:, None] < order, -math.inf)
    pairs = (C.contiguous() @ B.transpose(-1, -2).contiguous()) * torch.exp(decay).float() * step[..., None, :]
    y = pairs @ x.contiguous()
    left = torch.exp(total[..., -1:] - total).float() * step
    states = (x * left[..., None]).transpose(-1, -2).contiguous() @ B.contiguous()
    order = torch.arange(chunks, device=u.device)
    across = (begin[..., :, None] - end[..., None, :]).masked_fill(order[:, None] <= order, -math.inf)
    before = (torch.exp(across).float() @ states.flatten(-2)).reshape(states.shape)
    if state is not None:
        before = before + torch.exp(begin).float()[..., None, None] * state[:, :, None]
    y = y + torch.exp(total).float()[..., None] * (C.contiguous() @ before.transpose(-1, -2).contiguous())
    last = before[:, :, -1] * torch.exp(total[:, :, -1, -1]).float()[..., None, None] + states[:, :, -1]
    if D is not None:
        y = y + D[:, None, None, None] * x
    y = y.permute(0, 2, 3, 1, 4).reshape(R, chunks * CHUNK, H, P)[valid]
    return y.to(u.dtype), last


def _step(s):
    c = s["case"]
    H, P, G, N, pool = c["heads"], c["head_dim"], c["groups"], c["state_dim"], c["pool"]
    slots = s["slots"].long()
    half = (s["half"][slots] ^ (s["arrivals"][slots] >> 16)) & 1
    window = torch.cat([s["conv"][slots + pool * half], s["u"][:, None]], dim=1)
    u = (window.float() * s["weight"].T).sum(dim=1) + s["bias"]
    u = u * torch.sigmoid(u)
    x = u[:, :H * P].reshape(-1, H, P)
    B, C = (t.reshape(-1, G, N).repeat_interleave(H // G, dim=1) for t in (u[:, H * P:H * P + G * N], u[:, H * P + G * N:]))
    step = _softplus(s["dt"].float() + s["dt_bias"])
    ssm = (s["ssm"][slots] * torch.exp(-torch.exp(s["A_log"]) * step)[..., None, None]
           + (step[..., None] * x)[..., None] * B[:, :, None])
    y = (ssm * C[:, :, None]).sum(dim=-1) + s["D"][:, None] * x
    s["ssm"][slots] = ssm
    s["conv"][slots + pool * (1 - half)] = window[:, 1:]
    s["arrivals"][slots] += 1 << 16
    return y.to(s["u"].dtype), s["ssm"], s["conv"], s["arrivals"]


def _linear(x, weight, scales, residual):
    """Each row's groups of 128 in e4m3 under their own scale, then the
    product of the values that both sides' codes stand for. With a residual
    the layer adds two arrays of one type: the product is one of them."""
    M, K = x.shape
    N = weight.shape[0]
    nb, kb = scales.shape
    rows = torch.zeros(M, kb * BLOCK, device=x.device)
    rows[:, :K] = x.float()
    rows = rows.reshape(M, kb, BLOCK)
    # a tensor to divide by: torch multiplies by the reciprocal of a number
    own_scale = rows.abs().amax(dim=-1, keepdim=True) / torch.full((1,), E4M3_MAX, device=x.device)
    own_scale = own_scale.clamp(min=2.0 ** -126)
    rows = ((rows / own_scale).to(torch.float8_e4m3fn).float() * own_scale).reshape(M, kb * BLOCK)[:, :K]
    w = weight.float() * scales.repeat_interleave(BLOCK, 0)[:N].repeat_interleave(BLOCK, 1)[:, :K]
    y = rows.contiguous() @ w.T
    return y.to(x.dtype) if residual is None else (y.to(x.dtype).float() + residual.float()).to(x.dtype)


def run(s: dict):
    c = s["case"]
    if own:
        import mlx_lean_moe_amd as gdn

        if c["kind"] == "conv":
            return gdn.conv_silu(s["x"], s["conv_state"], s["weight"], s["bias"], s["runs"])
        if c["kind"] == "scan":
            H, P, G, N, T = c["heads"], c["head_dim"], c["groups"], c["state_dim"], s["u"].shape[0]
            x, B, C = torch.split(s["u"], [H * P, G * N, G * N], dim=-1)
            return gdn.selective_scan(x.view(T, H, P), s["dt"], B.view(T, G, N), C.view(T, G, N), s["A_log"],
                                      s["dt_bias"], s["D"], s["state"], cu_seqlens=s["runs"])
        if c["kind"] == "step":
            y, conv, ssm = gdn.selective_step(
                s["u"], s["dt"], s["conv"], s["ssm"], s["weight"], s["bias"], s["A_log"], s["dt_bias"], s["D"],
                s["dims"], state_out=s["ssm"], slots=s["slots"], conv_half=s["half"], conv_arrivals=s["arrivals"])
            return y, ssm, conv, s["arrivals"]
        return gdn.quantized_linear(s["x"], s["weights"], residual=s["residual"])
    if c["kind"] == "conv":
        return _conv(s["x"], s["conv_state"], s["weight"], s["bias"], s["cu"])
    if c["kind"] == "scan":
        return _scan(s["u"], s["dt"], s["A_log"], s["dt_bias"], s["D"], s["state"], s["cu"], s["longest"], c["heads"],
                     c["head_dim"], c["groups"], c["state_dim"])
    if c["kind"] == "step":
        return _step(s)
    return _linear(s["x"], s["weight"], s["scales"], s["residual"])


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------


def work(case: dict) -> dict:
    es = ACT[case["act"]].itemsize
    if case["kind"] == "conv":
        T, C, R = sum(_lengths(case)), case["channels"], case["runs"]
        return {"bytes": 2 * T * C * es + 2 * R * (CONV_K - 1) * C * es + C * (CONV_K + case["bias"]) * 4,
                "flops": T * C * (2 * CONV_K + 4)}
    if case["kind"] == "linear":
        M, N, K = case["rows"], case["out"], case["hidden"]
        scales = -(-N // BLOCK) * -(-K // BLOCK) * 4
        return {"bytes": M * K * es + N * K + scales + M * N * es * (1 + case["residual"]), "flops": 2 * M * N * K}
    H, P, G, N = case["heads"], case["head_dim"], case["groups"], case["state_dim"]
    if case["kind"] == "scan":
        T, R = sum(_lengths(case)), case["runs"]
        return {"bytes": T * (2 * H * P + 2 * G * N + H) * es + R * H * P * N * 4 * (1 + case["state"]),
                "flops": 5 * T * H * P * N}
    B, C = case["batch"], H * P + 2 * G * N
    return {"bytes": 2 * B * H * P * N * 4 + B * es * (C + H + 2 * (CONV_K - 1) * C + H * P) + C * (CONV_K + 1) * 4,
            "flops": B * H * P * N * 5}


# ---------------------------------------------------------------------------
# float64
# ---------------------------------------------------------------------------


def _runs_apart(cu: list[int]):
    return [(i, a, b) for i, (a, b) in enumerate(zip(cu, cu[1:]))]


def _exact_conv(s):
    x, st = s["x"].double(), s["conv_state"].double()
    w = s["weight"].double()
    outs, states = [], []
    for i, a, b in _runs_apart(s["offsets"]):
        rows = torch.cat([st[i], x[a:b]])
        n = b - a
        u = sum(rows[j:j + n] * w[:, j] for j in range(CONV_K))
        if s["bias"] is not None:
            u = u + s["bias"].double()
        outs.append(u / (1 + torch.exp(-u)))
        states.append(rows[n:])
    return torch.cat(outs), torch.stack(states)


def _exact_scan(s):
    """Token by token, all runs side by side."""
    c = s["case"]
    H, P, G, N, R = c["heads"], c["head_dim"], c["groups"], c["state_dim"], c["runs"]
    u, T = s["u"].double(), s["u"].shape[0]
    step = torch.nn.functional.softplus(s["dt"].double() + s["dt_bias"].double(), threshold=700.0)
    decay = torch.exp(-torch.exp(s["A_log"].double()) * step)
    state = s["state"].double().clone() if s["state"] is not None else torch.zeros(R, H, P, N, dtype=torch.float64, device=DEV)
    y = torch.empty(T, H, P, dtype=torch.float64, device=DEV)
    lens = [b - a for _, a, b in _runs_apart(s["offsets"])]
    by_length = sorted(range(R), key=lambda i: -lens[i])
    state = state[by_length]
    first = torch.tensor([s["offsets"][i] for i in by_length], device=DEV)
    for t in range(max(lens)):
        n = sum(length > t for length in lens)  # the runs still going, in front
        at = first[:n] + t
        x = u[at, :H * P].reshape(n, H, P)
        B = u[at, H * P:H * P + G * N].reshape(n, G, 1, 1, N)
        C = u[at, H * P + G * N:].reshape(n, G, 1, 1, N)
        S = state[:n]
        S *= decay[at][..., None, None]
        S.view(n, G, H // G, P, N).addcmul_((x * step[at][..., None]).reshape(n, G, H // G, P, 1), B)
        y[at] = (S.view(n, G, H // G, P, N) * C).sum(-1).reshape(n, H, P)
    if s["D"] is not None:
        y += s["D"].double()[:, None] * u[:, :H * P].reshape(T, H, P)
    last = torch.empty_like(state)
    last[by_length] = state
    return y, last


def _exact_step(s):
    c = s["case"]
    H, P, G, N, pool = c["heads"], c["head_dim"], c["groups"], c["state_dim"], c["pool"]
    conv, ssm, slots = s["conv"].double(), s["ssm"].double(), s["slots"].tolist()
    half = s["half"].tolist()
    w, b = s["weight"].double(), s["bias"].double()
    now = torch.tensor([v + pool * half[v] for v in slots], device=DEV)
    then = torch.tensor([v + pool * (1 - half[v]) for v in slots], device=DEV)
    at = torch.tensor(slots, device=DEV)
    old, new = conv[now], s["u"].double()
    u = old[:, 0] * w[:, 0] + old[:, 1] * w[:, 1] + old[:, 2] * w[:, 2] + new * w[:, 3] + b
    u = u / (1 + torch.exp(-u))
    conv[then] = torch.stack([old[:, 1], old[:, 2], new], dim=1)
    step = torch.nn.functional.softplus(s["dt"].double() + s["dt_bias"].double(), threshold=700.0)
    x = u[:, :H * P].reshape(-1, G, H // G, P)
    B = u[:, H * P:H * P + G * N].reshape(-1, G, 1, 1, N)
    C = u[:, H * P + G * N:].reshape(-1, G, 1, 1, N)
    S = (ssm[at] * torch.exp(-torch.exp(s["A_log"].double()) * step)[..., None, None]).reshape(-1, G, H // G, P, N)
    S = S + (x * step.reshape(-1, G, H // G, 1))[..., None] * B
    y = (S * C).sum(-1) + s["D"].double().reshape(G, H // G, 1) * x
    ssm[at] = S.reshape(-1, H, P, N)
    arrivals = s["arrivals"].clone()
    arrivals[at] += 65536
    return y.reshape(-1, H, P), ssm, conv, arrivals


def _e4m3(r):
    """The nearest e4m3 value (ties to the even code) of finite float64 values within its range."""
    e = torch.floor(torch.log2(r.abs().clamp(min=2.0 ** -6)))
    unit = torch.exp2(e - 3)
    return (torch.round(r / unit) * unit).clamp(-E4M3_MAX, E4M3_MAX)


def _exact_linear(s):
    """Scales and quotients are held in 32 bits by definition: both are
    rounded to float32 here as well. (The float64 quotient of two float32
    values rounds to the float32 value that one rounding gives.)"""
    x = s["x"].double()
    M, K = x.shape
    N = s["weight"].shape[0]
    codes = s["weight"].double()
    scales = s["scales"].double()
    y = torch.zeros(M, N, dtype=torch.float64, device=DEV)
    for b in range(-(-K // BLOCK)):
        part = x[:, b * BLOCK:(b + 1) * BLOCK]
        scale = (part.abs().amax(dim=1, keepdim=True) / 448).float().double().clamp(min=2.0 ** -126)
        q = _e4m3((part / scale).float().double()) * scale
        w = codes[:, b * BLOCK:(b + 1) * BLOCK] * scales[:, b].repeat_interleave(BLOCK)[:N, None]
        y += q @ w.T.contiguous()
    return y if s["residual"] is None else y + s["residual"].double()


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    return {"conv": _exact_conv, "scan": _exact_scan, "step": _exact_step, "linear": _exact_linear}[case["kind"]](s)
