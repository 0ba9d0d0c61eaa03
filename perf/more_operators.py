"""The norm in front of a layer and low-rank adapters beside its projections as
timed cases: ``rms_norm`` with the residual's addition, the same with its output
in e4m3 codes under a scale for each 128 columns, and ``add_low_rank``, the
adapters of many requests at once added to a shared projection's output.

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
GROUP = 128
E4M3_MAX = 448.0
EPS = 1e-6
ACT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------


def listed() -> list[dict]:
    return [
        # one token's norm at the layer's hidden size, the stream updated on the way
        dict(name="norm_1", kind="norm", rows=1, width=2048, act="bf16", residual=True, codes=False),
        # a prompt's
        dict(name="norm_4096", kind="norm", rows=4096, width=2048, act="bf16", residual=True, codes=False),
        # float32 activations, an odd prompt and a width of no round size
        dict(name="norm_1531_f32", kind="norm", rows=1531, width=2501, act="f32", residual=False, codes=False),
        # a decode batch in front of e4m3 weights
        dict(name="norm_codes_64_f16", kind="norm", rows=64, width=4096, act="f16", residual=False, codes=True),
        # prompts in front of e4m3 weights
        dict(name="norm_codes_8192", kind="norm", rows=8192, width=2048, act="bf16", residual=True, codes=True),
        # one request's token: its adapter beside the stacked input projection (qkv, z)
        dict(name="adapters_1", kind="adapters", rows=1, runs=1, hidden=2048, out=8192, more=4096, count=8, least=16,
             most=16, without=0.0, act="bf16"),
        # a decode batch in which every request has one of 32 adapters
        dict(name="adapters_64_of_32", kind="adapters", rows=64, runs=64, hidden=2048, out=8192, more=4096, count=32,
             least=16, most=16, without=0.0, act="bf16"),
        # a large decode batch over the output projection, ranks of several sizes, some requests without an adapter
        dict(name="adapters_200_f16", kind="adapters", rows=200, runs=200, hidden=4096, out=2048, more=0, count=12,
             least=4, most=64, without=0.2, act="f16"),
        # a few prompts in float32, odd widths
        dict(name="adapters_777_f32", kind="adapters", rows=777, runs=5, hidden=1024, out=1231, more=0, count=4, least=8,
             most=8, without=0.0, act="f32"),
        # prompts of many requests packed into one stream
        dict(name="adapters_4096_packed", kind="adapters", rows=4096, runs=16, hidden=2048, out=8192, more=4096, count=6,
             least=8, most=32, without=0.1, act="bf16"),
        # one long prompt with an adapter of a large rank
        dict(name="adapters_8192", kind="adapters", rows=8192, runs=1, hidden=2048, out=4096, more=0, count=3, least=64,
             most=64, without=0.0, act="bf16"),
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(("norm", "norm", "adapters", "adapters", "adapters"))
    act = rng.choice(("bf16", "bf16", "f32", "f16"))
    rows = _log_int(rng, 1, 8192)
    if kind == "norm":
        codes = rng.random() < 0.5
        width = rng.choice((2048, 4096, 128, 16 * _log_int(rng, 1, 1024), _log_int(rng, 1, 16384)))
        if codes:
            width = max(16, width // 16 * 16)
        return dict(kind=kind, rows=max(1, min(rows, 8192 * 2048 // width // (2 if act == "f32" else 1))), width=width,
                    act=act, residual=rng.random() < 0.6, codes=codes)
    hidden = rng.choice((2048, 4096, 1024, 8 * _log_int(rng, 8, 512), _log_int(rng, 40, 3000)))
    out = rng.choice((8192, 4096, 2048, 64, _log_int(rng, 1, 6000)))
    more = rng.choice((0, 0, 4096, 64, _log_int(rng, 1, 4000)))
    most = rng.choice((8, 16, 16, 32, 64, _log_int(rng, 1, 100)))
    least = rng.choice((most, most, max(1, most // 4)))
    # no more bytes than the largest listed case's
    rows = max(1, min(rows, 4096 * (2 * 12288 + 2048) // (2 * (out + more) + hidden) // (2 if act == "f32" else 1)))
    return dict(kind=kind, rows=rows, runs=rng.choice((1, rows, _log_int(rng, 1, rows))), hidden=hidden, out=out, more=more,
                count=_log_int(rng, 1, 32), least=least, most=most, without=rng.choice((0.0, 0.0, 0.3)), act=act)


def _adapter_plan(case: dict) -> tuple[list[int], list[int]]:
    """Each adapter's rank, and each row's adapter (-1: none): the requests'
    lengths and adapters, from the case alone."""
    rng = random.Random(case["rows"] * 1009 + case["count"] * 31 + case["runs"])
    ranks = [_log_int(rng, case["least"], case["most"]) for _ in range(case["count"])]
    ranks[0] = case["most"]
    cuts = sorted(rng.sample(range(1, case["rows"]), case["runs"] - 1)) if case["runs"] > 1 else []
    ends = cuts + [case["rows"]]
    index, begin = [], 0
    for i, end in enumerate(ends):
        a = rng.randrange(case["count"]) if i else 0
        if i and rng.random() < case["without"]:
            a = -1
        index += [a] * (end - begin)
        begin = end
    return ranks, index


def _widths(case: dict) -> list[int]:
    return [case["out"]] + ([case["more"]] if case["more"] else [])


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


def prepare(case: dict, seed: int) -> dict:
    m = _Maker(seed)
    act = ACT[case["act"]]
    s = dict(case=case)
    if case["kind"] == "norm":
        M, K = case["rows"], case["width"]
        # a residual stream: rows of different size, some large channels
        x = m.normal(M, K) * torch.exp(m.normal(M, 1, scale=0.5)) * (1 + 20 * (m.uniform(K) < 0.01))
        s.update(x=x.to(act), residual=m.normal(M, K, dtype=act) if case["residual"] else None,
                 weight=m.uniform(K, lo=0.5, hi=1.5))
        return s
    M, K = case["rows"], case["hidden"]
    ranks, index = _adapter_plan(case)
    s["x"] = m.normal(M, K, dtype=act)
    s["y"] = [m.normal(M, N, dtype=act) for N in _widths(case)]
    # each projection's adapters: (A, B, scale), the scale the usual 2 rank / rank
    s["adapters"] = [[(m.normal(r, K, scale=K ** -0.5, dtype=act), m.normal(N, r, scale=0.1 * r ** -0.5, dtype=act), 2.0)
                      for r in ranks] for N in _widths(case)]
    if own:
        import mlx_lean_moe_amd as gdn

        s["laid_out"] = gdn.LowRankAdapters(s["adapters"])
        s["rows"] = gdn.AdapterRows(index, len(ranks), device=DEV)
    else:
        s["index"] = torch.tensor(index, device=DEV)
        # every adapter's rows of A side by side, B's columns likewise, and whose each is
        s["A"] = [torch.cat([a for a, _, _ in block]) for block in s["adapters"]]
        s["B"] = [torch.cat([b for _, b, _ in block], dim=1) for block in s["adapters"]]
        s["whose"] = torch.tensor([a for a, r in enumerate(ranks) for _ in range(r)], device=DEV)
        s["scale"] = torch.tensor([c for (_, _, c), r in zip(s["adapters"][0], ranks) for _ in range(r)], device=DEV)
    return s


# ---------------------------------------------------------------------------
# the operators from elementary operations
# ---------------------------------------------------------------------------


def _norm(x, residual, weight, codes):
    """The norm in 32 bits; in 64 where codes are made of it, since on which
    side of a border of e4m3 a value falls must not depend on the order of a sum."""
    stream = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    v = stream.double() if codes else stream.float()
    v = v / torch.sqrt((v * v).mean(dim=-1, keepdim=True) + EPS) * weight.to(v.dtype)
    y = v.to(x.dtype)
    out = [] if residual is None else [stream]
    if not codes:
        return [y] + out
    M, K = x.shape
    groups = -(-K // GROUP)
    rows = torch.zeros(M, groups * GROUP, device=x.device)
    rows[:, :K] = y.float()
    rows = rows.reshape(M, groups, GROUP)
    # a tensor to divide by: torch multiplies by the reciprocal of a number
    scale = rows.abs().amax(dim=-1, keepdim=True) / torch.full((1,), E4M3_MAX, device=x.device)
    scale = scale.clamp(min=2.0 ** -126)
    code = (rows / scale).to(torch.float8_e4m3fn).reshape(M, groups * GROUP)[:, :K]
    return [code, scale.reshape(M, groups)] + out


def _adapt(s):
    """Every adapter's factors times every row, those of other adapters masked."""
    x = s["x"].float()
    mask = torch.where(s["index"][:, None] == s["whose"], s["scale"], 0.0)
    for y, A, B in zip(s["y"], s["A"], s["B"]):
        low = (x @ A.float().T) * mask
        y.copy_((y.float() + low @ B.float().T).to(y.dtype))
    return s["y"]


def run(s: dict):
    c = s["case"]
    if own:
        import mlx_lean_moe_amd as gdn

        if c["kind"] == "adapters":
            return gdn.add_low_rank(s["y"], s["x"], s["laid_out"], s["rows"])
        got = gdn.rms_norm(s["x"], s["weight"], EPS, residual=s["residual"], quantize=c["codes"])
        normed, stream = got if c["residual"] else (got, None)
        out = [] if stream is None else [stream]
        return ([normed.codes, normed.scales] if c["codes"] else [normed]) + out
    if c["kind"] == "adapters":
        return _adapt(s)
    return _norm(s["x"], s["residual"], s["weight"], c["codes"])


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------


def work(case: dict) -> dict:
    es = ACT[case["act"]].itemsize
    if case["kind"] == "norm":
        M, K = case["rows"], case["width"]
        read = M * K * es * (1 + case["residual"]) + K * 4
        out = M * K + M * -(-K // GROUP) * 4 if case["codes"] else M * K * es
        return {"bytes": read + out + M * K * es * case["residual"], "flops": 4 * M * K}
    ranks, index = _adapter_plan(case)
    K, N = case["hidden"], sum(_widths(case))
    blocks = len(_widths(case))
    rows = sum(a >= 0 for a in index)
    used = sum(ranks[a] for a in set(index) if a >= 0)
    return {"bytes": rows * (K + 2 * N) * es + used * (blocks * K + N) * es + 4 * len(index),
            "flops": 2 * sum(ranks[a] for a in index if a >= 0) * (blocks * K + N)}


# ---------------------------------------------------------------------------
# float64
# ---------------------------------------------------------------------------


def _e4m3(r):
    """The nearest e4m3 value (ties to the even code) of finite float64 values within its range."""
    e = torch.floor(torch.log2(r.abs().clamp(min=2.0 ** -6)))
    unit = torch.exp2(e - 3)
    return (torch.round(r / unit) * unit).clamp(-E4M3_MAX, E4M3_MAX)


def _exact_norm(s):
    """What the operator holds in fewer bits by definition (the stream, the
    row that is put in codes, scales and quotients) is rounded here as well."""
    c = s["case"]
    stream = s["x"].double()
    if c["residual"]:
        stream = (stream + s["residual"].double()).to(s["x"].dtype).double()
    power = torch.linalg.vector_norm(stream, dim=1) ** 2 / c["width"]
    y = stream * torch.rsqrt(power + EPS)[:, None] * s["weight"].double()
    out = [stream] if c["residual"] else []
    if not c["codes"]:
        return [y] + out
    y = y.to(s["x"].dtype).double()
    codes, scales = torch.empty_like(y), []
    for at in range(0, c["width"], GROUP):
        part = y[:, at:at + GROUP]
        scale = (part.abs().amax(dim=1) / 448).float().double().clamp(min=2.0 ** -126)
        codes[:, at:at + GROUP] = _e4m3((part / scale[:, None]).float().double())
        scales.append(scale)
    return [codes, torch.stack(scales, dim=1)] + out


def _exact_adapters(s):
    """Adapter by adapter, the rows that have it."""
    _, index = _adapter_plan(s["case"])
    outs = [y.double() for y in s["y"]]
    for a in sorted(set(index) - {-1}):
        rows = torch.tensor([i for i, v in enumerate(index) if v == a], device=DEV)
        x = s["x"][rows].double()
        for y, block in zip(outs, s["adapters"]):
            A, B, scale = block[a]
            y[rows] += scale * ((x @ A.double().T.contiguous()) @ B.double().T.contiguous())
    return outs


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    return _exact_norm(s) if case["kind"] == "norm" else _exact_adapters(s)
