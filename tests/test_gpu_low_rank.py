"""GPU parity of add_low_rank with the formula in float64.

The inner sum t = x A^T is float32: K products, each sum off by at most half a last
place, twice over for the matrix cores' own order. 16-bit adapters then take c t in two
pieces of their type. bfloat16: the upper 8 bits leave less than 2^-7 of the power of
two below c t, and rounding that to 8 bits is off by at most 2^-16 of it. float16: 11
bits and 11 of what they leave, 2^-22, where the row's largest of 16 lies above 2^13 and
the pieces' smallest step is 2^-24 (2^-25 off): 2^-38 of that largest. The outer sum is
float32 over the ranks (twice as many terms for the pieces), and the result is rounded
once."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import mlx_lean_moe_amd as gdn

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
U = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}
PIECES = {"bf16": 2.0 ** -16, "f16": 2.0 ** -21, "f32": 0.0}


class _Maker:
    def __init__(self, gpu, act, seed=0):
        self.g = torch.Generator(device=gpu)
        self.g.manual_seed(seed)
        self.gpu, self.dtype = gpu, DT[act]

    def __call__(self, *shape, scale=1.0):
        return (torch.randn(*shape, generator=self.g, device=self.gpu) * scale).to(self.dtype)


def _pairs(m, ranks, K, N):
    return [None if r == 0 else (m(r, K, scale=K ** -0.5), m(N, r, scale=r ** -0.5), 0.5 + 0.25 * i) for i, r in enumerate(ranks)]


def _reference(y, x, block, index):
    """Result and tolerance for one projection, in 64 bits."""
    act = next(a for a, d in DT.items() if d == x.dtype)
    ref, tol = y.double(), torch.zeros(y.shape, dtype=torch.float64, device=y.device)
    for a, pair in enumerate(block):
        rows = torch.tensor([i for i, v in enumerate(index) if v == a], dtype=torch.long, device=y.device)
        if pair is None or not len(rows):
            continue
        A, B, c = pair[0].double(), pair[1].double(), float(np.float32(pair[2]))
        xr = x[rows].double()
        t = xr @ A.T.contiguous()
        mag = (xr.abs() @ A.abs().T.contiguous()) @ B.abs().T.contiguous()
        K, r = A.shape[1], A.shape[0]
        ref[rows] += c * (t @ B.T.contiguous())
        tol[rows] += c * mag * (2 * (K + 4 * r + 24) * 2.0 ** -24 + PIECES[act])
        if act == "f16":
            tol[rows] += c * 2.0 ** -38 * t.abs().amax(1, keepdim=True) * B.abs().sum(1)
    touched = torch.tensor([v >= 0 and block[v] is not None for v in index], device=y.device)
    # one rounding: half a last place, U of the value, and among the type's smallest numbers, which lie
    # 2 U times its smallest normal number apart, half of that step (float16: 2^-24 apart, off by 2^-25)
    tol += torch.where(touched[:, None], U[act] * (ref.abs() + tol) + U[act] * torch.finfo(x.dtype).tiny, 0.0)
    return ref, tol


def _check(got, ref, tol):
    assert torch.isfinite(got).all()
    off = (got.double() - ref).abs()
    assert (off <= tol).all(), f"{int((off > tol).sum())} of {off.numel()}; worst {float((off / tol.clamp(min=1e-300)).max()):.3g}"


def _run(gpu, act, index, ranks, K, widths, seed=0):
    """One call over all projections, checked; ``ranks``: a list for each projection."""
    m = _Maker(gpu, act, seed)
    M = len(index)
    x, ys = m(M, K), [m(M, N) for N in widths]
    blocks = [_pairs(m, r, K, N) for r, N in zip(ranks, widths)]
    adapters = gdn.LowRankAdapters(blocks)
    rows = gdn.AdapterRows(index, len(ranks[0]), device=gpu)
    before = [y.clone() for y in ys]
    outs = gdn.add_low_rank(ys, x, adapters, rows)
    assert outs is ys
    for y, b, block in zip(ys, before, blocks):
        ref, tol = _reference(b, x, block, index)
        _check(y, ref, tol)
    return x, before, ys, adapters, rows


def _index(M, S, seed=0, without=0.0, runs=None):
    rng = np.random.default_rng(seed)
    if runs is None:
        v = rng.integers(0, S, M)
    else:
        v = np.repeat(rng.integers(0, S, runs), -(-M // runs))[:M]
    v[rng.random(M) < without] = -1
    return v.tolist()


@pytest.mark.parametrize("act", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 33, 70])
@pytest.mark.parametrize("K,N,r", [(8, 1, 1), (64, 15, 16), (100, 64, 3), (129, 65, 17), (256, 300, 32), (1000, 257, 50),
                                   (2048, 512, 64), (2050, 130, 100)])
def test_one_projection(gpu, act, M, K, N, r):
    _run(gpu, act, _index(M, 3, seed=M + K), [[r, max(1, r // 2), r]], K, [N], seed=M)


@pytest.mark.parametrize("act", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("M,S,runs", [(64, 32, None), (200, 12, None), (777, 4, 5), (1100, 2, 1), (1024, 1, 1), (300, 300, None),
                                      (2500, 40, 40)])
def test_batches_of_requests(gpu, act, M, S, runs):
    ranks = [(8, 16, 4, 64, 1, 33)[a % 6] for a in range(S)]
    _run(gpu, act, _index(M, S, seed=M, without=0.2, runs=runs), [ranks, ranks[::-1]], 512, [320, 77], seed=S)


@pytest.mark.parametrize("act", ["bf16", "f32"])
def test_projections_without_some_adapters(gpu, act):
    _run(gpu, act, [0, 1, 2, 3, -1, 0, 0, 2], [[16, 0, 5, 0], [0, 0, 40, 8], [3, 0, 0, 0]], 256, [100, 64, 260])
    # a projection that no adapter changes may be left out
    m = _Maker(gpu, act)
    block = _pairs(m, [4, 20], 64, 48)
    adapters = gdn.LowRankAdapters([None, block, None])
    assert adapters.widths == (0, 48, 0)
    x, y = m(5, 64), m(5, 48)
    before, index = y.clone(), [1, 0, -1, 1, 1]
    gdn.add_low_rank([None, y, None], x, adapters, gdn.AdapterRows(index, 2, device=gpu))
    _check(y, *_reference(before, x, block, index))


@pytest.mark.parametrize("act", ["bf16", "f16", "f32"])
def test_large_ranks_and_many_outputs(gpu, act):
    _run(gpu, act, [0] * 80 + [1] * 3, [[300, 7]], 320, [1030])
    _run(gpu, act, [0, 1], [[700, 130]] * 2, 96, [40, 20])


@pytest.mark.parametrize("act", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("M", [5, 150])
def test_strides_and_alignment(gpu, act, M):
    K, widths = 200, (130, 63)
    m = _Maker(gpu, act, 3)
    blocks = [_pairs(m, [16, 9], K, N) for N in widths]
    adapters, index = gdn.LowRankAdapters(blocks), _index(M, 2, without=0.1)
    rows = gdn.AdapterRows(index, 2, device=gpu)
    wide, stacked = m(M, K + 9), m(M, sum(widths) + 11)
    for at in (0, 1, 3, 8):
        x, buf = wide[:, at:at + K], stacked.clone()
        outs = [buf[:, at:at + 130], buf[:, at + 130:at + 193]]
        before = [o.clone() for o in outs]
        gdn.add_low_rank(outs, x, adapters, rows)
        for o, b, block in zip(outs, before, blocks):
            _check(o, *_reference(b, x, block, index))
        untouched = torch.ones(buf.shape[1], dtype=torch.bool)
        untouched[at:at + 193] = False
        assert torch.equal(buf[:, untouched], stacked[:, untouched])
    # x in columns
    xt, y = wide[:, :K].T.contiguous().T, [m(M, N) for N in widths]
    again = [o.clone() for o in y]
    gdn.add_low_rank(y, xt, adapters, rows)
    gdn.add_low_rank(again, xt.contiguous(), adapters, rows)
    assert all(torch.equal(a, b) for a, b in zip(y, again))


def test_rows_without_adapters_are_left_alone(gpu):
    m = _Maker(gpu, "bf16")
    block = _pairs(m, [16], 64, 48)
    adapters = gdn.LowRankAdapters([block])
    x, y = m(40, 64), m(40, 48)
    x[::2] = float("nan")  # rows without an adapter: not read into others
    y[::2] = float("inf")
    before = y.clone()
    index = [-1, 0] * 20
    assert gdn.add_low_rank(y, x, adapters, gdn.AdapterRows(index, 1, device=gpu)) is y
    assert torch.equal(y[::2], before[::2]) and torch.isfinite(y[1::2]).all() and not torch.equal(y, before)
    y = before.clone()
    gdn.add_low_rank(y, x, adapters, gdn.AdapterRows([-1] * 40, 1, device=gpu))
    assert torch.equal(y, before)
    none = gdn.add_low_rank(y[:0], x[:0], adapters, gdn.AdapterRows([], 1, device=gpu))
    assert none.shape == (0, 48)


@pytest.mark.parametrize("act", ["bf16", "f16", "f32"])
def test_values_that_are_not_finite_stay_in_their_row(gpu, act):
    m = _Maker(gpu, act)
    K, N = 96, 80
    block = _pairs(m, [5, 20], K, N)
    adapters = gdn.LowRankAdapters([block])
    index = [0, 0, 1, 0, 1, 1] * 12
    rows = gdn.AdapterRows(index, 2, device=gpu)
    x, y = m(72, K), m(72, N)
    clean = gdn.add_low_rank(y.clone(), x, adapters, rows)
    x2 = x.clone()
    x2[3, 7], x2[40, 0] = float("inf"), float("nan")
    got = gdn.add_low_rank(y.clone(), x2, adapters, rows)
    keep = [i for i in range(72) if i not in (3, 40)]
    assert torch.equal(got[keep], clean[keep]) and got[40].isnan().all() and not torch.isfinite(got[3]).any()
    # large values: t near the type's end and beyond it
    big = {"bf16": 1e30, "f16": 3e4, "f32": 1e30}[act]
    x3 = x * big if act != "f16" else x.clamp(-1, 1) * big
    got = gdn.add_low_rank(torch.zeros_like(y), x3, adapters, rows)
    ref, tol = _reference(torch.zeros_like(y), x3, block, index)
    fine = ref.abs() + tol < torch.finfo(DT[act]).max * (1 - 2 * U[act])
    assert fine.any() and ((got.double() - ref).abs() <= tol)[fine].all()
    # factors among the type's smallest numbers, which the matrix cores take as they are
    tiny = [(A, (B.double() * torch.finfo(DT[act]).tiny * 0.3).to(B.dtype), c) for A, B, c in block]
    tiny += [((A.double() * torch.finfo(DT[act]).tiny * 0.3).to(A.dtype), B, c) for A, B, c in block]
    assert all((t != 0).any() and (t.abs() < torch.finfo(DT[act]).tiny).sum() > t.numel() / 2
               for t in (tiny[0][1], tiny[1][1], tiny[2][0], tiny[3][0]))
    if act == "f16":
        index2 = [i + 2 * (r % 2) for r, i in enumerate(index)]
        x5 = x * 500
        got = gdn.add_low_rank(torch.zeros_like(y), x5, gdn.LowRankAdapters([tiny]), gdn.AdapterRows(index2, 4, device=gpu))
        ref, tol = _reference(torch.zeros_like(y), x5, tiny, index2)
        assert ((got.double() - ref).abs() <= tol).all() and (ref.abs() > 2.0 ** -16).any()
        # inner products far beyond the type: infinite results, and none where B is zero
        far = [(A, B * (torch.arange(N, device=gpu)[:, None] % 2), 2.0 ** 110) for A, B, _ in block]
        got = gdn.add_low_rank(y.clone(), x, gdn.LowRankAdapters([far]), rows)
        assert torch.equal(got[:, ::2], y[:, ::2]) and not torch.isfinite(got[:, 1::2]).any()
    # and small ones
    x4 = x * (1e-6 if act == "f16" else 1e-30)
    got = gdn.add_low_rank(torch.zeros_like(y), x4, adapters, rows)
    ref, tol = _reference(torch.zeros_like(y), x4, block, index)
    assert ((got.double() - ref).abs() <= tol).all()


@pytest.mark.parametrize("act", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("r", [16, 64])
def test_results_do_not_depend_on_the_batch(gpu, act, r):
    """A row's bits are the same from call to call and whichever rows and projections it
    comes with: one launch, two, and every cut of both add in the same order."""
    m = _Maker(gpu, act)
    blocks = [_pairs(m, [r, 7, r, r], 1100, N) for N in (600, 70)]
    adapters, alone = gdn.LowRankAdapters(blocks), gdn.LowRankAdapters(blocks[1:])
    M = 9000
    x, ys, index = m(M, 1100), [m(M, 600), m(M, 70)], _index(M, 4, without=0.1)
    rows = gdn.AdapterRows(index, 4, device=gpu)
    first = gdn.add_low_rank([y.clone() for y in ys], x, adapters, rows)
    again = gdn.add_low_rank([y.clone() for y in ys], x, adapters, rows)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    order = torch.randperm(M, generator=torch.Generator().manual_seed(1)).to(gpu)
    for at in (order[:1], order[:2], order[:17], order[:300], order[:2000], order):
        part = gdn.AdapterRows([index[i] for i in at.tolist()], 4, device=gpu)
        got = gdn.add_low_rank([y[at] for y in ys], x[at], adapters, part)
        assert all(torch.equal(g, f[at]) for g, f in zip(got, first))
        assert torch.equal(gdn.add_low_rank(ys[1][at], x[at], alone, part), first[1][at])


@pytest.mark.parametrize("act", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("ranks", [[16], [30], [64, 1], [100]])
def test_prompts_of_many_rows(gpu, act, ranks):
    """Two launches, with the first product's larger workgroups."""
    _run(gpu, act, [0] * 8300 + [-1] * 5 + [len(ranks) - 1] * 70, [ranks], 104, [70])


def test_numbers_from_tensors_and_runs(gpu):
    m = _Maker(gpu, "bf16")
    block = _pairs(m, [4, 8, 16], 64, 40)
    adapters = gdn.LowRankAdapters([block])
    x, y = m(90, 64), m(90, 40)
    index = [2] * 50 + [-1] * 10 + [0] * 30
    want = gdn.add_low_rank(y.clone(), x, adapters, gdn.AdapterRows(index, 3, device=gpu))
    _check(want, *_reference(y, x, block, index))
    for form in (np.array(index), torch.tensor(index, dtype=torch.int32), torch.tensor(index, device=gpu)):
        assert torch.equal(gdn.add_low_rank(y.clone(), x, adapters, gdn.AdapterRows(form, 3, device=gpu)), want)
    runs = gdn.PackedRuns([0, 50, 50, 60, 90], device=gpu)
    assert torch.equal(gdn.add_low_rank(y.clone(), x, adapters, gdn.AdapterRows.of_runs(runs, [2, 1, -1, 0], 3)), want)


def test_graph_with_other_adapters_each_replay(gpu):
    m = _Maker(gpu, "bf16")
    widths = (300, 64)
    blocks = [_pairs(m, [16, 8, 40, 1], 512, N) for N in widths]
    adapters = gdn.LowRankAdapters(blocks)
    rows = gdn.AdapterRows([0] * 70, 4, device=gpu, distinct=4)
    x, base = m(70, 512), [m(70, N) for N in widths]
    ys = [b.clone() for b in base]
    gdn.add_low_rank(ys, x, adapters, rows)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for y, b in zip(ys, base):
            y.copy_(b)
        gdn.add_low_rank(ys, x, adapters, rows)
    for seed in range(5):
        index = _index(70, 4, seed=seed, without=0.3) if seed != 2 else [-1] * 70
        rows.assign(index)
        x.copy_(m(70, 512))
        graph.replay()
        torch.cuda.synchronize()
        for y, b, block in zip(ys, base, blocks):
            _check(y, *_reference(b, x, block, index))


def test_two_streams_at_once(gpu):
    m = _Maker(gpu, "bf16")
    adapters = gdn.LowRankAdapters([_pairs(m, [16] * 8, 2048, 2048)])
    index = _index(64, 8)
    rows = gdn.AdapterRows(index, 8, device=gpu)
    x, y = m(64, 2048), m(64, 2048)
    want = gdn.add_low_rank(y.clone(), x, adapters, rows)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    torch.cuda.synchronize()
    for i in range(8):
        with torch.cuda.stream(streams[i % 2]):
            got.append(gdn.add_low_rank(y.clone(), x, adapters, rows))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_a_saved_output_is_noticed(gpu):
    m = _Maker(gpu, "f32")
    adapters = gdn.LowRankAdapters([_pairs(m, [4], 64, 48)])
    rows = gdn.AdapterRows([0, -1, 0], 1, device=gpu)
    x, y, w = m(3, 64), m(3, 48), m(48, 5).requires_grad_()
    loss = (y @ w).sum()
    with torch.no_grad():
        gdn.add_low_rank(y, x, adapters, rows)
    with pytest.raises(RuntimeError, match="inplace operation"):
        loss.backward()
    with torch.inference_mode():
        gdn.add_low_rank(m(3, 48), x, adapters, rows)


def test_refusals(gpu):
    m = _Maker(gpu, "bf16")
    K, N = 64, 48
    pair = lambda r=4, k=K, n=N: (m(r, k), m(n, r), 1.0)
    for bad in ([], [None], [[None]], [[pair()], [pair(), pair()]], [[pair(), pair(k=65)]], [[pair(), pair(n=47)]],
                [[(m(4, K), m(N, 5), 1.0)]], [[(m(4, K), m(N, 4).float(), 1.0)]], [[pair()]] * 9, [[pair(n=0)]],
                [[(m(0, K), m(N, 0), 1.0)]], [[(m(4, K).double(), m(N, 4).double(), 1.0)]]):
        with pytest.raises(ValueError):
            gdn.LowRankAdapters(bad)
    with pytest.raises(RuntimeError):
        gdn.LowRankAdapters([[tuple(t.cpu() if isinstance(t, torch.Tensor) else t for t in pair())]])
    with pytest.raises(RuntimeError, match="no gradient"):
        gdn.LowRankAdapters([[(m(4, K).requires_grad_(), m(N, 4), 1.0)]])
    adapters = gdn.LowRankAdapters([[pair(), pair()]])
    rows = gdn.AdapterRows([0, 1, -1], 2, device=gpu)
    x, y = m(3, K), m(3, N)
    for call in (lambda: gdn.add_low_rank(y, x[:, :-1], adapters, rows), lambda: gdn.add_low_rank(y, x[0], adapters, rows),
                 lambda: gdn.add_low_rank(y, x.float(), adapters, rows),
                 lambda: gdn.add_low_rank(y.float(), x, adapters, rows), lambda: gdn.add_low_rank(y[:2], x, adapters, rows),
                 lambda: gdn.add_low_rank([y, y], x, adapters, rows), lambda: gdn.add_low_rank([None], x, adapters, rows),
                 lambda: gdn.add_low_rank(y, x[:2], adapters, rows),
                 lambda: gdn.add_low_rank(y, x, adapters, gdn.AdapterRows([0, 0, 0], 3, device=gpu)),
                 lambda: gdn.add_low_rank(y.T.contiguous().T, x, adapters, rows),
                 lambda: gdn.add_low_rank(y[:1].expand(3, N), x, adapters, rows),
                 lambda: gdn.add_low_rank(y, x.cpu(), adapters, rows),
                 lambda: gdn.add_low_rank(y, x, adapters, gdn.AdapterRows([0, 1, -1], 2, device="cpu"))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(ValueError, match="keep"):
        gdn.add_low_rank(y, gdn.rms_norm(x, None, 1e-6, quantize=True), adapters, rows)
    square = gdn.LowRankAdapters([[(m(4, K), m(K, 4), 1.0)] * 2])
    with pytest.raises(ValueError, match="overlaps x"):
        gdn.add_low_rank(x, x, square, rows)
    two = gdn.LowRankAdapters([[pair(), pair()]] * 2)
    buf = m(3, 2 * N)
    with pytest.raises(ValueError, match="another"):
        gdn.add_low_rank([buf[:, :N], buf[:, N - 1:-1]], x, two, rows)
    gdn.add_low_rank([buf[:, :N], buf[:, N:]], x, two, rows)
    for call in (lambda: gdn.add_low_rank(y.requires_grad_(), x, adapters, rows),
                 lambda: gdn.add_low_rank(y.detach(), x.requires_grad_(), adapters, rows)):
        with pytest.raises(RuntimeError, match="no gradient"):
            call()
    with torch.no_grad():
        gdn.add_low_rank(y, x, adapters, rows)
