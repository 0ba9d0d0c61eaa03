"""GPU parity of the block-scaled 8-bit projections with their float64
definition.

Codes and scales are exact by definition (float32 quotients). float32 results
are float32 sums: a term passes the 128 sums of its block, one product and one
sum per block. 16-bit results are one rounding (two with a residual) from sums
of the 8-bit matrix cores, which keep at least 11 bits below the largest
product of a block (13 were measured): 2^-11 of the absolute sum."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import mlx_lean_moe_amd as gdn
from mlx_lean_moe_amd import quant
from oracle import state_space_ref as R

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
U = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}
FP8 = gdn.QuantScheme(8, 128, "fp8_block")


def _np(t):
    return t.detach().double().cpu().numpy()


def _weights(gpu, N, K, seed=0):
    g = torch.Generator(device=gpu)
    g.manual_seed(seed)
    w = (torch.randn(N, K, generator=g, device=gpu) * 60).clamp(-440, 440).to(torch.float8_e4m3fn)
    s = torch.rand(-(-N // 128), -(-K // 128), generator=g, device=gpu) * 0.02 + 1e-3
    return {"weight": w, "scales": s}


def _x(gpu, M, K, act, seed=0):
    g = torch.Generator(device=gpu)
    g.manual_seed(seed + 100)
    return (torch.randn(M, K, generator=g, device=gpu) * torch.exp(torch.randn(M, 1, generator=g, device=gpu))).to(DT[act])


def _check(y, x, W, act, residual=None):
    K = x.shape[1]
    ref, mag = R.fp8_block_matmul(x.float().cpu().numpy(), _np(W["weight"].float()), _np(W["scales"]))
    tol = (mag * (128 + K / 128 + 8) * 2.0 ** -24) if act == "f32" else mag * 2.0 ** -11
    tol = tol + U[act] * (np.abs(ref) + tol) + 2.0 ** -24 * U[act]
    if residual is not None:
        ref = ref + _np(residual)
        tol = tol + U[act] * (np.abs(ref) + tol)
    got = _np(y)
    assert got.shape == ref.shape and np.isfinite(got).all()
    bad = np.abs(got - ref) > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.size}; worst ratio {(np.abs(got - ref) / tol).max():.3g}"


@pytest.mark.parametrize("act", ["bf16", "f32", "f16"])
@pytest.mark.parametrize("M", [1, 2, 15, 17, 33, 64, 65, 130, 300])
@pytest.mark.parametrize("N,K", [(1, 16), (4, 112), (64, 128), (127, 144), (129, 272), (300, 1024), (512, 2048)])
def test_against_the_definition(gpu, act, M, N, K):
    W, x = _weights(gpu, N, K), _x(gpu, M, K, act)
    y = gdn.quantized_linear(x, W, FP8)
    assert y.dtype == DT[act]
    _check(y, x, W, act)


@pytest.mark.parametrize("act", ["bf16", "f32"])
@pytest.mark.parametrize("M,N,K", [(600, 1000, 1040), (1025, 640, 2048), (520, 260, 96), (200, 2048, 4096), (4, 2048, 4096),
                                   (2049, 384, 256)])
def test_larger_products_with_residual(gpu, act, M, N, K):
    W, x = _weights(gpu, N, K, 1), _x(gpu, M, K, act, 1)
    res = _x(gpu, M, N, act, 2)
    y = gdn.quantized_linear(x, gdn.LinearWeights(W, FP8), residual=res)
    _check(y, x, W, act, res)
    plain = gdn.quantized_linear(x, W, FP8)
    if act == "bf16":  # the layer's sum of two arrays, bit for bit
        assert torch.equal(y, plain + res)


@pytest.mark.parametrize("act", ["bf16", "f32"])
@pytest.mark.parametrize("M,N,K", [(1, 6100, 256), (16, 6100, 144), (1, 12170, 128), (16, 12170, 272), (12, 130, 4096),
                                   (13, 130, 4096), (1, 20, 49168)])
def test_few_rows_of_many_outputs_and_of_long_rows(gpu, act, M, N, K):
    """Each width of the workgroups that quantize the rows themselves, and both
    sides of where they leave that to a launch of its own."""
    W, x = _weights(gpu, N, K, 4), _x(gpu, M, K, act, 4)
    res = _x(gpu, M, N, act, 5)
    _check(gdn.quantized_linear(x, W, FP8, residual=res), x, W, act, res)


@pytest.mark.parametrize("act", ["bf16", "f32"])
@pytest.mark.parametrize("M,N,K", [(2100, 8261, 256), (2100, 8256, 256), (4100, 4160, 144)])
def test_columns_in_two_launches(gpu, act, M, N, K):
    """Products whose last round of tiles is cut off, with odd and even rows."""
    W, x = _weights(gpu, N, K, 6), _x(gpu, M, K, act, 6)
    res = _x(gpu, M, N, act, 7)
    _check(gdn.quantized_linear(x, W, FP8, residual=res), x, W, act, res)
    if N % 8 == 0:
        _check(gdn.quantized_linear(x, W, FP8), x, W, act)


@pytest.mark.parametrize("act", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("M", [1, 16, 40, 200, 700])
def test_codes_and_scales_are_the_definitions(gpu, act, M):
    """A weight of one code per row hands the quantized x through: in float32
    results its values are exact, so are codes and scales, ties included."""
    K = 400
    x = _x(gpu, M, K, act, 3)
    x[0] = torch.arange(K, device=gpu) % 17 * 0.5  # many ties under power-of-two scales
    x[0, ::128] = 448.0
    x[-1, :128] = 0.0
    eye = torch.eye(K, device=gpu).to(torch.float8_e4m3fn)
    W = {"weight": eye, "scales": torch.ones(4, 4, device=gpu)}
    q, s = R.quantize_rows(x.float().cpu().numpy())
    want = (q * np.repeat(s.astype(np.float64), 128, axis=1)[:, :K])
    y = gdn.quantized_linear(x.float(), W, FP8)
    assert np.array_equal(_np(y), want.astype(np.float32).astype(np.float64))


def test_non_finite_rows_stay_their_own(gpu):
    W = _weights(gpu, 200, 304)
    for M in (5, 100, 600):
        for act in ("bf16", "f32"):
            x = _x(gpu, M, 304, act)
            clean = gdn.quantized_linear(x, W, FP8)
            x[1, 7], x[3, 303] = float("nan"), float("-inf")
            y = gdn.quantized_linear(x, W, FP8)
            assert torch.isnan(y[[1, 3]]).all()
            keep = [i for i in range(M) if i not in (1, 3)]
            assert torch.equal(y[keep], clean[keep])


def test_extreme_magnitudes(gpu):
    """Rows of float32's smallest and largest values: scales stay normal. The
    product of both scales may not: it is then rounded by up to 2^-150, which
    the sum of |q w| multiplies."""
    W = _weights(gpu, 64, 256)
    W["scales"] = torch.full((1, 2), 1e-3, device=gpu)
    x = torch.randn(4, 256, device=gpu)
    x = x * torch.tensor([1e-38, 1e-30, 1.0, 1e33], device=gpu)[:, None]
    x[0, :128] = 0
    ref, mag = R.fp8_block_matmul(x.cpu().numpy(), _np(W["weight"].float()), _np(W["scales"]))
    got = _np(gdn.quantized_linear(x, W, FP8))
    q, _ = R.quantize_rows(x.cpu().numpy())
    codes = np.abs(q) @ np.abs(_np(W["weight"].float())).T
    assert (np.abs(got - ref) <= mag * 2.0 ** -16 + codes * 2.0 ** -149 + 2.0 ** -149).all()


def test_layouts_and_leading_axes(gpu):
    W, x = _weights(gpu, 130, 272), _x(gpu, 24, 272, "bf16")
    want = gdn.quantized_linear(x, W, FP8)
    assert torch.equal(gdn.quantized_linear(x.reshape(2, 3, 4, 272), W, FP8), want.reshape(2, 3, 4, 130))
    assert torch.equal(gdn.quantized_linear(x[0], W, FP8), want[0])
    wide = torch.empty(24, 275, dtype=torch.bfloat16, device=gpu)
    wide[:, 1:273] = x
    raw = {"weight": W["weight"].view(torch.uint8), "scales": W["scales"].T.contiguous().T}
    assert torch.equal(gdn.quantized_linear(wide[:, 1:273], raw, FP8), want)
    assert gdn.quantized_linear(x[:0], W, FP8).shape == (0, 130)
    off = torch.empty(130 * 272 + 1, dtype=torch.uint8, device=gpu)[1:].view(130, 272).copy_(raw["weight"])
    assert torch.equal(gdn.quantized_linear(x, {"weight": off, "scales": W["scales"]}, FP8), want)


def test_dequantize(gpu):
    W = _weights(gpu, 200, 144)
    dense = _np(W["weight"].float()) * np.repeat(np.repeat(_np(W["scales"]), 128, 0)[:200], 128, 1)[:, :144]
    assert np.array_equal(_np(gdn.dequantize(W, FP8, torch.float32)), dense.astype(np.float32))
    got = gdn.dequantize(W, FP8)
    assert got.dtype == torch.bfloat16
    assert torch.equal(got, torch.tensor(dense.astype(np.float32), device=gpu).bfloat16())
    kept = gdn.LinearWeights(W, FP8).with_dense()
    assert kept.dense is None


def test_stacked_projections_split(gpu):
    parts = [_weights(gpu, n, 256, i) for i, n in enumerate((256, 128, 70))]
    x = _x(gpu, 40, 256, "bf16")
    stacked = gdn.LinearWeights(quant.concat_quantized(parts), FP8)
    for got, p in zip(quant.quantized_linear_split(x, stacked, [256, 128, 70]), parts):
        assert torch.equal(got, gdn.quantized_linear(x, p, FP8))


@pytest.mark.parametrize("M", [3, 90, 600])
def test_streams_and_graph(gpu, M):
    W = _weights(gpu, 512, 1024)
    x = _x(gpu, M, 1024, "bf16")
    gdn.quantized_linear(x, W, FP8)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = gdn.quantized_linear(x, W, FP8)
    side = torch.cuda.Stream()
    for i in range(4):
        x.copy_(_x(gpu, M, 1024, "bf16", 10 + i))
        want = gdn.quantized_linear(x, W, FP8)
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            other = gdn.quantized_linear(x, W, FP8)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(other, want)


def test_state_space_layer_end_to_end(gpu):
    """A whole layer as it is used: 8-bit input projection, conv, scan, gated
    norm, 8-bit output projection with the residual, for a packed prompt; then
    a token from the pool, against the same layer in float64 on the values the
    bfloat16 hand-overs hold."""
    torch.manual_seed(0)
    hidden, H, P, G, N = 256, 8, 64, 2, 64
    d = gdn.StateSpaceDims(G, H, N, P, 4)
    Win, Wout = _weights(gpu, H * P + d.conv_dim + H, hidden, 1), _weights(gpu, hidden, H * P, 2)
    Win["scales"] *= 0.1
    cw, cb = torch.randn(d.conv_dim, 4, device=gpu) * 0.4, torch.randn(d.conv_dim, device=gpu) * 0.1
    A_log, dtb, D = torch.rand(H, device=gpu) * 2, torch.randn(H, device=gpu) - 3, torch.rand(H, device=gpu)
    nw = torch.rand(P, device=gpu) + 0.5
    lens = [90, 0, 33]
    runs = gdn.PackedRuns([0, 90, 90, 123])

    def project(x):
        return torch.split(gdn.quantized_linear(x, Win, FP8), [H * P, d.conv_dim, H], dim=-1)

    def finish(y, z, x):
        o = gdn.gated_rms_norm(y, z.unflatten(-1, (H, P)), nw, 1e-6)
        return o, gdn.quantized_linear(o.reshape(len(x), H * P), Wout, FP8, residual=x)

    x = torch.randn(123, hidden, device=gpu).bfloat16()
    conv0 = torch.zeros(3, 3, d.conv_dim, device=gpu, dtype=torch.bfloat16)
    z, xbc, dt = project(x)
    u, conv = gdn.conv_silu(xbc, conv0, cw, cb, runs)
    xs, B, C = torch.split(u, [H * P, G * N, G * N], dim=-1)
    y, ssm = gdn.selective_scan(xs.unflatten(-1, (H, P)), dt, B.unflatten(-1, (G, N)), C.unflatten(-1, (G, N)), A_log,
                                dtb, D, cu_seqlens=runs)
    o, out = finish(y, z, x)
    _check(out, o.reshape(123, H * P), Wout, "bf16", x)
    ref, state, ya, sa = R.scan(_np(xs).reshape(-1, H, P), _np(dt), _np(B).reshape(-1, G, N), _np(C).reshape(-1, G, N),
                                _np(A_log), _np(dtb), _np(D), None, lens)
    assert (np.abs(_np(y) - ref) <= 2.0 ** -8 * (np.abs(ref) + 1.02 * ya)).all()
    zz, yy = _np(z).reshape(-1, H, P), _np(y)
    norm = yy / np.sqrt((yy ** 2).mean(-1, keepdims=True) + 1e-6) * _np(nw) * R.silu(zz)
    assert (np.abs(_np(o) - norm) <= 2.1 * 2.0 ** -8 * np.abs(norm) + 1e-6).all()

    pool = gdn.RecurrentStatePool(4, 4, d.conv_dim, H, P, N, dtype=torch.bfloat16, device=gpu)
    cache = gdn.RecurrentCache(4, d.conv_dim, H, P, N, dtype=torch.bfloat16, device=gpu)
    for run, slot in ((0, 2), (2, 0)):
        cache.update(conv[run], ssm[run], lens[run])
        pool.load(slot, cache)
        cache.size = 0
    slots = pool.device_slots([2, 0])
    xt = torch.randn(2, hidden, device=gpu).bfloat16()
    z, xbc, dt = project(xt)
    y, _, _ = gdn.selective_step(xbc, dt, pool.conv_buf, pool.ssm_state, cw, cb, A_log, dtb, D, d, slots=slots,
                                 conv_half=pool.conv_half_dev, conv_arrivals=pool.conv_arrivals)
    pool.advance([2, 0], slots, device_flipped=True)
    o, out = finish(y, z, xt)
    _check(out, o.reshape(2, H * P), Wout, "bf16", xt)
    um, new, _, _ = R.conv_silu(_np(xbc), _np(conv[[0, 2]]), _np(cw), _np(cb), [1, 1])
    ref, state, ya, _ = R.scan(um[:, :H * P].reshape(2, H, P), _np(dt), um[:, H * P:H * P + G * N].reshape(2, G, N),
                               um[:, H * P + G * N:].reshape(2, G, N), _np(A_log), _np(dtb), _np(D), _np(ssm[[0, 2]]), [1, 1])
    assert np.array_equal(_np(pool.conv_state[[2, 0]]), new)
    assert (np.abs(_np(y) - ref) <= 2.0 ** -8 * np.abs(ref) + 2.0 ** -14 * ya + 1e-9).all()
    assert np.abs(_np(pool.ssm_state[[2, 0]]) - state).max() <= 1e-5 * np.abs(state).max()
    assert pool.size.tolist() == [34, 0, 91, 0]
