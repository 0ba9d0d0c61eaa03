"""GPU parity of rms_norm, its residual and its 8-bit output with the formulas in
float64.

The result is by definition the exact value rounded to float32 and then to the
rows' type. float64 sums of up to 2^17 squares, in whatever order, differ by
less than 2^-36 of their size, so float32 results may differ by one of their last
places, and 16-bit ones not at all unless a value lies that near a tie."""

from __future__ import annotations

import pytest
import torch

import mlx_lean_moe_amd as gdn
from mlx_lean_moe_amd import quant

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
FP8 = gdn.QuantScheme(8, 128, "fp8_block")


def _x(gpu, *shape, act="bf16", seed=0):
    g = torch.Generator(device=gpu)
    g.manual_seed(seed)
    t = torch.randn(*shape, generator=g, device=gpu) * torch.exp(torch.randn(*shape[:-1], 1, generator=g, device=gpu))
    return t.to(DT[act])


def _w(gpu, K, seed=9):
    g = torch.Generator(device=gpu)
    g.manual_seed(seed)
    return torch.rand(K, generator=g, device=gpu) + 0.5


def _ref(x, w, eps, residual=None):
    """(normed in 64 bits, stream)"""
    s = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    v = s.double()
    v = v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)
    return (v if w is None else v * w.double()), s


def _equal(a, b):
    """The same bits, NaN where NaN."""
    return a.shape == b.shape and a.dtype == b.dtype and bool(((a == b) | (a.isnan() & b.isnan())).all())


def _check(got, ref, act):
    want = ref.to(DT[act])
    if act == "f32":
        fine = torch.isfinite(want)
        assert torch.equal(fine, torch.isfinite(got))
        off = (got.double() - ref).abs()[fine]
        assert (off <= 2.0 ** -23 * ref.abs()[fine] + 2.0 ** -149).all()
    else:
        assert _equal(got, want)


def _codes(y):
    """Codes and scales that the product makes of y, from torch operations."""
    K = y.shape[-1]
    rows = torch.nn.functional.pad(y.float(), (0, -K % 128)).unflatten(-1, (-1, 128))
    s = rows.abs().amax(-1, keepdim=True) / torch.full((1,), 448.0, device=y.device)
    s = s.clamp(min=2.0 ** -126)
    return (rows / s).to(torch.float8_e4m3fn).flatten(-2)[..., :K], s[..., 0]


@pytest.mark.parametrize("act", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("M,K", [(1, 1), (3, 7), (2, 8), (17, 16), (5, 127), (33, 128), (4, 129), (9, 500), (6, 513),
                                 (3, 2047), (1, 2048), (70, 2048), (2, 2056), (5, 4096), (3, 5000), (2, 8192), (2, 8200),
                                 (3, 16384), (2, 16385), (2, 40000)])
def test_against_the_definition(gpu, act, M, K):
    x, r, w = _x(gpu, M, K, act=act), _x(gpu, M, K, act=act, seed=1), _w(gpu, K)
    _check(gdn.rms_norm(x, w, 1e-6), _ref(x, w, 1e-6)[0], act)
    _check(gdn.rms_norm(x, None, 1e-5), _ref(x, None, 1e-5)[0], act)
    y, s = gdn.rms_norm(x, w, 1e-6, residual=r)
    ref, stream = _ref(x, w, 1e-6, r)
    assert torch.equal(s, stream)
    _check(y, ref, act)
    # the fused addition is the addition and then the norm
    assert torch.equal(y, gdn.rms_norm(s, w, 1e-6))


@pytest.mark.parametrize("act", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("M,K", [(1, 16), (3, 112), (17, 128), (5, 144), (33, 512), (4, 528), (1, 2048), (300, 2048),
                                 (7, 4096), (2, 8192), (3, 16384), (2, 16400), (2, 40000)])
def test_codes_are_those_of_the_rows(gpu, act, M, K):
    x, r, w = _x(gpu, M, K, act=act), _x(gpu, M, K, act=act, seed=1), _w(gpu, K)
    y, s = gdn.rms_norm(x, w, 1e-6, residual=r)
    q, s2 = gdn.rms_norm(x, w, 1e-6, residual=r, quantize=True)
    kept, _ = gdn.rms_norm(x, w, 1e-6, residual=r, quantize=True, keep_rows=True)
    assert torch.equal(s, s2) and torch.equal(kept.rows, y) and q.rows is None
    codes, scales = _codes(y)
    for got in (q, kept):
        assert got.shape == x.shape and got.dtype == x.dtype
        assert torch.equal(got.codes.float(), codes.float()) and torch.equal(got.scales, scales)
        # a code is off by at most half a step (2^-4 of the value, or half the smallest code)
        tol = y.float().abs() * 2.0 ** -4 + got.scales.repeat_interleave(128, -1)[:, :K] * 2.0 ** -10
        assert ((got.dequantize() - y.float()).abs() <= tol).all()


@pytest.mark.parametrize("act", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("M", [1, 2, 16, 17, 65, 300])
@pytest.mark.parametrize("N,K", [(1, 16), (64, 144), (300, 1024), (2048, 2048), (6100, 256), (12352, 2048)])
def test_products_of_codes_are_those_of_the_rows(gpu, act, M, N, K):
    g = torch.Generator(device=gpu)
    g.manual_seed(2)
    W = {"weight": (torch.randn(N, K, generator=g, device=gpu) * 60).clamp(-440, 440).to(torch.float8_e4m3fn),
         "scales": torch.rand(-(-N // 128), -(-K // 128), generator=g, device=gpu) * 0.02 + 1e-3}
    x, w, res = _x(gpu, M, K, act=act), _w(gpu, K), _x(gpu, M, N, act=act, seed=3)
    y = gdn.rms_norm(x, w, 1e-6)
    q = gdn.rms_norm(x, w, 1e-6, quantize=True)
    assert torch.equal(gdn.quantized_linear(q, W, FP8), gdn.quantized_linear(y, W, FP8))
    assert torch.equal(gdn.quantized_linear(q, gdn.LinearWeights(W, FP8), residual=res),
                       gdn.quantized_linear(y, W, FP8, residual=res))


@pytest.mark.parametrize("M", [1, 40, 2100])
def test_codes_times_stacked_projections(gpu, M):
    """The blocks that quantized_linear_split gives of rows and of their codes."""
    sizes, K = [384, 128, 70], 272
    g = torch.Generator(device=gpu)
    g.manual_seed(3)
    W = gdn.LinearWeights({"weight": (torch.randn(582, K, generator=g, device=gpu) * 60).clamp(-440, 440).to(torch.float8_e4m3fn),
                           "scales": torch.rand(5, 3, generator=g, device=gpu)}, FP8)
    x = _x(gpu, M, K)
    q = gdn.rms_norm(x, None, 1e-6, quantize=True)
    for got, want in zip(quant.quantized_linear_split(q, W, sizes), quant.quantized_linear_split(gdn.rms_norm(x, None, 1e-6), W, sizes)):
        assert torch.equal(got, want)


@pytest.mark.parametrize("act", ["bf16", "f16", "f32"])
def test_values_that_are_not_ordinary(gpu, act):
    K = 272
    big = {"bf16": 1e38, "f16": 6e4, "f32": 1e38}[act]
    small = {"bf16": 1e-39, "f16": 6e-8, "f32": 1e-41}[act]
    x = _x(gpu, 12, K, act=act)
    x[0] = 0
    x[1, 5] = float("inf")
    x[2, 7] = float("nan")
    x[3] *= big / 100
    x[4] = small
    x[5] = 0
    x[5, 3] = small
    x[6, ::2] = 0
    x[7, 200] = big
    w = _w(gpu, K)
    w[9], w[10], w[11], w[12] = 0.0, 1e30, 1e-38, -2.0
    for eps in (1e-6, 0.0, 1e-30):
        ref, _ = _ref(x, w, eps)
        got = gdn.rms_norm(x, w, eps)
        if act == "f32":
            assert torch.equal(got.isnan(), ref.isnan())
            got, ref = got.nan_to_num(), ref.float().nan_to_num()
            assert ((got - ref).abs() <= 2.0 ** -23 * ref.abs() + 2.0 ** -149).all()
        else:
            assert _equal(got, ref.float().to(DT[act]))
        q = gdn.rms_norm(x, w, eps, quantize=True)
        codes, scales = _codes(gdn.rms_norm(x, w, eps))
        fine = torch.isfinite(scales)
        wide = fine.repeat_interleave(128, -1)[:, :K]
        assert torch.equal(q.scales[fine], scales[fine]) and torch.equal(q.codes.float()[wide], codes.float()[wide])
        assert torch.equal(torch.isfinite(q.scales), fine)
        # a group with a value that is not finite is NaN
        assert q.codes.float()[~wide].isnan().all()
        assert (q._data[:12 * 384].view(12, 384)[:, K:][fine[:, -1]] == 0).all()


def test_results_do_not_depend_on_the_batch(gpu):
    x, w = _x(gpu, 1100, 2048), _w(gpu, 2048)
    whole = gdn.rms_norm(x, w, 1e-6, quantize=True)
    for rows in (slice(0, 1), slice(1099, 1100), slice(17, 64)):
        part = gdn.rms_norm(x[rows], w, 1e-6, quantize=True)
        assert torch.equal(part.codes.float(), whole.codes.float()[rows]) and torch.equal(part.scales, whole.scales[rows])


@pytest.mark.parametrize("act", ["bf16", "f32"])
@pytest.mark.parametrize("K", [128, 250, 2048, 3000])
def test_strides_alignment_and_ranks(gpu, act, K):
    w = _w(gpu, K)
    wide = _x(gpu, 6, 2 * K + 3, act=act)
    res = _x(gpu, 6, K + 1, act=act, seed=4)
    for x in (wide[:, :K], wide[:, 1:K + 1], wide[:, K + 3:], wide[::2, 3:K + 3], wide.T.contiguous().T[:, :K]):
        r = res[:x.shape[0], 1:]
        y, s = gdn.rms_norm(x, w, 1e-6, residual=r)
        y2, s2 = gdn.rms_norm(x.contiguous(), w, 1e-6, residual=r.contiguous())
        assert torch.equal(y, y2) and torch.equal(s, s2)
    x = wide[:, :K].contiguous()
    y = gdn.rms_norm(x, w, 1e-6)
    assert torch.equal(gdn.rms_norm(x[2], w, 1e-6), y[2])
    assert torch.equal(gdn.rms_norm(x.view(2, 3, K), w.to(torch.bfloat16).float(), 1e-6),
                       gdn.rms_norm(x, w.to(torch.bfloat16), 1e-6).view(2, 3, K))
    assert gdn.rms_norm(x[:0], w, 1e-6).shape == (0, K)
    assert gdn.rms_norm(x.permute(1, 0).contiguous().permute(1, 0), w, 1e-6).equal(y)
    if K % 16 == 0:
        q = gdn.rms_norm(x.view(2, 3, K), w, 1e-6, quantize=True, keep_rows=True)
        assert q.codes.shape == (2, 3, K) and q.scales.shape == (2, 3, -(-K // 128)) and q.ndim == 3
        flat = q.reshape(6, K)
        assert flat.shape == (6, K) and torch.equal(flat.rows, y) and torch.equal(flat.codes.float(), q.codes.float().view(6, K))
        assert q.reshape(-1, K).shape == (6, K)
        one = gdn.rms_norm(x[2], w, 1e-6, quantize=True)
        assert one.codes.shape == (K,) and torch.equal(one.codes.float(), flat.codes.float()[2])
        none = gdn.rms_norm(x[:0], w, 1e-6, quantize=True)
        assert none.codes.shape == (0, K) and none.scales.shape == (0, -(-K // 128)) and none.dequantize().shape == (0, K)
        W = {"weight": torch.ones(4, K, device=gpu).to(torch.float8_e4m3fn), "scales": torch.ones(1, -(-K // 128), device=gpu)}
        assert gdn.quantized_linear(none, W, FP8).shape == (0, 4)
        assert gdn.quantized_linear(one, W, FP8).shape == (4,)
        assert gdn.quantized_linear(q, W, FP8).shape == (2, 3, 4)


@pytest.mark.parametrize("act", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("K", [100, 128, 2048, 16400])
def test_the_stream_in_place(gpu, act, K):
    w = _w(gpu, K)
    x, r = _x(gpu, 19, K, act=act), _x(gpu, 19, K, act=act, seed=5)
    y, s = gdn.rms_norm(x, w, 1e-6, residual=r)
    for which in ("x", "residual", "slice", "other"):
        xc, rc = x.clone(), r.clone()
        buf = torch.full((19, K + 5), 7.0, dtype=DT[act], device=gpu)
        out = {"x": xc, "residual": rc, "slice": buf[:, 2:K + 2], "other": torch.empty_like(x)}[which]
        y2, s2 = gdn.rms_norm(xc, w, 1e-6, residual=rc, sum_out=out)
        assert s2 is out and torch.equal(out, s) and torch.equal(y2, y)
        if which == "slice":
            assert (buf[:, :2] == 7).all() and (buf[:, K + 2:] == 7).all()
        if which != "x":
            assert torch.equal(xc, x)
        if which != "residual":
            assert torch.equal(rc, r)
    # x as its own residual
    xc = x.clone()
    y2, s2 = gdn.rms_norm(xc, w, 1e-6, residual=xc, sum_out=xc)
    assert torch.equal(s2, (x.float() * 2).to(DT[act]))


@pytest.mark.parametrize("act", ["bf16", "f32"])
def test_the_stream_beside_its_inputs(gpu, act):
    """Columns of one buffer: the sum's lie between x's and the residual's and share none."""
    K, w = 96, _w(gpu, 96)
    buf = torch.full((19, 3 * K + 4), 7.0, dtype=DT[act], device=gpu)
    x, s, r = buf[:, :K], buf[:, K:2 * K], buf[:, 2 * K:3 * K]
    x.copy_(_x(gpu, 19, K, act=act))
    r.copy_(_x(gpu, 19, K, act=act, seed=5))
    want, stream = gdn.rms_norm(x.clone(), w, 1e-6, residual=r.clone())
    before = buf.clone()
    got, out = gdn.rms_norm(x, w, 1e-6, residual=r, sum_out=s)
    assert out is s and torch.equal(got, want) and torch.equal(s, stream)
    assert torch.equal(x, before[:, :K]) and torch.equal(buf[:, 2 * K:], before[:, 2 * K:])
    for out in (buf[:, K - 1:2 * K - 1], buf[:, K + 1:2 * K + 1]):  # the last column of x, the first of the residual
        with pytest.raises(ValueError, match="overlap"):
            gdn.rms_norm(x, w, 1e-6, residual=r, sum_out=out)
    with pytest.raises(ValueError, match="overlap"):  # in x's columns, another distance apart
        gdn.rms_norm(x[:9], w, 1e-6, residual=r[:9], sum_out=buf.view(-1).as_strided((9, K), (2 * K, 1), 11))


def test_a_saved_stream_written_in_place_is_noticed(gpu):
    x, w = _x(gpu, 3, 96, act="f32"), torch.ones(96, device=gpu, requires_grad=True)
    saved = x.clone()
    loss = (saved * w).sum()
    with torch.no_grad():
        gdn.rms_norm(saved, None, 1e-6, residual=x, sum_out=saved)
    with pytest.raises(RuntimeError, match="inplace operation"):
        loss.backward()
    with torch.inference_mode():
        kept = x.clone()
        gdn.rms_norm(kept, None, 1e-6, residual=x, sum_out=kept)
    gdn.rms_norm(kept, None, 1e-6, residual=x, sum_out=x.clone())


def test_rows_beyond_one_row_of_the_grid(gpu):
    M, K = (1 << 21) * 16 + 21, 16
    x, w = torch.ones(M, K, dtype=torch.bfloat16, device=gpu), _w(gpu, K)
    x[-1], x[0, 3], x[(1 << 21) * 16 - 1, 5] = 3, 5, 7
    y = gdn.rms_norm(x, w, 1e-6)
    want = gdn.rms_norm(x[:1], w, 1e-6)
    at = [0, 1, (1 << 21) * 16 - 1, (1 << 21) * 16, M - 1]
    assert torch.equal(y[at], torch.cat([gdn.rms_norm(x[i:i + 1], w, 1e-6) for i in at]))
    assert torch.equal(y[1:(1 << 21) * 16 - 1], y[1:2].expand((1 << 21) * 16 - 2, K)) and not torch.equal(want, y[1:2])
    q = gdn.rms_norm(x, w, 1e-6, quantize=True)
    assert torch.equal(q.codes[at].float(), _codes(y[at])[0].float()) and torch.equal(q.scales[at], _codes(y[at])[1])
    del x, y, q
    torch.cuda.empty_cache()


def test_streams_and_graphs(gpu):
    x, r, w = _x(gpu, 40, 2048), _x(gpu, 40, 2048, seed=6), _w(gpu, 2048)
    want, s = gdn.rms_norm(x, w, 1e-6, residual=r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, s2 = gdn.rms_norm(x, w, 1e-6, residual=r)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want) and torch.equal(s, s2)
    torch.cuda.synchronize()
    stream = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, out = gdn.rms_norm(stream, w, 1e-6, residual=r, quantize=True, sum_out=stream)
    for i in range(4):  # the stream moves on with every replay
        before = stream.clone()
        graph.replay()
        want, s = gdn.rms_norm(before, w, 1e-6, residual=r)
        torch.cuda.synchronize()
        assert torch.equal(stream, s) and torch.equal(q.codes.float(), _codes(want)[0].float())


def test_refusals(gpu):
    x, w = _x(gpu, 4, 96), _w(gpu, 96)
    bad = [dict(weight=w[:5]), dict(residual=x[:2]), dict(residual=x.float()), dict(sum_out=x), dict(keep_rows=True),
           dict(residual=x, sum_out=x.float()), dict(residual=x, sum_out=x[:2]),
           dict(residual=x.clone(), sum_out=x.view(-1).as_strided((4, 96), (48, 1))),
           dict(weight=torch.ones(96, dtype=torch.float64, device=gpu)), dict(weight=w.long())]
    for more in bad:
        args = {"weight": w, **more}
        with pytest.raises(ValueError):
            gdn.rms_norm(x, args.pop("weight"), 1e-6, **args)
    with pytest.raises(ValueError, match="multiple of 16"):
        gdn.rms_norm(x[:, :90], w[:90], 1e-6, quantize=True)
    with pytest.raises(ValueError):
        gdn.rms_norm(x[:, :0], w[:0], 1e-6)
    with pytest.raises(ValueError):
        gdn.rms_norm(x.double(), w, 1e-6)
    with pytest.raises((ValueError, RuntimeError)):
        gdn.rms_norm(x, w.cpu(), 1e-6)
    flat = torch.zeros(5 * 96, dtype=x.dtype, device=gpu)
    with pytest.raises(ValueError, match="overlap"):  # one row on
        gdn.rms_norm(flat[:4 * 96].view(4, 96), w, 1e-6, residual=x, sum_out=flat[96:].view(4, 96))
    q = gdn.rms_norm(x, w, 1e-6, quantize=True)
    with pytest.raises(ValueError, match="keep"):
        gdn.quantized_linear(q, torch.ones(3, 96, device=gpu, dtype=x.dtype))
    kept = gdn.rms_norm(x, w, 1e-6, quantize=True, keep_rows=True)
    dense = torch.ones(3, 96, device=gpu, dtype=x.dtype)
    assert torch.equal(gdn.quantized_linear(kept, dense), gdn.quantized_linear(kept.rows, dense))
    W = {"weight": torch.ones(4, 112, device=gpu).to(torch.float8_e4m3fn), "scales": torch.ones(1, 1, device=gpu)}
    with pytest.raises(ValueError, match="width"):
        gdn.quantized_linear(q, W, FP8)
    with pytest.raises(ValueError, match="width"):
        q.reshape(2, 192)
    for call in (lambda t: gdn.rms_norm(t, w, 1e-6), lambda t: gdn.rms_norm(x, w, 1e-6, residual=t)):
        with pytest.raises(RuntimeError, match="no gradient"):
            call(x.clone().requires_grad_())
        with torch.no_grad():
            call(x.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="no gradient"):
        gdn.rms_norm(x, w.clone().requires_grad_(), 1e-6)
