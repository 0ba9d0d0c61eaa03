"""Refusals and host logic of the state-space operators and the block-scaled
8-bit projections (no GPU)."""

from __future__ import annotations

import ctypes
import json
import struct

import numpy as np
import pytest
import torch

import mlx_lean_moe_amd as gdn
from mlx_lean_moe_amd import _lib, quant, weights
from oracle import state_space_ref as R

FP8 = gdn.QuantScheme(8, 128, "fp8_block")


def _p(i):
    return ctypes.c_void_p(1 << (20 + i))


def _err():
    return _lib.load().gdn_last_error().decode()


def _refused(rc, code, what):
    assert rc == code and what in _err(), (rc, _err())


def test_dims():
    d = gdn.StateSpaceDims(2, 8, 128, 64, 4)
    assert d.inner_dim == 512 and d.conv_dim == 512 + 2 * 2 * 128


def test_packed_runs():
    r = gdn.PackedRuns([0, 3, 3, 10], device="cpu")
    assert (len(r), r.tokens, r.longest) == (3, 10, 7) and r.on_device.tolist() == [0, 3, 3, 10]
    assert gdn.PackedRuns(torch.tensor([0, 4]), device="cpu").offsets == (0, 4)
    for bad in ([0], [1, 4], [0, 4, 3], [[0, 4]], []):
        with pytest.raises(ValueError):
            gdn.PackedRuns(bad, device="cpu")


# ---------------------------------------------------------------------------
# C ABI
# ---------------------------------------------------------------------------


def _conv(**kw):
    a = dict(x=_p(0), xs=64, ci=_p(1), co=_p(2), w=_p(3), b=None, cu=None, N=2, T=8, out=_p(4), C=64, K=4, dt=1)
    a.update(kw)
    return _lib.load().gdn_conv_silu(*a.values(), None)


def test_conv_silu_refusals():
    E = _lib.GDN_EINVAL
    _refused(_conv(N=0), E, "bad sizes")
    _refused(_conv(dt=3), E, "dtype")
    _refused(_conv(K=5), _lib.GDN_EUNSUPPORTED, "taps")
    _refused(_conv(K=1), _lib.GDN_EUNSUPPORTED, "taps")
    _refused(_conv(T=9), E, "divisible")
    _refused(_conv(T=1 << 31, N=1), E, "too many")
    _refused(_conv(xs=63), E, "x_stride")
    _refused(_conv(out=None), E, "null")
    _refused(_conv(co=ctypes.c_void_p((1 << 21) + 64)), E, "overlaps")


def _scan(**kw):
    a = dict(x=_p(0), xs=128, B=_p(1), Bs=64, C=_p(2), Cs=64, act=1, dt=_p(3), dts=2, dtd=1, A=_p(4), db=_p(5),
             D=None, si=None, so=_p(6), y=_p(7), yd=1, cu=None, N=1, T=64, longest=0, G=1, H=2, P=64, S=64, ws=None, wb=0)
    a.update(kw)
    return _lib.load().gdn_selective_scan(*a.values(), None)


def test_selective_scan_refusals():
    E = _lib.GDN_EINVAL
    _refused(_scan(H=3, G=2), E, "bad sizes")
    _refused(_scan(T=1 << 31), E, "bad sizes")
    _refused(_scan(yd=4), E, "dtype")
    for kw in (dict(P=60), dict(S=60), dict(S=264)):
        _refused(_scan(xs=1024, Bs=1024, Cs=1024, **kw), _lib.GDN_EUNSUPPORTED, "multiples of 8")
    _refused(_scan(N=3), E, "divisible")
    _refused(_scan(so=None), E, "null")
    _refused(_scan(B=None), E, "null")
    _refused(_scan(xs=127), E, "row stride")
    _refused(_scan(dts=1), E, "row stride")
    _refused(_scan(xs=132), E, "aligned")
    _refused(_scan(x=ctypes.c_void_p(8)), E, "aligned")
    _refused(_scan(si=ctypes.c_void_p((1 << 26) + 16)), E, "overlaps")
    of_dtypes = _lib.load().gdn_selective_scan_workspace_size
    size = lambda *sizes: of_dtypes(1, 1, *sizes)  # bfloat16
    assert of_dtypes(0, 0, 1, 4096, 4096, 1, 2, 64, 64) > 0 and of_dtypes(0, 9, 1, 4096, 4096, 1, 2, 64, 64) == 0
    need = size(1, 4096, 4096, 1, 2, 64, 64)
    assert need > 0 and size(1, 64, 64, 1, 2, 64, 64) == 0 and size(1, 4096, 4096, 1, 2, 60, 64) == 0
    # runs that are all short need no workspace, whatever their number
    assert size(64, 4096, 64, 1, 2, 64, 64) == 0 and size(64, 4096, 0, 1, 2, 64, 64) > 0
    _refused(_scan(T=4096, ws=_p(9), wb=need - 1), E, "workspace")


def _step(**kw):
    a = dict(x=_p(0), xs=256, dt=_p(1), dts=2, ci=_p(2), co=_p(3), w=_p(4), b=None, A=_p(5), db=_p(6), D=None,
             si=_p(7), so=_p(7), y=_p(8), yd=1, B=1, G=1, H=2, P=64, N=64, K=4, act=1, slots=None, pool=0, half=None,
             arr=None)
    a.update(kw)
    return _lib.load().gdn_selective_step(*a.values(), None)


def test_selective_step_refusals():
    E, U = _lib.GDN_EINVAL, _lib.GDN_EUNSUPPORTED
    _refused(_step(G=3), E, "bad sizes")
    _refused(_step(act=5), E, "dtype")
    for kw in (dict(N=60), dict(N=264), dict(P=257), dict(K=5), dict(K=1)):
        _refused(_step(xs=4096, **kw), U, "got")
    _refused(_step(y=None), E, "null")
    _refused(_step(slots=_p(9)), E, "pool size")
    _refused(_step(half=_p(9)), E, "needs slots")
    _refused(_step(slots=_p(9), pool=4, arr=_p(10)), E, "needs conv_half")
    _refused(_step(slots=_p(9), pool=4, half=_p(10)), E, "one array")
    _refused(_step(xs=255), E, "row strides")
    _refused(_step(dts=1), E, "row strides")
    _refused(_step(co=ctypes.c_void_p((1 << 22) + 16)), E, "overlaps")
    _refused(_step(so=ctypes.c_void_p((1 << 27) + 16)), E, "overlaps")
    _refused(_step(si=ctypes.c_void_p(8), so=ctypes.c_void_p(8)), E, "aligned")
    assert _step(B=0) == 0


def test_fp8_refusals():
    lib, E = _lib.load(), _lib.GDN_EINVAL
    args = lambda **kw: [{**dict(x=_p(0), xd=1, w=_p(1), s=_p(2), y=_p(3), yd=1, r=None, M=4, N=64, K=256, ws=_p(4),
                                 wb=1 << 20), **kw}[k] for k in "x xd w s y yd r M N K ws wb".split()] + [None]
    for kw, what in ((dict(K=250), "bad sizes"), (dict(N=0), "bad sizes"), (dict(M=-1), "bad sizes"),
                     (dict(xd=7), "dtype"), (dict(w=None), "null"), (dict(x=ctypes.c_void_p(8)), "aligned"),
                     (dict(M=40, ws=None), "workspace"), (dict(M=40, wb=1000), "workspace")):
        _refused(lib.gdn_fp8_matmul(*args(**kw)), E, what)
    assert lib.gdn_fp8_matmul(*args(M=0)) == 0
    assert lib.gdn_fp8_matmul_workspace_size(1, 4, 64, 250) == 0
    for a in ((_p(0), _p(1), _p(2), 9, 64, 64), (_p(0), _p(1), _p(2), 0, 64, 60), (_p(0), None, _p(2), 0, 64, 64),
              (ctypes.c_void_p(8), _p(1), _p(2), 0, 64, 64)):
        assert lib.gdn_fp8_dequantize(*a, None) == E


# ---------------------------------------------------------------------------
# Python
# ---------------------------------------------------------------------------


def _raises(match, kind=ValueError):
    return pytest.raises(kind, match=match)


def test_conv_silu_checks_before_the_device():
    z = torch.zeros
    with _raises("2 to 4 taps"):
        gdn.conv_silu(z(4, 8), z(1, 4, 8), z(8, 5))
    with _raises("do not match"):
        gdn.conv_silu(z(4, 8), z(1, 3, 9), z(8, 4))
    with _raises("do not match"):
        gdn.conv_silu(z(4, 8), z(1, 3, 8), z(8, 3))
    with _raises("bias"):
        gdn.conv_silu(z(4, 8), z(1, 3, 8), z(8, 4), z(7))
    with _raises("must be"):
        gdn.conv_silu(z(8), z(1, 3, 8), z(8, 4))
    with _raises("ROCm", RuntimeError):
        gdn.conv_silu(z(4, 8), z(1, 3, 8), z(8, 4))


def test_selective_scan_checks_before_the_device():
    z = torch.zeros

    def call(x=z(1, 4, 2, 8), dt=z(1, 4, 2), B=z(1, 4, 1, 8), C=z(1, 4, 1, 8), **kw):
        gdn.selective_scan(x, dt, B, C, z(2), z(2), **kw)

    for kw, match in ((dict(x=z(4, 2, 8)), "x must be"), (dict(C=z(1, 4, 1, 16)), "x must be"),
                      (dict(dt=z(1, 4, 3)), "leading"), (dict(B=z(1, 5, 1, 8), C=z(1, 5, 1, 8)), "leading"),
                      (dict(x=z(1, 4, 2, 12)), "multiples of 8"), (dict(B=z(1, 4, 1, 264), C=z(1, 4, 1, 264)), "at most"),
                      (dict(B=z(1, 4, 3, 8), C=z(1, 4, 3, 8)), "multiple of the groups")):
        with _raises(match):
            call(**kw)
    with _raises("ROCm", RuntimeError):
        call()


def test_selective_step_checks_before_the_device():
    z, d = torch.zeros, gdn.StateSpaceDims(1, 2, 8, 8, 4)

    def call(dims=d, xbc=z(1, 32), dt=z(1, 2), w=z(32, 4)):
        gdn.selective_step(xbc, dt, z(1, 3, 32), z(1, 2, 8, 8), w, None, z(2), z(2), None, dims)

    for kw, match in ((dict(dims=gdn.StateSpaceDims(1, 2, 12, 8, 4)), "needs state_dim"),
                      (dict(dims=gdn.StateSpaceDims(1, 2, 8, 264, 4)), "needs state_dim"),
                      (dict(dims=gdn.StateSpaceDims(1, 2, 8, 8, 5)), "needs state_dim"),
                      (dict(xbc=z(1, 33)), "do not match"), (dict(dt=z(2, 2)), "do not match"),
                      (dict(w=z(32, 3)), "do not match"), (dict(xbc=z(32)), "must be")):
        with _raises(match):
            call(**kw)
    with _raises("ROCm", RuntimeError):
        call()


def test_gradients_are_refused():
    z = torch.zeros
    from mlx_lean_moe_amd import state_space

    with _raises("no gradient", RuntimeError):
        state_space._no_gradient(z(1), z(1, requires_grad=True))
    with torch.no_grad():
        state_space._no_gradient(z(1, requires_grad=True))


def _fp8(N, K, dtype=torch.float8_e4m3fn):
    return {"weight": torch.zeros(N, K).to(torch.float8_e4m3fn).view(dtype), "scales": torch.ones(-(-N // 128), -(-K // 128))}


def test_fp8_scheme_and_layout_checks():
    for bits, group in ((4, 128), (8, 64)):
        with pytest.raises(ValueError):
            gdn.QuantScheme(bits, group, "fp8_block")
    x = torch.zeros(2, 256)
    cases = [(dict(_fp8(4, 256), biases=torch.ones(1, 2)), "no biases"), (dict(_fp8(4, 256), scales=torch.ones(2, 2)), "scales"),
             (dict(_fp8(4, 256), scales=torch.ones(1, 2).bfloat16()), "scales"), (_fp8(4, 128), "input width"),
             (dict(_fp8(4, 256), weight=torch.zeros(4, 256)), "float8_e4m3fn"),
             (dict(_fp8(4, 256), weight=torch.zeros(4, 64, dtype=torch.int32)), "float8_e4m3fn")]
    for tensors, match in cases:
        with _raises(match):
            gdn.quantized_linear(x, tensors, FP8)
    with _raises("multiple of 16"):
        gdn.quantized_linear(torch.zeros(2, 250), _fp8(4, 250), FP8)
    for dtype in (torch.float8_e4m3fn, torch.uint8):
        with _raises("ROCm", RuntimeError):
            gdn.quantized_linear(x, _fp8(4, 256, dtype), FP8)


def test_fp8_stacking_keeps_blocks_whole():
    a, b, c = _fp8(256, 64), _fp8(128, 64), _fp8(70, 64)
    s = quant.concat_quantized([a, b, c])
    assert s["weight"].shape == (454, 64) and s["scales"].shape == (4, 1)
    assert not quant.stackable([c, a])
    with _raises("whole blocks"):
        quant.concat_quantized([a, c, b])
    packed = [{"weight": torch.zeros(3, 8, dtype=torch.int32), "scales": torch.zeros(3, 1)}] * 2
    assert quant.stackable(packed)


def test_fp8_layer_stacks_only_where_the_blocks_allow():
    d = gdn.LinearAttentionDims(1, 2, 64, 64, 4)
    z = torch.zeros
    layer = lambda n: gdn.Qwen3_5LinearAttention(
        d, _fp8(d.conv_dim, 128), _fp8(d.value_dim, 128), _fp8(n, 128), _fp8(n, 128), z(d.conv_dim, 4, 1), z(2), z(2),
        z(64), _fp8(128, 128), quant=FP8)
    assert layer(2)._in_stacked is None  # a's two rows would shift b's blocks
    assert layer(128)._in_stacked.tensors["weight"].shape[0] == d.conv_dim + d.value_dim + 256


def test_fp8_projections_are_read_from_a_checkpoint(tmp_path):
    rng = np.random.default_rng(0)
    codes = rng.integers(0, 120, (130, 144), dtype=np.uint8)
    scales = rng.random((2, 2), np.float32)
    entries, blob = {}, b""
    for name, tag, arr in (("p.weight", "F8_E4M3", codes), ("p.scales", "F32", scales), ("bad.weight", "F8_E4M3", codes),
                           ("bad.scales", "F32", scales[:1])):
        raw = arr.tobytes()
        entries[name] = {"dtype": tag, "shape": list(arr.shape), "data_offsets": [len(blob), len(blob) + len(raw)]}
        blob += raw
    head = json.dumps(entries).encode()
    (tmp_path / "model.safetensors").write_bytes(struct.pack("<Q", len(head)) + head + blob)
    with weights.CheckpointReader(tmp_path) as reader:
        got = weights.read_projection(reader, "p", FP8)
        assert got.quant == FP8 and got.tensors["weight"].dtype == torch.float8_e4m3fn
        assert np.array_equal(got.tensors["weight"].view(torch.uint8).numpy(), codes)
        assert np.array_equal(got.tensors["scales"].numpy(), scales)
        quant._check_quantized(got.tensors, FP8, 144)
        with _raises("scales of shape", weights.LayoutError):
            weights.read_projection(reader, "bad", FP8)


# ---------------------------------------------------------------------------
# the oracle
# ---------------------------------------------------------------------------


def test_oracle_e4m3_is_torchs():
    x = torch.cat([torch.arange(0, 1 << 15).to(torch.int16).view(torch.bfloat16).float(), torch.randn(4096) * 100])
    x = x[torch.isfinite(x) & (x.abs() <= 464)]
    x = torch.cat([x, -x])
    assert np.array_equal(R.e4m3(x.numpy()), x.to(torch.float8_e4m3fn).double().numpy())


def test_oracle_scan_splits_and_conv_is_torchs():
    rng = np.random.default_rng(1)
    n = rng.standard_normal
    args = lambda a, b: (x[a:b], dt[a:b], B[a:b], C[a:b], A, db, D)
    x, dt, B, C, A, db, D = n((9, 4, 3)), n((9, 4)), n((9, 2, 5)), n((9, 2, 5)), n(4), n(4), n(4)
    y, S, _, _ = R.scan(*args(0, 9), None, [9])
    y1, S1, _, _ = R.scan(*args(0, 4), None, [4])
    y2, S2, _, _ = R.scan(*args(4, 9), S1, [5])
    np.testing.assert_allclose(np.concatenate([y1, y2]), y, rtol=1e-12)
    np.testing.assert_allclose(S2, S, rtol=1e-12)
    xc, w, b = n((1, 6, 20)), n((6, 4)), n(6)
    ref = torch.nn.functional.silu(torch.nn.functional.conv1d(
        torch.nn.functional.pad(torch.tensor(xc), (3, 0)), torch.tensor(w)[:, None], torch.tensor(b), groups=6))
    out, st, _, _ = R.conv_silu(xc[0].T, np.zeros((1, 3, 6)), w, b, [20])
    np.testing.assert_allclose(out, ref[0].T.numpy(), rtol=1e-12)
    assert np.array_equal(st[0], xc[0].T[-3:])
