"""`Qwen3_5LinearAttention` with its input's norm inside and low-rank adapters beside
its projections: over prompts, single tokens, a pool and captured graphs. The result
is that of the operators called one after the other, bit for bit, and near that of
projections with the adapters multiplied into them."""

from __future__ import annotations

import json
import struct

import numpy as np
import pytest
import torch

import mlx_lean_moe_amd as gdn
from mlx_lean_moe_amd import quant, weights as W

pytestmark = pytest.mark.gpu

HIDDEN, HK, HV = 512, 2, 4
D = gdn.LinearAttentionDims(HK, HV, 128, 128, 4)
WIDTHS = {"in_proj_qkv": D.conv_dim, "in_proj_z": D.value_dim, "in_proj_a": HV, "in_proj_b": HV, "out_proj": HIDDEN}
NAMES = tuple(WIDTHS)
EPS = 1e-6


def _gen(gpu, seed):
    return torch.Generator(gpu).manual_seed(seed)


def _affine(w, bits=4, group=64):
    """MLX's packing of w in groups."""
    N, K = w.shape
    v = w.reshape(N, K // group, group)
    lo, hi = v.amin(-1), v.amax(-1)
    scale = ((hi - lo) / (2 ** bits - 1)).clamp(min=1e-8)
    q = ((v - lo[..., None]) / scale[..., None]).round().clamp(0, 2 ** bits - 1).to(torch.int64).reshape(N, -1, 32 // bits)
    words = (q << (torch.arange(32 // bits, device=w.device) * bits)).sum(-1)
    words = torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)
    return {"weight": words.contiguous(), "scales": scale.bfloat16(), "biases": lo.bfloat16()}


def _fp8(w):
    N, K = w.shape
    wide = torch.zeros(-(-N // 128) * 128, -(-K // 128) * 128, device=w.device)
    wide[:N, :K] = w
    blocks = wide.view(-(-N // 128), 128, -(-K // 128), 128)
    scales = blocks.abs().amax((1, 3)) / 448
    return {"weight": (blocks / scales[:, None, :, None]).reshape(wide.shape)[:N, :K].contiguous().to(torch.float8_e4m3fn),
            "scales": scales.contiguous()}


def _layer(gpu, kind, seed=0, norm=False, dense_ab=False):
    g = _gen(gpu, seed)
    r = lambda *s: torch.randn(*s, device=gpu, generator=g)
    dense = {n: r(N, HIDDEN if n != "out_proj" else D.value_dim) * (HIDDEN ** -0.5) for n, N in WIDTHS.items()}
    scheme = {"dense": None, "affine4": gdn.QuantScheme(4, 64), "fp8": gdn.QuantScheme(8, 128, "fp8_block")}[kind]
    make = {"dense": lambda w: w, "affine4": lambda w: gdn.LinearWeights(_affine(w), scheme),
            "fp8": lambda w: gdn.LinearWeights(_fp8(w), scheme)}[kind]
    p = {n: w if dense_ab and n in ("in_proj_a", "in_proj_b") else make(w) for n, w in dense.items()}
    rest = [r(D.conv_dim, 4, 1) * 0.3, torch.rand(HV, device=gpu, generator=g), r(HV) - 2,
            torch.rand(128, device=gpu, generator=g) + 0.5]
    weight = torch.rand(HIDDEN, device=gpu, generator=g) + 0.5
    layer = gdn.Qwen3_5LinearAttention(D, p["in_proj_qkv"], p["in_proj_z"], p["in_proj_a"], p["in_proj_b"], *rest,
                                       p["out_proj"], rms_norm_eps=EPS, input_norm_weight=weight if norm else None)
    return layer, dense, rest, weight


def _adapters(gpu, act, seed=5, names=NAMES, S=3):
    g = _gen(gpu, seed)
    r = lambda *s: torch.randn(*s, device=gpu, generator=g)
    out = {}
    for n in names:
        K = HIDDEN if n != "out_proj" else D.value_dim
        out[n] = [(r(rank, K).mul(K ** -0.5).to(act), r(WIDTHS[n], rank).mul(0.3 * rank ** -0.5).to(act), 1.0 + 0.5 * i)
                  for i, rank in enumerate((16, 4, 33)[:S])]
    return out


def _by_hand(layer, x, cache, adapters, rows, residual=None, norm=None):
    """The layer from its operators."""
    if norm is not None:
        x = gdn.rms_norm(x, norm, EPS)
    if layer._in_stacked is not None:
        qkv, z, ab = quant.quantized_linear_split(x, layer._in_stacked, [D.conv_dim, D.value_dim, 2 * HV])
        a, b = ab.split([HV, HV], dim=-1)
    else:
        qkv, z, a, b = (layer._proj(x, getattr(layer, n)) for n in NAMES[:4])
    ins = [adapters.get(n) for n in NAMES[:4]]
    if any(p is not None for p in ins):
        gdn.add_low_rank([qkv, z, a, b], x, gdn.LowRankAdapters(ins), rows)
    conv, ssm = cache.state()
    z = z.reshape(-1, HV, 128)
    if len(x) == 1:
        out, conv, ssm = gdn.fused_decode_step(qkv, z, a, b, conv[None].to(x.dtype), ssm[None], layer.conv1d_weight, layer.A_log,
                                               layer.dt_bias, layer.norm_weight, EPS, D)
        out = out.reshape(1, -1)
    else:
        out, conv, ssm = layer.core(qkv, z, a, b, conv[None], ssm[None])
    y = layer._proj(out, layer.out_proj, residual)
    if adapters.get("out_proj") is not None:
        gdn.add_low_rank(y, out, gdn.LowRankAdapters([adapters["out_proj"]]), rows)
    cache.update(conv[0], ssm[0], advance=len(x))
    return y


@pytest.mark.parametrize("kind,act", [("dense", torch.bfloat16), ("dense", torch.float32), ("affine4", torch.bfloat16),
                                      ("affine4", torch.float32), ("fp8", torch.bfloat16), ("fp8", torch.float32)])
@pytest.mark.parametrize("names", [NAMES, ("in_proj_qkv",), ("out_proj",), ("in_proj_z", "in_proj_b", "out_proj")])
def test_layer_is_its_operators(gpu, kind, act, names):
    layer, _, _, weight = _layer(gpu, kind, norm=True)
    adapters = _adapters(gpu, act, names=names)
    layer.set_adapters(**adapters)
    x = torch.randn(150, HIDDEN, device=gpu, generator=_gen(gpu, 1)).to(act)
    index = [0] * 60 + [-1] * 30 + [2] * 60
    one, other = layer.new_cache(act), layer.new_cache(act)
    rows = gdn.AdapterRows(index, 3, device=gpu)
    want = _by_hand(layer, x, other, adapters, rows, x, weight)
    got = layer(x, one, residual=x, adapter_rows=rows)
    assert torch.isfinite(got).all() and torch.equal(got, want) and torch.equal(one.ssm_state, other.ssm_state)
    for t in range(4):
        row = gdn.AdapterRows([(0, 1, -1, 2)[t]], 3, device=gpu)
        want = _by_hand(layer, x[t:t + 1], other, adapters, row, x[t:t + 1], weight)
        assert torch.equal(layer(x[t], one, residual=x[t], adapter_rows=row), want[0])
        assert torch.equal(one.ssm_state, other.ssm_state)
    # without the rows' adapters the layer is what it was
    plain, _, _, _ = _layer(gpu, kind, norm=True)
    assert torch.equal(layer(x, layer.new_cache(act)), plain(x, plain.new_cache(act)))


@pytest.mark.parametrize("kind,act", [("dense", torch.bfloat16), ("affine4", torch.bfloat16), ("fp8", torch.bfloat16),
                                      ("fp8", torch.float32)])
@pytest.mark.parametrize("dense_ab", [False, True])
def test_norm_inside_is_norm_in_front(gpu, kind, act, dense_ab):
    inside, _, _, weight = _layer(gpu, kind, norm=True, dense_ab=dense_ab)
    plain, _, _, _ = _layer(gpu, kind, dense_ab=dense_ab)
    x = torch.randn(90, HIDDEN, device=gpu, generator=_gen(gpu, 2)).to(act)
    a, b, c = (layer.new_cache(act) for layer in (inside, plain, plain))
    y = gdn.rms_norm(x, weight, EPS)
    assert torch.equal(inside(x, a, residual=x), plain(y, b, residual=x))
    if kind == "fp8":  # codes made in front of the layer
        q = gdn.rms_norm(x, weight, EPS, quantize=True, keep_rows=dense_ab)
        want = plain(y, layer_cache := plain.new_cache(act), residual=x)
        assert torch.equal(plain(q, c, residual=x), want) and torch.equal(c.ssm_state, layer_cache.ssm_state)
        one = gdn.rms_norm(x[3], weight, EPS, quantize=True, keep_rows=dense_ab)
        assert torch.equal(plain(one, c), plain(y[3], layer_cache))
        if dense_ab:
            with pytest.raises(ValueError, match="keep"):
                plain(gdn.rms_norm(x, weight, EPS, quantize=True), c)
        with pytest.raises(ValueError, match="itself"):
            inside(q, a)
        with pytest.raises(ValueError, match="plain rows"):
            gdn.PrefillGraph(plain, q)
    assert torch.equal(inside(x[5], a, residual=x[5]), plain(y[5], b, residual=x[5]))


def test_adapters_multiplied_into_the_projections(gpu):
    """float32 from end to end: the layer with an adapter is that of W + c B A."""
    layer, dense, rest, _ = _layer(gpu, "dense")
    adapters = _adapters(gpu, torch.float32)
    layer.set_adapters(**adapters)
    x = torch.randn(140, HIDDEN, device=gpu, generator=_gen(gpu, 3))
    for which in range(3):
        merged = {n: w + adapters[n][which][2] * (adapters[n][which][1] @ adapters[n][which][0]) for n, w in dense.items()}
        other = gdn.Qwen3_5LinearAttention(D, *[merged[n] for n in NAMES[:4]], *rest, merged["out_proj"], rms_norm_eps=EPS)
        got = layer(x, layer.new_cache(), adapter_rows=gdn.AdapterRows([which] * 140, 3, device=gpu))
        want = other(x, other.new_cache())
        # float32 projections of 512 terms: 2^-24 sqrt(512) of their size, through a recurrence and a norm; an
        # adapter left out or scaled wrongly is off by tenths
        assert float((got - want).abs().max() / want.abs().max()) < 1e-4


@pytest.mark.parametrize("kind", ["dense", "affine4", "fp8"])
def test_pool_and_graphs(gpu, kind):
    layer, _, _, _ = _layer(gpu, kind, seed=4, norm=True)
    act = torch.bfloat16
    layer.set_adapters(**_adapters(gpu, act))
    g = _gen(gpu, 6)
    r = lambda *s: torch.randn(*s, device=gpu, generator=g).to(act)
    pool = lambda: gdn.RecurrentStatePool(6, 4, D.conv_dim, HV, 128, 128, dtype=act, device=gpu)
    eager, graphed, slots = pool(), pool(), [4, 0, 3]
    rows, chunk_rows = gdn.AdapterRows([0, 1, 2], 3, device=gpu), gdn.AdapterRows([0] * 70, 3, device=gpu)
    step = gdn.DecodeGraph(layer, graphed, slots, r(3, HIDDEN), residual_example=r(3, HIDDEN), adapter_rows=rows)
    chunk = gdn.PrefillGraph(layer, r(70, HIDDEN), residual_example=r(70, HIDDEN), adapter_rows=chunk_rows)
    one, other = layer.new_cache(act), layer.new_cache(act)
    for i in range(5):
        x, index = r(3, HIDDEN), [[0, 1, 2], [-1, 2, 2], [1, 1, 1], [-1, -1, -1], [2, 0, -1]][i]
        rows.assign(index)
        want = layer.decode_batch(x, eager, slots=slots, residual=x, adapter_rows=gdn.AdapterRows(index, 3, device=gpu))
        torch.cuda.synchronize()
        got = step.step(x, x)
        # (the sums of x A^T may be split otherwise for another batch's plan: here both plans are alike)
        assert torch.equal(got, want) and torch.equal(eager.ssm_state, graphed.ssm_state)
        x, which = r(70, HIDDEN), (0, 2, -1, 1, 0)[i]
        chunk_rows.assign([which] * 70)
        want = layer(x, one, residual=x, adapter_rows=chunk_rows)
        torch.cuda.synchronize()
        assert torch.equal(chunk.step(other, x, x), want) and torch.equal(one.ssm_state, other.ssm_state)
    # a graph keeps the adapters that it was captured with
    saved = [t.clone() for t in (one.conv_state, one.ssm_state)]
    x = r(70, HIDDEN)
    want = layer(x, one, residual=x, adapter_rows=chunk_rows)
    layer.set_adapters(out_proj=_adapters(gpu, act, seed=50)["out_proj"])
    other.update(saved[0], saved[1], advance=0)
    torch.cuda.synchronize()
    assert torch.equal(chunk.step(other, x, x), want)


@pytest.mark.parametrize("kind,act", [("affine4", torch.bfloat16), ("fp8", torch.float16), ("dense", torch.float32)])
def test_quantized_linear_with_adapters(gpu, kind, act):
    layer, dense, _, _ = _layer(gpu, kind)
    w = dense["in_proj_qkv"].to(act) if kind == "dense" else layer.in_proj_qkv
    adapters = gdn.LowRankAdapters([_adapters(gpu, act)["in_proj_qkv"]])
    x = torch.randn(2, 5, HIDDEN, device=gpu, generator=_gen(gpu, 7)).to(act)
    res = torch.randn(2, 5, D.conv_dim, device=gpu, generator=_gen(gpu, 8)).to(act)
    rows = gdn.AdapterRows([0, 1, 2, -1, 0] * 2, 3, device=gpu)
    want = gdn.quantized_linear(x, w, residual=res)
    gdn.add_low_rank(want.view(10, -1), x.view(10, -1), adapters, rows)
    assert torch.equal(gdn.quantized_linear(x, w, residual=res, adapters=adapters, adapter_rows=rows), want)
    one = gdn.AdapterRows([1], 3, device=gpu)
    assert gdn.quantized_linear(x[0, 0], w, adapters=adapters, adapter_rows=one).shape == (D.conv_dim,)
    with pytest.raises(ValueError, match="together"):
        gdn.quantized_linear(x, w, adapters=adapters)
    with pytest.raises(ValueError, match="together"):
        gdn.quantized_linear(x, w, adapter_rows=rows)


def test_refusals(gpu):
    layer, _, _, _ = _layer(gpu, "dense")
    x = torch.randn(3, HIDDEN, device=gpu).bfloat16()
    rows = gdn.AdapterRows([0, 1, 2], 3, device=gpu)
    with pytest.raises(ValueError, match="no adapters"):
        layer(x, layer.new_cache(torch.bfloat16), adapter_rows=rows)
    good = _adapters(gpu, torch.bfloat16)
    for bad in (dict(in_proj_qkv=good["in_proj_z"]), dict(out_proj=good["in_proj_z"][:2], in_proj_z=good["in_proj_z"]),
                dict(out_proj=[(good["in_proj_qkv"][0][0][:, :500], good["out_proj"][0][1], 1.0)])):
        with pytest.raises(ValueError):
            layer.set_adapters(**bad)
    layer.set_adapters(**good)
    with pytest.raises(ValueError):
        layer(x, layer.new_cache(torch.bfloat16), adapter_rows=gdn.AdapterRows([0, 1], 3, device=gpu))
    with pytest.raises(ValueError):
        layer(x.float(), layer.new_cache(), adapter_rows=rows)
    layer.set_adapters()
    with pytest.raises(ValueError, match="no adapters"):
        layer(x, layer.new_cache(torch.bfloat16), adapter_rows=rows)


def test_a_refused_step_leaves_the_pool_as_it_was(gpu):
    """What only out_proj's adapters would notice, at the step's end."""
    layer, _, _, _ = _layer(gpu, "dense")
    x = torch.randn(3, HIDDEN, device=gpu).bfloat16()
    rows = lambda index, count, device=gpu: gdn.AdapterRows(index, count, device=device)
    only_out = _adapters(gpu, torch.bfloat16, names=("out_proj",))
    with pytest.raises(ValueError, match="projection"):
        layer.set_adapters(out_proj=[(A, B[:-1].contiguous(), c) for A, B, c in only_out["out_proj"]])
    pool = gdn.RecurrentStatePool(4, 4, D.conv_dim, HV, 128, 128, dtype=torch.bfloat16, device=gpu)
    layer.decode_batch(x, pool, slots=[3, 0, 1])
    kept = [t.clone() for t in (pool.ssm_state, pool.conv_buf, pool.conv_half_dev)]
    sizes = pool.size.clone()
    for adapters, bad in ((only_out, rows([0, 1], 3)), (only_out, rows([0, 1, 1], 2)), (only_out, rows([0, 1, 2], 3, "cpu")),
                          (_adapters(gpu, torch.float32, names=("out_proj",)), rows([0, 1, 2], 3))):
        layer.set_adapters(**adapters)
        with pytest.raises(ValueError):
            layer.decode_batch(x, pool, slots=[3, 0, 1], adapter_rows=bad)
        assert torch.equal(pool.size, sizes)
        for was, now in zip(kept, (pool.ssm_state, pool.conv_buf, pool.conv_half_dev)):
            assert torch.equal(was, now)


def test_norm_from_a_checkpoint(gpu, tmp_path):
    g = torch.Generator().manual_seed(0)
    prefix = "language_model.model.layers.0"
    tensors = {f"linear_attn.{n}.weight": torch.randn(N, HIDDEN if n != "out_proj" else D.value_dim, generator=g) * 0.05
               for n, N in WIDTHS.items()}
    tensors |= {"linear_attn.conv1d.weight": torch.randn(D.conv_dim, 4, 1, generator=g), "linear_attn.A_log": torch.rand(HV, generator=g),
                "linear_attn.dt_bias": torch.randn(HV, generator=g), "linear_attn.norm.weight": torch.rand(128, generator=g),
                "input_layernorm.weight": torch.rand(HIDDEN, generator=g) + 0.5}
    entries, blob = {}, b""
    for name, t in tensors.items():
        raw = t.numpy().astype(np.float32).tobytes()
        entries[f"{prefix}.{name}"] = {"dtype": "F32", "shape": list(t.shape), "data_offsets": [len(blob), len(blob) + len(raw)]}
        blob += raw
    head = json.dumps(entries).encode()
    (tmp_path / "model.safetensors").write_bytes(struct.pack("<Q", len(head)) + head + blob)
    config = {"linear_num_key_heads": HK, "linear_num_value_heads": HV, "linear_key_head_dim": 128,
              "linear_value_head_dim": 128, "linear_conv_kernel_dim": 4}
    plain = W.load_linear_attention(tmp_path, 0, device=gpu, hf_config=config)
    inside = W.load_linear_attention(tmp_path, 0, device=gpu, hf_config=config, input_norm=True)
    assert plain.input_norm_weight is None
    assert torch.equal(inside.input_norm_weight.cpu(), tensors["input_layernorm.weight"])
    x = torch.randn(20, HIDDEN, device=gpu)
    y = gdn.rms_norm(x, inside.input_norm_weight, EPS)
    assert torch.equal(inside(x, inside.new_cache(), residual=x), plain(y, plain.new_cache(), residual=x))
