"""`Qwen3_5LinearAttention` on fp8_block projections: loaded from a checkpoint,
stacked and apart, over prompts, single tokens, a pool and captured graphs. Its
projections are `quantized_linear` on the stored tensors, bit for bit, and the
rest is the layer's own core."""

from __future__ import annotations

import json
import struct

import pytest
import torch

import mlx_lean_moe_amd as gdn
from mlx_lean_moe_amd import weights as W

pytestmark = pytest.mark.gpu

FP8 = gdn.QuantScheme(8, 128, "fp8_block")
PREFIX = "language_model.model.layers.0.linear_attn"
HIDDEN = 272  # (the last block of K is short)


def _checkpoint(path, Hk, Hv, seed=0):
    """safetensors of one layer, e4m3 codes with scales; returns its config."""
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    C, V = 2 * Hk * 128 + Hv * 128, Hv * 128
    tensors = {}
    for name, n, k in (("in_proj_qkv", C, HIDDEN), ("in_proj_z", V, HIDDEN), ("in_proj_a", Hv, HIDDEN),
                       ("in_proj_b", Hv, HIDDEN), ("out_proj", HIDDEN, V)):
        tensors[f"{name}.weight"] = ("F8_E4M3", (r(n, k) * 60).clamp(-440, 440).to(torch.float8_e4m3fn).view(torch.uint8))
        tensors[f"{name}.scales"] = ("F32", (torch.rand(-(-n // 128), -(-k // 128), generator=g) + 0.5) / 60 / k ** 0.5)
    tensors["conv1d.weight"] = ("F32", r(C, 4, 1) * 0.3)
    tensors["A_log"] = ("F32", torch.rand(Hv, generator=g))
    tensors["dt_bias"] = ("F32", r(Hv) - 2)
    tensors["norm.weight"] = ("F32", torch.rand(128, generator=g) + 0.5)
    entries, blob = {}, b""
    for name, (tag, t) in tensors.items():
        raw = t.contiguous().numpy().tobytes()
        entries[f"{PREFIX}.{name}"] = {"dtype": tag, "shape": list(t.shape), "data_offsets": [len(blob), len(blob) + len(raw)]}
        blob += raw
    head = json.dumps(entries).encode()
    (path / "model.safetensors").write_bytes(struct.pack("<Q", len(head)) + head + blob)
    return {"linear_num_key_heads": Hk, "linear_num_value_heads": Hv, "linear_key_head_dim": 128,
            "linear_value_head_dim": 128, "linear_conv_kernel_dim": 4,
            "quantization_config": {"bits": 8, "group_size": 128, "mode": "fp8_block"}}


# (the front-end of float32 prompts takes no more than 16384 channels)
@pytest.mark.parametrize("act,Hk,Hv", [(torch.bfloat16, 2, 4), (torch.float32, 2, 4), (torch.bfloat16, 16, 128)])
def test_layer(gpu, tmp_path, act, Hk, Hv):
    """4 heads leave a and b no whole blocks: four products; 128 stack into one."""
    config = _checkpoint(tmp_path, Hk, Hv)
    layer = W.load_linear_attention(tmp_path, 0, device=gpu, hf_config=config)
    assert (layer._in_stacked is None) == (Hv == 4)
    layer.keep_dense_weights()  # nothing to keep: these products never run on dense weights
    d = layer.linear
    x = torch.randn(150, HIDDEN, device=gpu, generator=torch.Generator(gpu).manual_seed(1)).to(act)

    def project(rows):
        sizes = [d.conv_dim, d.value_dim, Hv, Hv]
        if layer._in_stacked is not None:
            qkv, z, a, b = gdn.quantized_linear(rows, layer._in_stacked).split(sizes, dim=-1)
        else:
            qkv, z, a, b = (gdn.quantized_linear(rows, w) for w in (layer.in_proj_qkv, layer.in_proj_z, layer.in_proj_a,
                                                                    layer.in_proj_b))
        return qkv, z.reshape(-1, Hv, 128), a, b

    cache = layer.new_cache(act)
    conv, ssm = (s[None] for s in cache.state())
    out, conv, ssm = layer.core(*project(x[:140]), conv.to(act), ssm)
    want = gdn.quantized_linear(out, layer.out_proj, residual=x[:140])
    y = layer(x[:140], cache, residual=x[:140])
    assert torch.isfinite(y).all() and torch.equal(y, want) and torch.equal(cache.ssm_state, ssm[0])
    for t in range(140, 150):
        out, conv, ssm = gdn.fused_decode_step(*project(x[t:t + 1]), conv, ssm, layer.conv1d_weight, layer.A_log,
                                               layer.dt_bias, layer.norm_weight, layer.rms_norm_eps, d)
        want = gdn.quantized_linear(out.reshape(1, -1), layer.out_proj, residual=x[t:t + 1])
        assert torch.equal(layer(x[t], cache, residual=x[t]), want[0])
    assert torch.equal(cache.ssm_state, ssm[0])


@pytest.mark.parametrize("Hk,Hv", [(2, 4), (16, 128)])
def test_pool_and_graphs(gpu, tmp_path, Hk, Hv):
    config = _checkpoint(tmp_path, Hk, Hv, 2)
    layer = W.load_linear_attention(tmp_path, 0, device=gpu, hf_config=config)
    d = layer.linear
    g = torch.Generator(gpu).manual_seed(3)
    r = lambda *s: torch.randn(*s, device=gpu, generator=g).bfloat16()
    pool = lambda: gdn.RecurrentStatePool(6, 4, d.conv_dim, Hv, 128, 128, dtype=torch.bfloat16, device=gpu)
    eager, graphed = pool(), pool()
    slots = [4, 0, 3]
    step = gdn.DecodeGraph(layer, graphed, slots, r(3, HIDDEN), residual_example=r(3, HIDDEN))
    chunk = gdn.PrefillGraph(layer, r(70, HIDDEN), residual_example=r(70, HIDDEN))
    one, other = layer.new_cache(torch.bfloat16), layer.new_cache(torch.bfloat16)
    for _ in range(4):
        x, res = r(3, HIDDEN), r(3, HIDDEN)
        want = layer.decode_batch(x, eager, slots=slots, residual=res)
        torch.cuda.synchronize()
        assert torch.equal(step.step(x, res), want)
        assert torch.equal(eager.ssm_state, graphed.ssm_state) and torch.equal(eager.conv_state, graphed.conv_state)
        x, res = r(70, HIDDEN), r(70, HIDDEN)
        want = layer(x, one, residual=res)
        torch.cuda.synchronize()
        assert torch.equal(chunk.step(other, x, res), want)
        assert torch.equal(one.ssm_state, other.ssm_state)
