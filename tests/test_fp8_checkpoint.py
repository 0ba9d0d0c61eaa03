"""Checkpoints whose e4m3 codes stand without the scales that the reader
knows: refused, never taken for plain weights (no GPU)."""

from __future__ import annotations

import json
import struct

import numpy as np
import pytest
import torch

import mlx_lean_moe_amd as gdn
from mlx_lean_moe_amd import weights

FP8 = gdn.QuantScheme(8, 128, "fp8_block")
AFFINE = gdn.QuantScheme(4, 64, "affine")


def _checkpoint(path, tensors):
    entries, blob = {}, b""
    for name, (tag, arr) in tensors.items():
        raw = arr.tobytes()
        entries[name] = {"dtype": tag, "shape": list(arr.shape), "data_offsets": [len(blob), len(blob) + len(raw)]}
        blob += raw
    head = json.dumps(entries).encode()
    (path / "model.safetensors").write_bytes(struct.pack("<Q", len(head)) + head + blob)


CODES = np.full((130, 144), 0x38, np.uint8)  # 1.0 each
SCALES = np.full((2, 2), 1e-3, np.float32)


@pytest.mark.parametrize("scheme", [FP8, AFFINE])
def test_codes_without_their_scales_are_refused(tmp_path, scheme):
    _checkpoint(tmp_path, {"p.weight": ("F8_E4M3", CODES), "p.weight_scale_inv": ("F32", SCALES),
                           "q.weight": ("F8_E4M3", CODES)})
    with weights.CheckpointReader(tmp_path) as reader:
        with pytest.raises(weights.LayoutError, match="without p.scales.*p.weight_scale_inv"):
            weights.read_projection(reader, "p", scheme)
        with pytest.raises(weights.LayoutError, match="without q.scales"):
            weights.read_projection(reader, "q", scheme)


def test_codes_as_bytes_without_scales_are_refused_under_fp8_block(tmp_path):
    _checkpoint(tmp_path, {"p.weight": ("U8", CODES)})
    with weights.CheckpointReader(tmp_path) as reader:
        with pytest.raises(weights.LayoutError, match="without p.scales"):
            weights.read_projection(reader, "p", FP8)


def test_codes_are_read_only_where_scales_are(tmp_path):
    """Any other read of an F8_E4M3 tensor is refused, as of every type that
    the reader does not know."""
    _checkpoint(tmp_path, {"p.weight": ("F8_E4M3", CODES), "p.scales": ("F32", SCALES), "u.weight": ("U8", CODES),
                           "u.scales": ("F32", SCALES), "f.weight": ("F32", SCALES)})
    with weights.CheckpointReader(tmp_path) as reader:
        for name in ("p", "u"):
            got = weights.read_projection(reader, name, FP8)
            assert got.quant == FP8 and (got.tensors["weight"].float() == 1).all()
            assert np.array_equal(got.tensors["scales"].numpy(), SCALES)
        with pytest.raises(ValueError, match="unsupported safetensors dtype"):
            reader.read_tensor("p.weight")
        with pytest.raises(ValueError, match="holds no e4m3 codes"):
            reader.read_tensor("f.weight", codes=True)
        with pytest.raises(ValueError):
            weights.read_projection(reader, "p", AFFINE)


def test_plain_projections_beside_fp8_block_ones_stay_plain(tmp_path):
    dense = np.arange(12, dtype=np.float32).reshape(3, 4)
    _checkpoint(tmp_path, {"p.weight": ("F32", dense)})
    with weights.CheckpointReader(tmp_path) as reader:
        got = weights.read_projection(reader, "p", FP8)
    assert got.quant is None and torch.equal(got.tensors, torch.tensor(dense))


def test_a_layer_of_such_a_checkpoint_is_refused(tmp_path):
    """What `Qwen3_5LinearAttention` would have widened and multiplied without
    scales."""
    prefix = "language_model.model.layers.0.linear_attn"
    shapes = {"in_proj_qkv": 256, "in_proj_z": 128, "in_proj_a": 2, "in_proj_b": 2, "out_proj": 128}
    tensors = {}
    for p, n in shapes.items():
        tensors[f"{prefix}.{p}.weight"] = ("F8_E4M3", np.full((n, 128), 0x38, np.uint8))
        tensors[f"{prefix}.{p}.weight_scale_inv"] = ("F32", np.full((-(-n // 128), 1), 1e-3, np.float32))
    _checkpoint(tmp_path, tensors)
    config = {"linear_num_key_heads": 1, "linear_num_value_heads": 2, "linear_key_head_dim": 64,
              "linear_value_head_dim": 64, "linear_conv_kernel_dim": 4,
              "quantization_config": {"bits": 8, "group_size": 128, "mode": "fp8_block"}}
    with pytest.raises(weights.LayoutError, match="in_proj_qkv.*weight_scale_inv"):
        weights.load_linear_attention(tmp_path, 0, device="cpu", hf_config=config)
