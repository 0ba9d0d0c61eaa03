"""MI355X-native gated-delta linear attention.

A drop-in for the gated-delta path of ``mlx-lean-moe``
(``src/mlx_lean_moe/model/qwen3_5/{gated_delta,linear_attention}.py``,
``src/mlx_lean_moe/cache/recurrent_cache.py``): the same Python surface over
hand-written HIP kernels for gfx950 in ``libgdn.so`` (C ABI in
``include/gdn.h``). Importable as ``mlx_lean_moe_amd``.
"""

from .config import QWEN3_5_LINEAR, LinearAttentionDims, StateSpaceDims
from .gated_delta import (beta_gate, forget_gate, gated_delta_scan, gated_delta_step,
                          gated_delta_update)
from .linear_attention import (DecodeGraph, PrefillGraph, Qwen3_5LinearAttention, conv_frontend,
                               fused_decode_step, fused_prefill_ok, gated_rms_norm, prefill_fused)
from .low_rank import AdapterRows, LowRankAdapters, add_low_rank
from .norm import rms_norm
from .quant import LinearWeights, QuantizedRows, QuantScheme, dequantize, quantized_linear
from .recurrent_cache import RecurrentCache, RecurrentStatePool
from .state_space import PackedRuns, conv_silu, selective_scan, selective_step

__all__ = [
    "AdapterRows",
    "DecodeGraph",
    "PrefillGraph",
    "LinearAttentionDims",
    "LinearWeights",
    "LowRankAdapters",
    "PackedRuns",
    "QuantScheme",
    "QuantizedRows",
    "QWEN3_5_LINEAR",
    "Qwen3_5LinearAttention",
    "RecurrentCache",
    "RecurrentStatePool",
    "StateSpaceDims",
    "add_low_rank",
    "beta_gate",
    "conv_frontend",
    "conv_silu",
    "dequantize",
    "forget_gate",
    "fused_decode_step",
    "fused_prefill_ok",
    "gated_delta_scan",
    "gated_delta_step",
    "gated_delta_update",
    "gated_rms_norm",
    "prefill_fused",
    "quantized_linear",
    "rms_norm",
    "selective_scan",
    "selective_step",
]
