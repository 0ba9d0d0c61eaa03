"""rms_norm's and the code product's refusals, without a GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

import mlx_lean_moe_amd as gdn
from mlx_lean_moe_amd import _lib

P = lambda i: ctypes.c_void_p((1 << 32) + (i << 28))  # distinct, aligned, never dereferenced


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="ROCm"):
        gdn.rms_norm(torch.zeros(2, 8), torch.ones(8), 1e-6)
    with pytest.raises(ValueError):
        gdn.rms_norm(torch.zeros(()), None, 1e-6)


def test_norm_argument_checks():
    lib = _lib.load()
    err = lambda: lib.gdn_last_error().decode()

    def call(**over):
        a = dict(x=P(0), xs=96, r=P(1), rs=96, s=P(2), ss=96, w=P(3), eps=1e-6, dt=1, out=P(4), codes=P(5), sc=P(6), ld=256,
                 rows=4, K=96)
        a.update(over)
        return lib.gdn_rms_norm(*a.values(), None)

    assert call(rows=0) == 0
    for over, what in [(dict(K=0), "sizes"), (dict(rows=-1), "sizes"), (dict(dt=3), "dtype"), (dict(x=None), "null"),
                       (dict(out=None, codes=None), "null"), (dict(s=None), "sum"), (dict(r=None), "sum"),
                       (dict(xs=95), "width"), (dict(rs=95), "width"), (dict(ss=95), "width"),
                       (dict(s=ctypes.c_void_p((1 << 32) + 16)), "overlaps x"),
                       (dict(s=P(0), ss=97, xs=96), "overlaps x"),
                       (dict(s=ctypes.c_void_p((1 << 32) + (1 << 28) + 96 * 2)), "overlaps residual"),
                       (dict(K=90), "multiple of 16"), (dict(sc=None), "scales"), (dict(ld=3), "apart"),
                       (dict(codes=ctypes.c_void_p(8)), "aligned")]:
        assert call(**over) == _lib.GDN_EINVAL and what in err(), (over, err())


def test_code_product_argument_checks():
    lib = _lib.load()
    err = lambda: lib.gdn_last_error().decode()
    assert lib.gdn_fp8_matmul_codes_workspace_size(1, 16, 64, 2048) == 0
    need = lib.gdn_fp8_matmul_codes_workspace_size(1, 200, 2048, 4096)
    assert 0 < need < lib.gdn_fp8_matmul_workspace_size(1, 200, 2048, 4096)
    assert lib.gdn_fp8_matmul_codes_workspace_size(1, 200, 2048, 4097) == 0

    def call(**over):
        a = dict(codes=P(0), rs=P(1), ld=256, w=P(2), sc=P(3), y=P(4), dt=1, res=None, M=200, N=2048, K=4096, ws=P(5), wsb=need)
        a.update(over)
        return lib.gdn_fp8_matmul_codes(*a.values(), None)

    assert call(M=0) == 0
    for over, what in [(dict(K=4104), "sizes"), (dict(dt=3), "dtype"), (dict(rs=None), "null"), (dict(ld=255), "apart"),
                       (dict(ld=128), "apart"), (dict(codes=ctypes.c_void_p(8)), "aligned"),
                       (dict(wsb=need - 1), "workspace"), (dict(ws=None), "workspace")]:
        assert call(**over) == _lib.GDN_EINVAL and what in err(), (over, err())
