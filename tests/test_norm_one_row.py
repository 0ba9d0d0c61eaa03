"""The sum of one row written over its input: the distance to a next row, which there
is not, does not matter."""

from __future__ import annotations

import ctypes

import pytest
import torch

import mlx_lean_moe_amd as gdn
from mlx_lean_moe_amd import _lib, norm

P = lambda i, more=0: ctypes.c_void_p((1 << 32) + (i << 28) + more)  # distinct, aligned, never dereferenced


def test_one_row_under_another_stride_is_itself():
    buf = torch.zeros(4, 96)
    x = buf[:1]
    for other in (buf.as_strided((1, 96), (1000, 1)), x.as_strided((1, 96), (96, 1)), buf[::2][:1]):
        norm._check_sum(other, 96, x, 96, "x")
        norm._check_sum(x, 96, other, 96, "x")
    for other in (buf.view(-1)[1:97].view(1, 96), buf.view(-1)[95:191].view(1, 96)):
        with pytest.raises(ValueError, match="overlap"):
            norm._check_sum(other, 96, x, 96, "x")
    norm._check_sum(buf[1:2], 96, x, 96, "x")
    # several rows: another stride is another place
    with pytest.raises(ValueError, match="overlap"):
        norm._check_sum(buf.as_strided((2, 96), (192, 1)), 192, buf[:2], 96, "x")


def test_one_row_at_the_c_boundary():
    lib = _lib.load()
    err = lambda: lib.gdn_last_error().decode()

    def call(**over):
        a = dict(x=P(0), xs=96, r=P(1), rs=96, s=P(2), ss=96, w=P(3), eps=1e-6, dt=1, out=P(4), codes=ctypes.c_void_p(8), sc=P(6),
                 ld=256, rows=1, K=96)
        a.update(over)
        assert lib.gdn_rms_norm(*a.values(), None) == _lib.GDN_EINVAL  # (the codes' alignment, looked at last)
        return err()

    for over in (dict(s=P(0), ss=97), dict(s=P(0), ss=96), dict(s=P(1), ss=200), dict(s=P(0, 192)), dict(x=P(1), s=P(1), ss=500)):
        assert "aligned" in call(**over), (over, err())
    assert "overlaps x" in call(s=P(0, 2)) and "overlaps x" in call(s=P(0, 190), ss=97)
    assert "overlaps residual" in call(s=P(1, 2))
    assert "overlaps x" in call(s=P(0), ss=97, rows=2)


@pytest.mark.gpu
@pytest.mark.parametrize("act", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("K", [96, 2048, 16400])
def test_one_row_in_place(gpu, act, K):
    g = torch.Generator(device=gpu)
    g.manual_seed(0)
    r = lambda: torch.randn(1, K, generator=g, device=gpu).to(act)
    x, res, w = r(), r(), torch.rand(K, generator=g, device=gpu)
    want, stream = gdn.rms_norm(x, w, 1e-6, residual=res)
    for which in ("x", "residual"):
        xc, rc = x.clone(), res.clone()
        own = (xc if which == "x" else rc).as_strided((1, K), (5 * K + 3, 1))
        got, out = gdn.rms_norm(xc, w, 1e-6, residual=rc, sum_out=own)
        assert out is own and torch.equal(got, want) and torch.equal(own, stream)
