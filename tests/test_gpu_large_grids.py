"""Calls of more threads than one grid dimension holds (2^32), checked in blocks
over the whole output."""

from __future__ import annotations

import pytest
import torch

import mlx_lean_moe_amd as gdn
from .scan64 import scan64

pytestmark = pytest.mark.gpu

FP8 = gdn.QuantScheme(8, 128, "fp8_block")


@pytest.fixture(autouse=True)
def _return_memory():
    yield
    torch.cuda.empty_cache()


def _needs(gpu, gib):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info(gpu)[0] < gib << 30:
        pytest.skip(f"needs {gib} GiB of device memory")


def test_step_of_2_to_the_23_heads(gpu):
    """131 073 sequences of 64 heads, a workgroup of 512 threads a head."""
    _needs(gpu, 16)
    B, H, P, N, K = (1 << 17) + 1, 64, 8, 8, 2
    d = gdn.StateSpaceDims(1, H, N, P, K)
    g = torch.Generator(device=gpu)
    g.manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, device=gpu)
    xbc, dt, conv, ssm = r(B, d.conv_dim), r(B, H), torch.zeros(B, K - 1, d.conv_dim, device=gpu), r(B, H, P, N)
    A_log, dt_bias, D = torch.zeros(H, device=gpu), torch.zeros(H, device=gpu), r(H)
    weight = torch.cat([torch.zeros(d.conv_dim, 1), torch.ones(d.conv_dim, 1)], 1).to(gpu)  # the token itself
    y, _, S = gdn.selective_step(xbc, dt, conv, ssm, weight, None, A_log, dt_bias, D, d)
    assert torch.isfinite(y).all()
    for b0 in (0, 1, B // 2 - 3, (1 << 15) - 2, (1 << 17) - 4, B - 5):
        at = slice(b0, b0 + 5)
        u = xbc[at].double()
        u = (u / (1 + torch.exp(-u))).split([H * P, N, N], dim=1)
        ref, state, ya, sa = scan64(u[0].view(5, H, P), dt[at], u[1].view(5, 1, N), u[2].view(5, 1, N), A_log, dt_bias,
                                    D, ssm[at], [1] * 5)
        # three operands of SiLU, each within 8 + 4 |u| < 32 roundings, and N + 40 more
        tol = (3 * 32 + N + 40) * 2.0 ** -24
        assert ((y[at].double() - ref).abs() <= tol * ya + 1e-30).all(), b0
        assert ((S[at].double() - state).abs() <= tol * sa + 1e-30).all(), b0


def test_fp8_rows_of_2_to_the_28_groups(gpu):
    """2^28 rows of 16 columns, 16 rows a workgroup of 256 threads: 2^32."""
    _needs(gpu, 80)
    M, K = 1 << 28, 16
    x = torch.zeros(M, K, dtype=torch.bfloat16, device=gpu)
    x[:, 0] = (torch.arange(M, device=gpu, dtype=torch.int32) % 251 - 125).bfloat16()
    W = {"weight": torch.ones(1, K, device=gpu).to(torch.float8_e4m3fn), "scales": torch.ones(1, 1, device=gpu)}
    y = gdn.quantized_linear(x, W, FP8)
    # a row of one value: its code is +-448 under a scale of |x| / 448, so the row
    # gives x but for that quotient's rounding, which bfloat16 takes back
    step = 1 << 24
    for m in range(0, M, step):
        assert torch.equal(y[m:m + step, 0], x[m:m + step, 0]), m


def test_fp8_one_row_of_2_to_the_28_outputs(gpu):
    """64 outputs a workgroup of 1024 threads, and some more than 2^32 threads."""
    _needs(gpu, 16)
    N, K = (1 << 28) + 70, 16
    w = torch.zeros(N, K, dtype=torch.uint8, device=gpu)
    w[:, 3] = (torch.arange(N, device=gpu, dtype=torch.int32) % 119).to(torch.uint8)
    x = torch.zeros(1, K, dtype=torch.bfloat16, device=gpu)
    x[0, 3] = 448.0
    scales = torch.full((-(-N // 128), 1), 2.0 ** -4, device=gpu)
    y = gdn.quantized_linear(x, {"weight": w, "scales": scales}, FP8)
    step = 1 << 24
    for n in range(0, N, step):
        want = w[n:n + step, 3].contiguous().view(torch.float8_e4m3fn).float() * 28
        assert torch.equal(y[0, n:n + step], want.bfloat16()), n


def test_dequantize_of_2_to_the_36_codes(gpu):
    _needs(gpu, 200)
    N, K = 1 << 21, 1 << 15
    w = torch.empty(N, K, dtype=torch.uint8, device=gpu)
    row = (torch.arange(K, device=gpu, dtype=torch.int32) * 7 % 120).to(torch.uint8)
    for n in range(0, N, 1 << 16):
        w[n:n + (1 << 16)] = row
    w[:, 5] = (torch.arange(N, device=gpu, dtype=torch.int32) % 119).to(torch.uint8)
    scales = torch.rand(N // 128, K // 128, device=gpu) + 0.5
    out = gdn.dequantize({"weight": w, "scales": scales}, FP8, torch.bfloat16)
    for n0 in range(0, N, N // 32):
        for n in (n0, n0 + N // 32 - 8):
            codes = w[n:n + 8].view(torch.float8_e4m3fn).float()
            s = scales[n // 128:n // 128 + 1].repeat_interleave(128, 1)
            assert torch.equal(out[n:n + 8], (codes * s).bfloat16()), n


def test_gates_of_2_to_the_32_elements(gpu):
    _needs(gpu, 40)
    rows, H = (1 << 26) + 3, 64
    a = (torch.arange(rows, device=gpu, dtype=torch.int32) % 61 - 30).bfloat16()[:, None].expand(rows, H).contiguous()
    A_log, dt_bias = torch.linspace(-3, 2, H, device=gpu), torch.linspace(-1, 1, H, device=gpu)
    g = gdn.forget_gate(a, A_log, dt_bias)
    want = gdn.forget_gate(a[:61], A_log, dt_bias)
    for r0 in (0, rows // 61 // 2 * 61, (rows // 61 - 1) * 61):
        assert torch.equal(g[r0:r0 + 61], want), r0
    assert torch.equal(g[-3:], gdn.forget_gate(a[-3:], A_log, dt_bias))


def test_gated_norm_of_2_to_the_26_rows(gpu):
    """A wave a row: 2^32 threads and some more."""
    _needs(gpu, 16)
    rows, D = (1 << 26) + 5, 8
    x = (torch.arange(rows, device=gpu, dtype=torch.int32) % 97 - 48).bfloat16()[:, None].expand(rows, D).contiguous()
    z = x.flip(0).contiguous()
    w = torch.linspace(0.5, 1.5, D, device=gpu)
    y = gdn.gated_rms_norm(x, z, w, 1e-6)
    for r0 in (0, rows // 2 - 50, rows - 100):
        assert torch.equal(y[r0:r0 + 100], gdn.gated_rms_norm(x[r0:r0 + 100], z[r0:r0 + 100], w, 1e-6)), r0


def test_dequantize_of_2_to_the_32_words(gpu):
    """8-bit affine codes, a word of four a thread: 2^32 threads and some more."""
    _needs(gpu, 80)
    N, K, gs = (1 << 20) + 16, 1 << 14, 128
    w = torch.randint(-2 ** 31, 2 ** 31 - 1, (N, K // 4), dtype=torch.int32, device=gpu)
    s = torch.rand(N, K // gs, device=gpu).bfloat16()
    out = gdn.dequantize({"weight": w, "scales": s, "biases": s}, gdn.QuantScheme(8, gs), torch.bfloat16)
    shifts = torch.arange(0, 32, 8, device=gpu, dtype=torch.int32)
    for n in (0, 5, N // 2, N - (1 << 16), N - 8):
        q = ((w[n:n + 8, :, None] >> shifts) & 255).reshape(8, K).float()
        sc = s[n:n + 8].float().repeat_interleave(gs, 1)
        assert torch.equal(out[n:n + 8], torch.addcmul(sc, sc, q).bfloat16()), n
