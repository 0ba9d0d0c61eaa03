"""The bits that add_low_rank keeps of its inner product.

x A^T is made exact: x holds 8 (float16: 11) bits of a number in each of its first
values and A is ones, so the sum is the number in any order. A second rank holds all
but the number's last part, and B takes one from the other: what is left is that
part, exactly, if the inner product has kept it, and the result is the part's
own bits."""

from __future__ import annotations

import pytest
import torch

import mlx_lean_moe_amd as gdn

pytestmark = pytest.mark.gpu

# bits of a part, parts: bfloat16 and float32 keep float32's 24 bits, float16 22
PARTS = {torch.bfloat16: (8, 3), torch.float16: (11, 2), torch.float32: (8, 3)}


@pytest.mark.parametrize("dtype", PARTS)
@pytest.mark.parametrize("rank", [2, 16, 30, 48, 64, 100])
@pytest.mark.parametrize("M", [1, 40, 5000])
def test_the_last_bits_of_the_inner_product(gpu, dtype, rank, M):
    bits, parts = PARTS[dtype]
    g = torch.Generator(device=gpu)
    g.manual_seed(M + rank)
    whole = torch.randint(1 << (bits - 1), 1 << bits, (M, parts), generator=g, device=gpu).double()
    step = 2.0 ** -bits
    x = torch.zeros(M, 40, device=gpu, dtype=dtype)
    x[:, 3:3 + parts] = (whole * step ** torch.arange(1, parts + 1, device=gpu, dtype=torch.float64)).to(dtype)
    A, B = torch.zeros(rank, 40, device=gpu, dtype=dtype), torch.zeros(70, rank, device=gpu, dtype=dtype)
    A[rank - 2:, 3:3 + parts] = 1
    A[rank - 1, 2 + parts] = 0
    sign = torch.where(torch.arange(70, device=gpu) % 3 == 0, -1.0, 1.0).to(dtype)
    B[:, rank - 2], B[:, rank - 1] = sign, -sign
    y = torch.zeros(M, 70, device=gpu, dtype=dtype)
    gdn.add_low_rank(y, x, gdn.LowRankAdapters([[(A, B, 1.0)]]), gdn.AdapterRows([0] * M, 1, device=gpu))
    last = whole[:, -1:] * step ** parts
    assert torch.equal(y.double(), last * sign.double())
