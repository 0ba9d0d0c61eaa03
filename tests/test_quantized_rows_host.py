"""QuantizedRows made by hand: what its products would read out of range, or as other
values, is refused when it is made (no GPU)."""

from __future__ import annotations

import pytest
import torch

import mlx_lean_moe_amd as gdn

BF16 = torch.bfloat16
NBYTES = gdn.QuantizedRows.nbytes(3, 144)


def _data(n=NBYTES, dtype=torch.uint8):
    return torch.zeros(n, dtype=dtype)


def test_codes_and_scales_lie_where_the_layout_says():
    data = _data()
    codes = data[:3 * 256].view(3, 256)
    codes[:, :144] = torch.arange(3 * 144).remainder(120).view(3, 144).to(torch.uint8)  # (0x78 and more: past 256)
    scales = data[3 * 256:].view(torch.float32).view(2, 256)
    scales[:, :3] = torch.tensor([[1.0, 2.0, 3.0], [4.0, 5.0, 6.0]])
    rows = torch.zeros(3, 144, dtype=BF16)
    q = gdn.QuantizedRows((3, 144), BF16, data, rows)
    assert q.shape == (3, 144) and q.dtype is BF16 and q.rows is rows
    assert torch.equal(q.scales, torch.tensor([[1.0, 4.0], [2.0, 5.0], [3.0, 6.0]]))
    assert torch.equal(q.codes.float(), codes[:, :144].view(torch.float8_e4m3fn).float())
    assert torch.equal(q.dequantize()[1, 128:], q.codes[1, 128:].float() * 5)
    flat = gdn.QuantizedRows((1, 3, 144), BF16, data, rows.view(1, 3, 144)).reshape(3, 144)
    assert flat.rows.shape == (3, 144) and torch.equal(flat.scales, q.scales)
    assert gdn.QuantizedRows((0, 144), BF16, _data(0)).codes.shape == (0, 144)
    assert gdn.QuantizedRows((16,), torch.float32, _data(gdn.QuantizedRows.nbytes(1, 16))).scales.shape == (1,)


@pytest.mark.parametrize("shape,dtype,data,rows", [
    ((3, 144), BF16, _data(NBYTES - 1), None),  # too short
    ((3, 144), BF16, _data(NBYTES + 1), None),
    ((3, 144), BF16, _data(3 * 256), None),  # no scales
    ((300, 144), BF16, _data(), None),  # of fewer rows
    ((3, 272), BF16, _data(), None),  # of narrower rows
    ((3, 144), BF16, _data(NBYTES, torch.int8), None),
    ((3, 144), BF16, _data(NBYTES // 4, torch.float32), None),
    ((3, 144), BF16, _data(2 * NBYTES)[::2], None),  # not one after the other
    ((3, 144), BF16, _data(NBYTES + 16)[8:-8], None),  # not where 16 bytes start
    ((3, 144), BF16, _data(2 * NBYTES).view(2, -1), None),
    ((3, 150), BF16, _data(), None),  # no multiple of 16
    ((3, 0), BF16, _data(), None),
    ((), BF16, _data(), None),
    ((-3, 144), BF16, _data(), None),
    ((3, 144), torch.float64, _data(), None),
    ((3, 144), torch.uint8, _data(), None),
    ((3, 144), BF16, _data(), torch.zeros(3, 128, dtype=BF16)),
    ((3, 144), BF16, _data(), torch.zeros(3, 144)),
    ((3, 144), BF16, _data(), torch.zeros(3, 144, dtype=BF16, device="meta")),
])
def test_what_does_not_fit_is_refused(shape, dtype, data, rows):
    with pytest.raises(ValueError):
        gdn.QuantizedRows(shape, dtype, data, rows)
