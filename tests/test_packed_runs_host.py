"""Offsets of packed runs that are no whole numbers (no GPU)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import mlx_lean_moe_amd as gdn
from mlx_lean_moe_amd import state_space


@pytest.mark.parametrize("offsets", [[0, 3.7], [0.0, 3.0], torch.tensor([0.0, 2.5]), np.array([0, 3.5]), [False, True],
                                     [0, 3j]])
def test_offsets_are_whole_numbers(offsets):
    with pytest.raises(ValueError, match="whole numbers"):
        gdn.PackedRuns(offsets, device="cpu")
    with pytest.raises(ValueError, match="whole numbers"):
        state_space._runs(offsets, 3, torch.device("cpu"))


@pytest.mark.parametrize("offsets", [[0, 3, 7], (0, 3, 7), torch.tensor([0, 3, 7], dtype=torch.int32),
                                     np.array([0, 3, 7], dtype=np.int16), torch.tensor([0, 3, 7], dtype=torch.uint8)])
def test_offsets_of_any_whole_type(offsets):
    assert gdn.PackedRuns(offsets, device="cpu").offsets == (0, 3, 7)
    runs = state_space._runs(offsets, 7, torch.device("cpu"))
    assert runs.offsets == (0, 3, 7) and runs.longest == 4
    with pytest.raises(ValueError, match="token count 8"):
        state_space._runs(offsets, 8, torch.device("cpu"))
