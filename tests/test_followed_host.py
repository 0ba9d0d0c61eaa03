"""Calls that autograd or forward mode follows are refused by the operators
that take no part in either (no GPU)."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from mlx_lean_moe_amd import quant, state_space


def test_tangents_are_refused():
    a, b = torch.zeros(3), torch.ones(3)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(a, b)
        for mode in (torch.enable_grad, torch.no_grad):
            with mode():
                with pytest.raises(RuntimeError, match="forward mode"):
                    state_space._no_gradient(b, None, dual)
                state_space._no_gradient(a, b, None)
                assert quant._followed(a, None, dual) and not quant._followed(a, b)
    state_space._no_gradient(a, b)


def test_gradients_are_refused_of_any_operand():
    a, leaf = torch.zeros(3), torch.zeros(3, requires_grad=True)
    with pytest.raises(RuntimeError, match="no gradient"):
        state_space._no_gradient(a, None, leaf * 2)
    assert quant._followed(a, leaf)
    with torch.no_grad():
        state_space._no_gradient(a, leaf)
        assert not quant._followed(a, leaf)
