"""torch.ops.dartkv: derivatives that an operator does not have are refused, not left out."""

from __future__ import annotations

import pytest
import torch

import dartkv_amd as dart  # noqa: F401  (registers the operators)

DEV = "cuda"


def _rotation():
    x = torch.randn(5, 4, 64, device=DEV)
    cos, sin = torch.rand(5, 32, device=DEV), torch.rand(5, 32, device=DEV)
    return x, x[:, :2].contiguous(), cos, sin


@pytest.mark.gpu
@pytest.mark.parametrize("which", [2, 3])
def test_angles_that_require_gradients_are_refused(which):
    args = list(_rotation())
    args[which].requires_grad_()
    for first in (False, True):
        args[0].requires_grad_(first)
        with pytest.raises(RuntimeError, match="cos and sin"):
            torch.ops.dartkv.rotate_heads(*args)
        with torch.no_grad():
            torch.ops.dartkv.rotate_heads(*args)
