"""What the operators for requests of different lengths refuse, whatever calls came before."""

from __future__ import annotations

import pytest
import torch

DEV = "cuda"


@pytest.mark.gpu
def test_key_starts_alone_are_refused_every_time():
    import dartkv_amd as dart
    q = torch.zeros(2, 4, 8, 64, dtype=torch.bfloat16, device=DEV)
    starts = torch.tensor([0, 8], dtype=torch.int32, device=DEV)
    for _ in range(2):
        with pytest.raises(ValueError, match="key_starts needs query_starts"):
            dart.prompt_attention(q, q[:, :2], q[:, 2:], None, starts)
        dart.prompt_attention(q, q[:, :2], q[:, 2:])
    with pytest.raises(TypeError, match="starts"):
        dart.prompt_attention(q[0].transpose(0, 1), q[0].transpose(0, 1), q[0].transpose(0, 1), [0, 8])


def test_forward_mode_tangents_are_refused():
    import torch.autograd.forward_ad as forward
    from dartkv_amd.prompt import no_gradients
    x = torch.zeros(3)
    with forward.dual_level():
        dual = forward.make_dual(x, torch.ones(3))
        with pytest.raises(RuntimeError, match="no backward pass"):
            no_gradients("prompt_attention", x, dual.view(3, 1))
        no_gradients("prompt_attention", x)
    no_gradients("prompt_attention", x)
