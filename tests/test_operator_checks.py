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
