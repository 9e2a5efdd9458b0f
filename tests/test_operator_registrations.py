"""torch.ops.dartkv: what the fakes say of prompts and block caches is what the operators give."""

from __future__ import annotations

import pytest
import torch

import dartkv_amd as dart  # noqa: F401  (registers the operators)

DEV = "cuda"


def _layouts(device):
    """Queries of layouts that a program has: [B, H, T, D] whole, tokens first, and the last dimension not the inner one."""
    x = torch.empty(2, 4, 64, 67, dtype=torch.bfloat16, device=device)
    return [torch.empty(2, 4, 67, 64, dtype=torch.bfloat16, device=device),
            torch.empty(2, 67, 4, 64, dtype=torch.bfloat16, device=device).transpose(1, 2),
            x.transpose(2, 3), x[..., 3:].transpose(2, 3),
            torch.empty(1, 4, 67, 64, dtype=torch.bfloat16, device=device).expand(2, -1, -1, -1)]


@pytest.mark.gpu
@pytest.mark.parametrize("which", range(5))
def test_prompt_fake_has_the_operators_strides(which):
    from torch._subclasses.fake_tensor import FakeTensorMode
    q = _layouts(DEV)[which].normal_() if which < 4 else _layouts(DEV)[which]
    kv = [torch.randn(2, 2, 67, 64, dtype=torch.float32, device=DEV).to(torch.bfloat16) for _ in range(2)]
    got = torch.ops.dartkv.prompt_attention(q, *kv)
    with FakeTensorMode() as mode:
        fake = torch.ops.dartkv.prompt_attention(*(mode.from_tensor(t) for t in (q, *kv)))
    assert fake.shape == got.shape and fake.stride() == got.stride() and fake.dtype == got.dtype


@pytest.mark.gpu
def test_opcheck_of_a_prompt_whose_last_dimension_is_not_the_inner_one():
    q = torch.randn(2, 4, 64, 67, device=DEV).to(torch.bfloat16).transpose(2, 3)
    torch.library.opcheck(torch.ops.dartkv.prompt_attention.default, (q, q[:, :2], q[:, 2:]))


def test_prompt_fake_strides_on_meta_tensors():
    for q in _layouts("meta"):
        fake = torch.ops.dartkv.prompt_attention(q, q[:, :2], q[:, 2:])
        assert fake.stride(-1) == 1 and fake.shape == q.shape
