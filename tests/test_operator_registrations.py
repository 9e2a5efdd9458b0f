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


def _pool(device=DEV):
    return [torch.zeros(4, 2, 16, 64, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn) for _ in range(2)] + \
        [torch.ones(4, 2, device=device) for _ in range(2)]


@pytest.mark.gpu
def test_append_operator_reports_what_is_not_finite():
    x = torch.randn(3, 2, 64, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(DEV)
    flag, pool = torch.zeros(1, dtype=torch.int32, device=DEV), _pool()
    slots = torch.arange(3, device=DEV)
    torch.ops.dartkv.append_blocks(x, x, slots, *pool)
    torch.ops.dartkv.append_blocks_reported(x, x, slots, *pool, flag)
    assert int(flag) == 0
    x[1, 0, 5] = float("inf")
    append = torch.compile(lambda *a: torch.ops.dartkv.append_blocks_reported(*a), backend="aot_eager", fullgraph=True)
    append(x, x, slots, *pool, flag)
    assert int(flag) == 1


def _tables():
    i32 = dict(dtype=torch.int32, device=DEV)
    return (torch.full((2, 2), -1, **i32), torch.zeros(2, **i32), torch.arange(3, -1, -1, **i32), torch.tensor([4, 0, 0, 0], **i32))


@pytest.mark.gpu
def test_opcheck_of_the_block_operators():
    """The operators that change their arguments, and the attention over what they leave."""
    ops, check = torch.ops.dartkv, torch.library.opcheck
    x = torch.randn(21, 2, 64, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(DEV)
    q = torch.randn(21, 4, 64, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(DEV)
    tokens = torch.tensor([20, 1], dtype=torch.int32, device=DEV)
    check(ops.reserve_blocks.default, (*_tables(), tokens, 21, 16))
    tables, pool = _tables(), _pool()
    slots, starts = ops.reserve_blocks(*tables, tokens, 21, 16)
    check(ops.release_blocks.default, (*(t.clone() for t in tables), tokens, 16))
    check(ops.release_blocks.default, (*(t.clone() for t in tables), None, 16))
    ops.append_blocks(x, x.flip(0), slots, *pool)
    # (the schema test compares arguments with an operation that torch has not for fp8)
    rest = ("test_autograd_registration", "test_faketensor")
    flag = torch.zeros(1, dtype=torch.int32, device=DEV)
    check(ops.append_blocks.default, (x, x, slots, *_pool()), test_utils=rest)
    check(ops.append_blocks_reported.default, (x, x, slots, *_pool(), flag), test_utils=rest)
    rest += ("test_aot_dispatch_dynamic",)
    check(ops.block_attention.default, (q, *pool, tables[0], tables[1], starts), test_utils=rest)
    check(ops.block_attention.default, (q[:2], *pool, tables[0], tables[1], None, 1, 0.1), test_utils=rest)
