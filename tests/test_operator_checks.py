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


@pytest.mark.gpu
def test_appends_refuse_gradients():
    import dartkv_amd as dart
    pool = [torch.zeros(2, 1, 16, 32, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn) for _ in range(2)] + \
        [torch.ones(2, 1, device=DEV) for _ in range(2)]
    x = torch.ones(3, 1, 32, dtype=torch.bfloat16, device=DEV)
    grad = torch.ones_like(x).requires_grad_()
    slots = torch.arange(3, device=DEV)
    for _ in range(2):
        for k, v in ((grad, x), (x, grad)):
            with pytest.raises(RuntimeError, match="no backward pass"):
                dart.append_blocks(k, v, slots, *pool)
        dart.append_blocks(x, x, slots, *pool)
    with torch.no_grad():
        dart.append_blocks(grad, grad, slots, *pool)


@pytest.mark.gpu
def test_plans_of_another_cache_are_refused():
    import dartkv_amd as dart
    one, other = (dart.BlockKVCache(2, 8, 1, 64, block_size=16) for _ in range(2))
    x = torch.ones(2, 1, 64, dtype=torch.bfloat16, device=DEV)
    tokens = torch.ones(2, dtype=torch.int32, device=DEV)
    mine, others = one.reserve(tokens, 2), other.reserve(tokens, 2)
    for call in (lambda: one.append(0, x, x, others), lambda: one.attention(0, x, others)):
        with pytest.raises(ValueError, match="another cache"):
            call()
    one.append(0, x, x, mine)
    assert torch.equal(one.attention(0, x, mine), x)


def test_counts_and_starts_past_31_bits_do_not_wrap():
    from dartkv_amd.prompt import int32_vector
    most = 2 ** 31 - 1
    got = int32_vector(torch.tensor([0, 5, 2 ** 32 + 1, -2 ** 32 + 7, 2 ** 31, most]), "tokens", torch.device("cpu"))
    assert got.dtype == torch.int32 and got.tolist() == [0, 5, most, -2 ** 31, most, most]


@pytest.mark.gpu
def test_a_count_past_31_bits_is_reported():
    import dartkv_amd as dart
    cache = dart.BlockKVCache(2, 8, 1, 64, block_size=16)
    plan = cache.reserve(torch.tensor([2 ** 32 + 1, 1], device=DEV), 2)
    assert plan.slots.tolist() == [-1, -1] and cache.lengths.tolist() == [0, 0]
    with pytest.raises(RuntimeError, match="more new tokens than total"):
        cache.check()


@pytest.mark.parametrize("scale", [1e-46, 1e-300, 1e-39])
def test_scales_that_vanish_in_fp32_are_refused(scale):
    """With a factor of 0 the masked logits would be -inf * 0."""
    from dartkv_amd import _lib
    from dartkv_amd.prompt import scale_factor
    with pytest.raises(ValueError, match="scale"):
        scale_factor(scale, 64, "prompt_attention")
    assert scale_factor(1e-37, 64, "prompt_attention") == 1e-37
    a = _lib.PromptAttentionArgs(query=256, keys=256, values=256, out=256, requests=1, Hq=4, Hkv=2, D=64, q_tokens=8,
                                 k_tokens=8, dtype=2, scale=scale, causal=1)
    b = _lib.BlockAttentionArgs(query=256, out=256, dtype=2, q_st=128, q_sh=32, o_st=128, o_sh=32, tokens=4, starts=256,
                                table=256, lengths=256, requests=2, max_blocks=4, blocks=8, block_size=16, key_codes=256,
                                value_codes=256, key_scale=256, value_scale=256, Hq=4, Hkv=2, D=32, scale=scale,
                                max_tokens=4, workspace=256, workspace_bytes=1 << 40)
    lib = _lib.load()
    for entry, args in ((lib.dkv_prompt_attention, a), (lib.dkv_block_attention, b)):
        assert entry(args, None) == 1 and "scale" in lib.dkv_last_error().decode()


@pytest.mark.gpu
def test_outputs_whose_rows_share_memory_are_refused():
    import dartkv_amd as dart
    q = torch.zeros(6, 4, 64, dtype=torch.bfloat16, device=DEV)
    starts = torch.tensor([0, 6], dtype=torch.int32, device=DEV)
    codes = [torch.zeros(2, 2, 16, 64, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn) for _ in range(2)]
    scales = [torch.ones(2, 2, device=DEV) for _ in range(2)]
    table, lengths = torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.full((1,), 6, dtype=torch.int32, device=DEV)
    calls = (lambda out: dart.prompt_attention(q, q[:, :2], q[:, 2:], starts, out=out),
             lambda out: dart.block_attention(q, *codes, *scales, table, lengths, starts, out=out))
    for call in calls:
        for out in (q.new_zeros(6, 1, 64).expand(-1, 4, -1), q.new_zeros(1, 4, 64).expand(6, -1, -1)):
            with pytest.raises(ValueError, match="rows of its own"):
                call(out)
        call(torch.empty_like(q))
    one = q.new_zeros(64).expand(1, 1, 64)  # (one row: its strides say nothing)
    dart.prompt_attention(q[:1, :1], q[:1, :1], q[:1, :1], torch.tensor([0, 1], dtype=torch.int32, device=DEV), out=one)
