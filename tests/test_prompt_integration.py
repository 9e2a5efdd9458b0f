"""prompt_attention in the Qwen3 adapter, and the new operators under torch.ops.dartkv."""

from __future__ import annotations

import pytest
import torch

transformers = pytest.importorskip("transformers")

import dartkv_amd as dart  # noqa: E402
from tests.test_prompt_attention import _check, _reference  # noqa: E402

DEV = "cuda"


def _model(dtype, prompt, **over):
    from dartkv_amd.integrations import attach_dart_fused_attention
    torch.manual_seed(0)
    kw = dict(vocab_size=128, hidden_size=256, intermediate_size=256, num_hidden_layers=2, num_attention_heads=4,
              num_key_value_heads=2, head_dim=64, max_position_embeddings=256, attn_implementation="sdpa",
              layer_types=["full_attention", "full_attention"])
    kw.update(over)
    model = transformers.Qwen3ForCausalLM(transformers.Qwen3Config(**kw)).to(device=DEV, dtype=dtype).eval()
    return attach_dart_fused_attention(model, prompt_attention=prompt)


def _cache():
    from dartkv_amd.integrations import DartHFCache
    return DartHFCache(dart.DartKVCacheConfig(bits=4, page_size=16, key_group_size=16, value_group_size=16, sink_tokens=4,
                                              hold_partial_pages=True, metadata_dtype=torch.float16))


@pytest.fixture
def calls(monkeypatch):
    from dartkv_amd.integrations import qwen3
    seen = []

    def record(query, keys, values, **kw):
        out = dart.prompt_attention(query, keys, values, **kw)
        seen.append((query, keys, values, kw["scale"], out))
        return out

    monkeypatch.setattr(qwen3, "prompt_attention", record)
    return seen


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_adapter_prefills_on_the_prompt_kernel(calls, dtype):
    ids = torch.randint(0, 128, (2, 37), generator=torch.Generator().manual_seed(1)).to(DEV)
    with torch.no_grad():
        want = _model(dtype, False)(ids, past_key_values=_cache(), use_cache=True).logits
        assert not calls
        model = _model(dtype, True)
        cache = _cache()
        got = model(ids, past_key_values=cache, use_cache=True).logits
        assert len(calls) == 2
        for q, k, v, scale, out in calls:
            for b in range(2):
                o, w = _reference(*(t[b].transpose(0, 1) for t in (q, k, v)), True, scale)
                _check(out[b].transpose(0, 1), o, w, dtype)
        # Both attentions are within the bound above of the same sums, so the logits differ by roundings of the two
        # layers: some steps of the type at the logits' size.
        assert float((got - want).float().norm() / want.float().norm()) < 16 * torch.finfo(dtype).eps
        model(got[:, -1:].argmax(-1), past_key_values=cache, use_cache=True)  # a decode step is not a prompt
        assert len(calls) == 2


@pytest.mark.gpu
def test_adapter_keeps_the_backend_for_other_calls(calls):
    ids = torch.randint(0, 128, (2, 12), generator=torch.Generator().manual_seed(1)).to(DEV)
    mask = torch.ones_like(ids)
    mask[0, :5] = 0
    with torch.no_grad():
        _model(torch.bfloat16, True)(ids, attention_mask=mask, past_key_values=_cache(), use_cache=True)  # padded
        _model(torch.float32, True)(ids, past_key_values=_cache(), use_cache=True)  # another type
        _model(torch.bfloat16, True, attn_implementation="eager")(ids, past_key_values=_cache(), use_cache=True)
    model = _model(torch.bfloat16, True)
    model(ids, use_cache=False).logits.float().sum().backward()  # gradients go through the backend
    assert model.model.layers[0].self_attn.q_proj.weight.grad is not None
    assert not calls


def _block_tensors():
    cache = dart.BlockKVCache(2, 8, 2, 64, block_size=16)
    x = torch.randn(40, 2, 64, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(DEV)
    plan = cache.reserve(torch.tensor([30, 10], device=DEV), 40)
    cache.append(0, x, x.flip(0), plan)
    q = torch.randn(40, 4, 64, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(DEV)
    return cache, plan, x, q


@pytest.mark.gpu
def test_operators_give_the_python_api_and_pass_opcheck():
    ops = torch.ops.dartkv
    cache, plan, x, q = _block_tensors()
    attend = (q, cache.key_codes[0], cache.value_codes[0], cache.key_scale[0], cache.value_scale[0], cache.table,
              cache.lengths, plan.starts)
    assert torch.equal(ops.block_attention(*attend, 40), dart.block_attention(*attend, max_tokens=40))
    starts = torch.tensor([0, 30, 40], dtype=torch.int32, device=DEV)
    assert torch.equal(ops.prompt_attention(q, x, x, starts), dart.prompt_attention(q, x, x, starts))
    torch.library.opcheck(ops.prompt_attention.default, (q, x, x, starts))
    batch = [t.view(2, 20, -1, 64).transpose(1, 2) for t in (q, x, x)]
    torch.library.opcheck(ops.prompt_attention.default, (*batch, None, None, True, 0.1))
    other = dart.BlockKVCache(2, 8, 2, 64, block_size=16)
    slots, begin = ops.reserve_blocks(other.table, other.lengths, other.free, other.state,
                                      torch.tensor([30, 10], device=DEV), 40, 16)
    assert torch.equal(slots, plan.slots) and torch.equal(begin, plan.starts) and torch.equal(other.table, cache.table)
    ops.append_blocks(x, x.flip(0), slots, other.key_codes[0], other.value_codes[0], other.key_scale[0],
                      other.value_scale[0])
    assert torch.equal(other.key_codes.view(torch.uint8), cache.key_codes.view(torch.uint8))
    ops.release_blocks(other.table, other.lengths, other.free, other.state, None, 16)
    assert other.lengths.tolist() == [0, 0] and int(other.state[0]) == 8


@pytest.mark.gpu
def test_prompt_operator_traces_whole_under_torch_compile():
    q = torch.randn(2, 4, 33, 64, device=DEV, dtype=torch.float16)

    def twice(t):
        return torch.ops.dartkv.prompt_attention(t, t[:, :2], t[:, 2:]) * 2

    assert torch.equal(torch.compile(twice, backend="aot_eager", fullgraph=True)(q), twice(q))


def test_fake_shapes():
    ops = torch.ops.dartkv
    q = torch.empty(2, 8, 5, 64, device="meta", dtype=torch.bfloat16)
    assert ops.prompt_attention(q, q[:, :2], q[:, :2]).shape == q.shape
    codes = torch.empty(4, 2, 16, 64, device="meta", dtype=torch.float8_e4m3fn)
    scale = torch.empty(4, 2, device="meta")
    table, lengths = (torch.empty(s, device="meta", dtype=torch.int32) for s in ((3, 2), (3,)))
    assert ops.block_attention(q[:, :, 0], codes, codes, scale, scale, table, lengths).shape == (2, 8, 64)
    free, state = torch.empty(4, device="meta", dtype=torch.int32), torch.empty(4, device="meta", dtype=torch.int32)
    slots, starts = ops.reserve_blocks(table, lengths, free, state, lengths, 9, 16)
    assert slots.shape == (9,) and slots.dtype == torch.int64 and starts.shape == (4,) and starts.dtype == torch.int32
