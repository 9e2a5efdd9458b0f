"""Which prefills the Qwen3 adapter runs on prompt_attention: those alone that its backend would run as causal attention."""

from __future__ import annotations

import types

import pytest
import torch

transformers = pytest.importorskip("transformers")

from dartkv_amd.integrations import qwen3  # noqa: E402

DEV = "cuda"


class _Stub:
    """A tensor's face for the guard, which looks at nothing else (no GPU)."""

    device = types.SimpleNamespace(type="cuda")

    def __init__(self, heads, tokens=12, dtype=torch.bfloat16, requires_grad=False):
        self.shape, self.dtype, self.requires_grad = (2, heads, tokens, 64), dtype, requires_grad


def _attn(**over):
    attn = dict(dart_prompt_attention=True, config=types.SimpleNamespace(_attn_implementation="sdpa"), head_dim=64,
                sliding_window=None, training=False, attention_dropout=0.0, is_causal=True)
    attn.update(over)
    return types.SimpleNamespace(**attn)


def _runs(attn=None, q=None, k=None, v=None, mask=None, **kwargs):
    return bool(qwen3._can_run_prompt(attn or _attn(), q or _Stub(4), k or _Stub(2), v or _Stub(2), mask, kwargs))


def test_values_that_require_gradients_keep_the_backend():
    assert _runs()
    assert not _runs(v=_Stub(2, requires_grad=True))
    assert not _runs(v=_Stub(2, dtype=torch.float16))
    with torch.no_grad():
        assert _runs(v=_Stub(2, requires_grad=True))


def _model(**over):
    from dartkv_amd.integrations import attach_dart_fused_attention
    torch.manual_seed(0)
    kw = dict(vocab_size=128, hidden_size=256, intermediate_size=256, num_hidden_layers=2, num_attention_heads=4,
              num_key_value_heads=2, head_dim=64, max_position_embeddings=256, attn_implementation="sdpa",
              layer_types=["full_attention", "full_attention"])
    kw.update(over)
    model = transformers.Qwen3ForCausalLM(transformers.Qwen3Config(**kw)).to(device=DEV, dtype=torch.bfloat16).eval()
    return attach_dart_fused_attention(model, prompt_attention=True)


@pytest.fixture
def calls(monkeypatch):
    seen, real = [], qwen3.prompt_attention

    def record(*args, **kw):
        seen.append(kw)
        return real(*args, **kw)

    monkeypatch.setattr(qwen3, "prompt_attention", record)
    return seen


@pytest.mark.gpu
def test_training_of_the_value_projection_alone(calls):
    model = _model()
    model.requires_grad_(False)
    proj = model.model.layers[0].self_attn.v_proj.weight
    proj.requires_grad_(True)
    ids = torch.randint(0, 128, (2, 12), generator=torch.Generator().manual_seed(1)).to(DEV)
    model(ids, use_cache=False).logits.float().sum().backward()
    assert proj.grad is not None and bool((proj.grad != 0).any())
    assert not calls


def test_attention_that_is_not_causal_keeps_the_backend():
    assert not _runs(_attn(is_causal=False))
    assert _runs(_attn(is_causal=False), is_causal=True)
    assert not _runs(is_causal=False)


@pytest.mark.gpu
def test_a_module_that_is_not_causal_sees_all_keys(calls):
    model = _model()
    ids = torch.randint(0, 128, (2, 12), generator=torch.Generator().manual_seed(1)).to(DEV)
    with torch.no_grad():
        causal = model(ids, use_cache=False).logits
        assert len(calls) == 2
        for layer in model.model.layers:
            layer.self_attn.is_causal = False
        full = model(ids, use_cache=False).logits
        assert len(calls) == 2
    assert not torch.equal(causal[:, 0], full[:, 0])  # (the first token sees the others now)


def test_arguments_that_the_kernel_does_not_know_keep_the_backend():
    assert not _runs(position_bias=torch.zeros(1))
    assert not _runs(output_attentions=True)
    assert _runs(position_bias=None, position_ids=torch.zeros(1), use_cache=True, output_attentions=False,
                 num_items_in_batch=3)
