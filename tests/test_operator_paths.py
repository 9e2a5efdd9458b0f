"""rotate_heads, token_logprobs and the sharing of blocks where the framework calls them: torch.ops.dartkv, the Qwen3
adapter, replayed decode steps."""

from __future__ import annotations

import pytest
import torch

import dartkv_amd as dart
from tests.test_rotate_heads import angles, inputs

DEV = "cuda"


@pytest.fixture(autouse=True)
def _seed():
    torch.manual_seed(0)


def _rotate_inputs(dtype=torch.float32):
    q, k = (t.to(DEV).contiguous() for t in inputs(10, 4, 2, 64, dtype, 1))
    cos, sin = (t.to(DEV) for t in angles(16, 32, torch.float32, 2))
    return q, k, cos, sin, torch.arange(10, device=DEV), torch.rand(64, device=DEV) + 0.5


@pytest.mark.gpu
def test_opcheck_of_rotate_heads():
    q, k, cos, sin, positions, w = _rotate_inputs()
    op, check = torch.ops.dartkv.rotate_heads.default, torch.library.opcheck
    check(op, (q, k, cos, sin, positions, w, w))
    check(op, (q.requires_grad_(), k.requires_grad_(), cos[:10], sin[:10], None, None, w.requires_grad_(), 1e-5, True))
    batch = torch.randn(2, 7, 6, 64, device=DEV).transpose(1, 2)
    check(op, (batch[:, :4], batch[:, 4:], cos[:7], sin[:7]))


@pytest.mark.gpu
def test_opcheck_of_token_logprobs():
    logits = torch.randn(6, 333, device=DEV, requires_grad=True)
    tokens = torch.randint(0, 333, (6,), device=DEV)
    torch.library.opcheck(torch.ops.dartkv.token_logprobs.default, (logits, tokens, 3))
    torch.library.opcheck(torch.ops.dartkv.token_logprobs.default, (logits.detach().view(2, 3, 333), tokens.view(2, 3)))


@pytest.mark.gpu
def test_compiled_gradients_are_the_eager_ones():
    q, k, cos, sin, positions, w = _rotate_inputs()
    logits, tokens = torch.randn(10, 512, device=DEV), torch.randint(0, 512, (10,), device=DEV)
    ops = torch.ops.dartkv

    def loss(q, w, logits):
        a, b = ops.rotate_heads(q, k, cos, sin, positions, w, w)
        out = ops.token_logprobs(logits, tokens, 2)
        return (a * a * a).sum() + (b * w).sum() + (out[0] - 0.1 * out[1] + out[2].sum(-1)).sum()

    def grads(f):
        leaves = [t.detach().clone().requires_grad_() for t in (q, w, logits)]
        return torch.autograd.grad(f(*leaves), leaves)

    def eager(q, w, logits):
        a, b = dart.rotate_heads(q, k, cos, sin, positions, q_weight=w, k_weight=w)
        out = dart.token_logprobs(logits, tokens, top=2)
        return (a * a * a).sum() + (b * w).sum() + (out.logprobs - 0.1 * out.entropy + out.top_logprobs.sum(-1)).sum()

    want = grads(eager)
    for f in (loss, torch.compile(loss, backend="aot_eager", fullgraph=True)):
        for a, b in zip(grads(f), want):  # (the same kernels; sums of two gradients of one tensor in another order)
            assert bool(((a - b).abs() <= 2.0 ** -20 * (a.abs() + b.abs() + 1)).all())


@pytest.mark.gpu
def test_opcheck_of_shared_blocks():
    ops, check = torch.ops.dartkv, torch.library.opcheck
    i32 = dict(dtype=torch.int32, device=DEV)
    tables = (torch.full((3, 4), -1, **i32), torch.zeros(3, **i32), torch.arange(11, -1, -1, **i32), torch.tensor([12, 0, 0, 0], **i32))
    shares, tokens, sources = torch.zeros(12, **i32), torch.tensor([20, 0, 3], **i32), torch.tensor([-1, 0, 0], **i32)
    pools = [torch.zeros(2, 12, 1, 16, 32, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn) for _ in range(2)] + \
        [torch.ones(2, 12, 1, device=DEV) for _ in range(2)]
    check(ops.reserve_shared_blocks.default, (*(t.clone() for t in tables), shares.clone(), tokens, 23, 16))
    ops.reserve_shared_blocks(*tables, shares, tokens, 23, 16)
    check(ops.fork_blocks.default, (*(t.clone() for t in tables), shares.clone(), sources, None, 16))
    ops.fork_blocks(*tables, shares, sources, tokens, 16)
    _, _, copies, positions = ops.reserve_shared_blocks(*tables, shares, torch.ones(3, **i32), 3, 16)
    assert positions.tolist() == [20, 0, 3] and copies.tolist()[0][2] == 3
    check(ops.release_shared_blocks.default, (*(t.clone() for t in tables), shares.clone(), tokens, 16))
    ops.release_shared_blocks(*tables, shares, tokens, 16)
    check(ops.compact_blocks.default, (*(t.clone() for t in tables), shares.clone(), 16))
    rest = ("test_autograd_registration", "test_faketensor")  # (fp8: no comparison of arguments)
    check(ops.copy_blocks.default, (copies, *pools), test_utils=rest)
    x, flag = torch.randn(3, 1, 32, device=DEV), torch.zeros(1, **i32)
    cos, sin = (t.to(DEV) for t in angles(30, 16, torch.float32, 3))
    check(ops.append_rotated_blocks.default, (x, x, x, cos, sin, positions, torch.arange(3, device=DEV), *(t[0] for t in pools), flag),
          test_utils=rest)


def _model(dtype, **attach):
    transformers = pytest.importorskip("transformers")
    from dartkv_amd.integrations import attach_dart_fused_attention
    torch.manual_seed(0)
    config = transformers.Qwen3Config(vocab_size=128, hidden_size=256, intermediate_size=256, num_hidden_layers=2,
                                      num_attention_heads=4, num_key_value_heads=2, head_dim=64, max_position_embeddings=256,
                                      attn_implementation="sdpa", layer_types=["full_attention", "full_attention"])
    model = transformers.Qwen3ForCausalLM(config).to(device=DEV, dtype=dtype).eval()
    for layer in model.model.layers:
        for norm in (layer.self_attn.q_norm, layer.self_attn.k_norm):
            norm.weight.data.uniform_(0.5, 1.5)
    return attach_dart_fused_attention(model, **attach)


@pytest.fixture
def calls(monkeypatch):
    from dartkv_amd.integrations import qwen3
    seen = []

    def record(*args, **kw):
        seen.append(args)
        return dart.rotate_heads(*args, **kw)

    monkeypatch.setattr(qwen3, "rotate_heads", record)
    return seen


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_adapter_rotates_on_the_kernel(calls, dtype):
    """Prefill, decode and a training step.  The modules round after each step (the kernel once): fp32 differs by
    roundings of 2^-24 that two layers carry on, bf16 by some steps of its type."""
    from dartkv_amd.integrations import DartHFCache
    ids = torch.randint(0, 128, (2, 37), generator=torch.Generator().manual_seed(1)).to(DEV)
    results = []
    for on in (False, True):
        model = _model(dtype, rotate_heads=on)
        logits = model(ids).logits
        loss = torch.nn.functional.cross_entropy(logits.float().flatten(0, 1), ids.flatten())
        grads = torch.autograd.grad(loss, [model.model.layers[0].self_attn.q_norm.weight,
                                           model.model.layers[1].self_attn.k_norm.weight,
                                           model.model.layers[0].self_attn.k_proj.weight])
        assert len(calls) == (2 if on else 0)
        with torch.no_grad():
            cache = DartHFCache(dart.DartKVCacheConfig(bits=8, page_size=16, key_group_size=16, value_group_size=16, sink_tokens=4,
                                                       hold_partial_pages=True, metadata_dtype=torch.float16))
            first = model(ids, past_key_values=cache, use_cache=True).logits
            second = model(ids[:, :1], past_key_values=cache, use_cache=True).logits
        assert len(calls) == (6 if on else 0)
        results.append([logits.detach(), *grads, first, second])
    for a, b in zip(*results):
        assert float((a - b).float().norm() / a.float().norm()) < (2.0 ** -14 if dtype == torch.float32 else 0.1)


@pytest.mark.gpu
def test_adapter_keeps_the_modules_for_other_calls(calls):
    """Another norm module, a tangent: the model's own modules run."""
    model = _model(torch.float32, rotate_heads=True)
    ids = torch.arange(9, device=DEV)[None]
    model(ids)
    assert len(calls) == 2

    class Norm(type(model.model.layers[0].self_attn.q_norm)):
        pass

    attn = model.model.layers[0].self_attn
    other = Norm(64).to(DEV)
    other.weight.data.copy_(attn.q_norm.weight)
    attn.q_norm = other
    model(ids)
    assert len(calls) == 3
    _model(torch.float32)(ids)
    assert len(calls) == 3


@pytest.mark.gpu
@pytest.mark.parametrize("use_graph", [False, True])
def test_decode_steps_report_log_probabilities(use_graph):
    from dartkv_amd.integrations import DartHFCache, GraphDecodeStep
    model = _model(torch.bfloat16)
    ids = torch.randint(0, 128, (1, 20), generator=torch.Generator().manual_seed(1)).to(DEV)
    cache = DartHFCache(dart.DartKVCacheConfig(bits=2, page_size=128, key_group_size=128, value_group_size=64, sink_tokens=8,
                                               hold_partial_pages=True, metadata_dtype=torch.float16))
    with torch.no_grad():
        out = model(ids, past_key_values=cache, use_cache=True, logits_to_keep=1)
        nxt, pos = out.logits[:, -1:].argmax(-1), torch.full((1, 1), 20, dtype=torch.long, device=DEV)
        step = GraphDecodeStep(model, cache, nxt, pos, use_graph=use_graph, top_logprobs=5)
        for _ in range(8):
            token = step.step()
            want = dart.token_logprobs(step.logits, token[:, 0], top=5)
            assert all(torch.equal(a, b) for a, b in zip(step.logprobs, want))
            assert torch.equal(step.logprobs.top_tokens[:, 0], token[:, 0])
            assert torch.equal(step.logprobs.logprobs, step.logprobs.top_logprobs[:, 0])
    assert (step.replays > 3) == use_graph
    with pytest.raises(ValueError, match="top_logprobs"):
        GraphDecodeStep(model, cache, nxt, pos, top_logprobs=65)


def test_fakes_on_meta_tensors():
    ops, meta = torch.ops.dartkv, dict(device="meta")
    q = torch.empty(2, 9, 4, 64, **meta).transpose(1, 2)
    a, b = ops.rotate_heads(q, q[:, :1], torch.empty(9, 32, **meta), torch.empty(9, 32, **meta))
    assert a.shape == q.shape and a.stride(-1) == 1 and b.shape == (2, 1, 9, 64)
    out = ops.token_logprobs(torch.empty(3, 2, 100, **meta), torch.empty(3, 2, dtype=torch.int64, **meta), 7)
    assert [tuple(t.shape) for t in out] == [(3, 2), (3, 2), (3, 2, 7), (3, 2, 7), (3, 2, 2)]
