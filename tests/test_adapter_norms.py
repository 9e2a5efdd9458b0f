"""When the Qwen3 adapter runs its norms and rotary embedding on rotate_heads: where the modules would compute the same,
and nothing watches or replaces them."""

from __future__ import annotations

import types

import pytest
import torch

transformers = pytest.importorskip("transformers")

from dartkv_amd.integrations import qwen3  # noqa: E402

DEV = "cuda"
modules = qwen3._qwen3_modules()


class _Stub:
    """A tensor's face for the guard, which looks at nothing else (no GPU)."""

    device = types.SimpleNamespace(type="cuda")

    def __init__(self, *shape, dtype=torch.bfloat16, requires_grad=False, device=None):
        self.shape, self.dtype, self.requires_grad = shape, dtype, requires_grad
        self.device = device or _Stub.device

    def dim(self):
        return len(self.shape)


def _norm(**weight):
    norm = modules.Qwen3RMSNorm(64)
    del norm.weight
    norm.__dict__["weight"] = _Stub(64, **weight)
    return norm


def _runs(q_norm=None, k_norm=None, dtype=torch.bfloat16, angles=torch.bfloat16):
    attn = types.SimpleNamespace(dart_rotate_heads=True, head_dim=64, q_norm=q_norm or _norm(), k_norm=k_norm or _norm())
    cos, sin = (_Stub(1, 9, 64, dtype=angles) for _ in range(2))
    return bool(qwen3._can_rotate(attn, modules, _Stub(2, 9, 4, 64, dtype=dtype), _Stub(2, 9, 2, 64, dtype=dtype), cos, sin))


@pytest.mark.parametrize("side", ["q_norm", "k_norm"])
def test_hooks_on_a_norm_keep_the_modules(side):
    assert _runs()
    for register in ("register_forward_hook", "register_forward_pre_hook", "register_full_backward_hook",
                     "register_full_backward_pre_hook"):
        norm = _norm()
        handle = getattr(norm, register)(lambda *args: None)
        assert not _runs(**{side: norm})
        handle.remove()
        assert _runs(**{side: norm})
    norm = _norm()
    norm.forward = lambda x: x
    assert not _runs(**{side: norm})


def test_hooks_on_all_modules_keep_the_modules():
    handle = torch.nn.modules.module.register_module_forward_hook(lambda *args: None)
    try:
        assert not _runs()
    finally:
        handle.remove()
    assert _runs()


def test_weights_elsewhere_keep_the_modules():
    assert not _runs(_norm(device=types.SimpleNamespace(type="cpu")), _norm(device=types.SimpleNamespace(type="cpu")))
    assert not _runs(k_norm=_norm(device=types.SimpleNamespace(type="meta")))


def test_types_that_the_modules_would_widen_keep_them():
    """weight * x and x * cos have the wider type of the two."""
    wide = dict(dtype=torch.float32)
    assert not _runs(_norm(**wide), _norm(**wide))
    assert not _runs(angles=torch.float32)
    assert _runs(_norm(**wide), _norm(**wide), torch.float32, torch.float32)
    assert _runs(dtype=torch.float32, angles=torch.float32)  # (16-bit weights under fp32 projections: fp32)


def test_a_trace_records_the_modules(monkeypatch):
    """torch.jit.trace would take what the kernel writes for a constant."""
    monkeypatch.setattr(torch.jit, "is_tracing", lambda: True)
    assert not _runs()


def _model(**attach):
    torch.manual_seed(0)
    config = transformers.Qwen3Config(vocab_size=128, hidden_size=256, intermediate_size=256, num_hidden_layers=2,
                                      num_attention_heads=4, num_key_value_heads=2, head_dim=64, max_position_embeddings=256,
                                      attn_implementation="sdpa", layer_types=["full_attention", "full_attention"])
    model = transformers.Qwen3ForCausalLM(config).to(DEV).eval()
    return qwen3.attach_dart_fused_attention(model, **attach)


@pytest.fixture
def calls(monkeypatch):
    seen, real = [], qwen3.rotate_heads

    def record(*args, **kw):
        seen.append(args)
        return real(*args, **kw)

    monkeypatch.setattr(qwen3, "rotate_heads", record)
    return seen


@pytest.mark.gpu
def test_a_hook_sees_and_changes_the_norms_output(calls):
    model, ids = _model(rotate_heads=True), torch.arange(9, device=DEV)[None]
    with torch.no_grad():
        plain = model(ids, use_cache=False).logits
        assert len(calls) == 2
        seen = []
        handle = model.model.layers[0].self_attn.q_norm.register_forward_hook(lambda m, i, out: seen.append(out) or 2 * out)
        changed = model(ids, use_cache=False).logits
        assert len(calls) == 3 and [tuple(t.shape) for t in seen] == [(1, 9, 4, 64)]
        handle.remove()
        again = model(ids, use_cache=False).logits
    assert len(calls) == 5
    assert not torch.equal(plain, changed) and torch.equal(plain, again)


@pytest.mark.gpu
def test_a_tangent_keeps_the_modules(calls):
    import torch.autograd.forward_ad as forward_ad
    attn = _model(rotate_heads=True).model.layers[0].self_attn
    attn.config._attn_implementation = "eager"
    hidden, cos, sin = torch.randn(1, 9, 256, device=DEV), torch.rand(1, 9, 64, device=DEV), torch.rand(1, 9, 64, device=DEV)
    with torch.no_grad(), forward_ad.dual_level():
        out, _ = attn(forward_ad.make_dual(hidden, torch.randn_like(hidden)), (cos, sin), None)
        tangent = forward_ad.unpack_dual(out).tangent
        assert tangent is not None and bool((tangent != 0).any())
    assert not calls


@pytest.mark.gpu
def test_fp32_weights_under_16_bit_projections(calls):
    """As under autocast: the modules give fp32 queries and keys, and so does the attached module."""
    results = []
    for on in (False, True):
        model = _model(rotate_heads=on)
        with torch.no_grad(), torch.autocast("cuda", torch.bfloat16):
            results.append(model(torch.arange(9, device=DEV)[None], use_cache=False).logits)
    assert not calls and torch.equal(*results)


@pytest.mark.gpu
def test_a_compiled_module_has_the_operator_in_its_graph(calls):
    attn = _model(rotate_heads=True).model.layers[0].self_attn
    hidden, cos, sin = torch.randn(2, 9, 256, device=DEV), torch.rand(1, 9, 64, device=DEV), torch.rand(1, 9, 64, device=DEV)
    graphs = []

    def backend(graph, inputs):
        graphs.append(graph)
        return graph.forward

    with torch.no_grad():
        want, _ = attn(hidden, (cos, sin), None)
        assert len(calls) == 1
        got, _ = torch.compile(attn, backend=backend, fullgraph=True)(hidden, (cos, sin), None)
    assert torch.equal(got, want)
    assert any("rotate_heads" in str(node.target) for node in graphs[0].graph.nodes)
