"""Backward passes of saved tensors that hooks give back in another layout, as offloading to the host does."""

from __future__ import annotations

import ctypes

import pytest
import torch

import dartkv_amd as dart
from dartkv_amd import _lib, logprobs, rotate

DEV = "cuda"


@pytest.fixture
def launches(monkeypatch):
    """The calls that would go to the library, without a GPU: (entry point, its arguments)."""
    seen = []

    def record(function, args, device, where, stream=None):
        seen.append((where, type(args).from_buffer_copy(args)))

    monkeypatch.setattr(_lib, "require_device", lambda *tensors: None)
    monkeypatch.setattr(_lib, "stream_ptr", lambda device: 0)
    monkeypatch.setattr(_lib, "launch", record)
    for module in (rotate, logprobs):
        monkeypatch.setattr(module, "_workspace", lambda device, n, stream: torch.empty(n, dtype=torch.uint8))
    _lib._templates.clear()
    yield seen
    _lib._templates.clear()


class _Unpacked:
    """Hooks that keep copies in the layout of ``change``, and what was given back."""

    def __init__(self, change):
        self.change, self.given = change, {}

    def __enter__(self):
        def unpack(packed):
            self.given[packed.data_ptr()] = packed
            return packed

        self.hooks = torch.autograd.graph.saved_tensors_hooks(lambda t: self.change(t.detach()), unpack)
        return self.hooks.__enter__()

    def __exit__(self, *exc):
        return self.hooks.__exit__(*exc)


def _contiguous(t):
    return t.clone(memory_format=torch.contiguous_format)


def _shifted(t):  # the same strides, rows that begin at odd elements
    out = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape)
    return out.copy_(t)


def _columns(t):
    return t.t().clone(memory_format=torch.contiguous_format).t() if t.dim() == 2 else t.clone()


def _rotation(device, dtype=torch.float32):
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(10, 8, 64, generator=g).to(device, dtype)
    w = (torch.rand(64, generator=g) + 0.5).to(device)
    cos, sin = (torch.rand(10, 64, generator=g).to(device)[:, :32] for _ in range(2))
    return qkv, cos, sin, w


@pytest.mark.parametrize("change", [_contiguous, _shifted])
def test_a_rotations_gradient_reads_the_tensors_it_is_given(launches, change):
    qkv, cos, sin, w = _rotation("cpu")
    for _ in range(2):  # (arguments anew, and from those that are kept)
        leaf, weight = qkv.clone().requires_grad_(), w.clone().requires_grad_()
        hooks = _Unpacked(change)
        with hooks:
            a, b = dart.rotate_heads(leaf[:, :4], leaf[:, 4:6], cos, sin, q_weight=weight, k_weight=weight)
        torch.autograd.grad((a, b), (leaf, weight), (torch.ones_like(a), torch.ones_like(b)))
        where, args = launches[-1]
        assert where == "dkv_rotate_heads_backward"
        for name, strides in (("query", ("q_st", "q_sh")), ("keys", ("k_st", "k_sh"))):
            tensor = hooks.given.get(getattr(args, name))
            if tensor is None:  # (a copy with aligned rows)
                assert change is _shifted
                assert (getattr(args, strides[0]), getattr(args, strides[1])) == ((256, 64) if name == "query" else (128, 64))
            else:
                assert (getattr(args, strides[0]), getattr(args, strides[1])) == tensor.stride()[:2]
            assert getattr(args, name) % 16 == 0
        assert args.c_st == (hooks.given[args.cos].stride(0) if args.cos in hooks.given else 32)


@pytest.mark.parametrize("change", [_contiguous, _columns])
def test_a_log_probabilitys_gradient_reads_the_tensors_it_is_given(launches, change):
    leaf = torch.randn(6, 50).requires_grad_()
    hooks = _Unpacked(change)
    with hooks:
        out = dart.token_logprobs(leaf[:, :40], torch.arange(6), top=3)
    out.logprobs.sum().backward()
    where, args = launches[-1]
    assert where == "dkv_token_logprobs_backward" and args.vocab == 40
    given = hooks.given.get(args.logits)
    assert args.stride == 40 and (given is None or given.stride() == (40, 1))
    rows = (ctypes.c_float * 240).from_address(args.logits) if given is not None else None
    assert rows is None or list(rows) == leaf.detach()[:, :40].reshape(-1).tolist()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients_of_offloaded_tensors_are_those_of_kept_ones(dtype):
    """The kernels add in one order, so layouts change nothing."""
    qkv, cos, sin, w = _rotation(DEV, dtype)
    logits = torch.randn(7, 999, device=DEV, dtype=dtype)

    def grads():
        leaves = [t.clone().requires_grad_() for t in (qkv, w, logits)]
        a, b = dart.rotate_heads(leaves[0][:, :4], leaves[0][:, 4:6], cos, sin, q_weight=leaves[1], k_weight=leaves[1])
        c, d = dart.rotate_heads(leaves[0].transpose(0, 1)[None, :4], leaves[0].transpose(0, 1)[None, 4:6], cos, sin)
        out = dart.token_logprobs(leaves[2][:, :901], torch.arange(7, device=DEV), top=2)
        loss = (a * a).float().sum() + (b * b * b).float().sum() + (c * c).float().sum() + (d * d).float().sum() \
            + (out.logprobs - out.entropy + out.top_logprobs.sum(-1)).sum()
        return torch.autograd.grad(loss, leaves)

    want = grads()
    with torch.autograd.graph.save_on_cpu():
        got = grads()
    for change in (_contiguous, _shifted, _columns):
        hooks = _Unpacked(change)
        with hooks:
            more = grads()
        assert all(torch.equal(a, b) for a, b in zip(more, want))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
