"""torch.ops.dartkv: derivatives that an operator does not have are refused, not left out."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import dartkv_amd as dart

DEV = "cuda"


def _rotation():
    x = torch.randn(5, 4, 64, device=DEV)
    cos, sin = torch.rand(5, 32, device=DEV), torch.rand(5, 32, device=DEV)
    return x, x[:, :2].contiguous(), cos, sin


@pytest.mark.gpu
@pytest.mark.parametrize("which", [2, 3])
def test_angles_that_require_gradients_are_refused(which):
    args = list(_rotation())
    args[which].requires_grad_()
    for first in (False, True):
        args[0].requires_grad_(first)
        with pytest.raises(RuntimeError, match="cos and sin"):
            torch.ops.dartkv.rotate_heads(*args)
        with torch.no_grad():
            torch.ops.dartkv.rotate_heads(*args)


@pytest.mark.gpu
def test_tangents_of_rotate_heads_are_refused():
    args = list(_rotation())
    for i in range(4):
        for grad in (False, True):
            with forward_ad.dual_level():
                dual = [a.detach() for a in args]
                dual[i] = forward_ad.make_dual(dual[i], torch.ones_like(dual[i]))
                if grad:
                    dual[0 if i else 1].requires_grad_()
                with pytest.raises(RuntimeError):
                    torch.ops.dartkv.rotate_heads(*dual)


@pytest.mark.gpu
def test_tangents_of_token_logprobs_are_refused():
    x, tokens = torch.randn(3, 50, device=DEV), torch.arange(3, device=DEV)
    with forward_ad.dual_level(), pytest.raises(RuntimeError):
        torch.ops.dartkv.token_logprobs(forward_ad.make_dual(x, torch.ones_like(x)), tokens)
    torch.ops.dartkv.token_logprobs(x, tokens)


@pytest.mark.gpu
@pytest.mark.parametrize("operator", [False, True])
def test_tangents_of_a_backward_pass_are_refused(operator):
    """Forward over reverse: the gradients that come in have tangents."""
    x, k, cos, sin = _rotation()
    logits, tokens = torch.randn(3, 50, device=DEV), torch.arange(3, device=DEV)
    rotate = torch.ops.dartkv.rotate_heads if operator else dart.rotate_heads
    logprobs = torch.ops.dartkv.token_logprobs if operator else dart.token_logprobs
    for leaf, call in ((x, lambda t: rotate(t, k, cos, sin)[0]), (logits, lambda t: logprobs(t, tokens)[0])):
        leaf = leaf.clone().requires_grad_()
        out = call(leaf)
        with forward_ad.dual_level():
            g = forward_ad.make_dual(torch.ones_like(out), torch.rand_like(out))
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(out, leaf, g)
        torch.autograd.grad(call(leaf), leaf, torch.ones_like(out))
