"""token_logprobs: what the tests of its values do not reach."""

from __future__ import annotations

import math

import pytest
import torch

import dartkv_amd as dart

from tests.test_token_logprobs import DEV, HALF_STEP, TINY, expected, rows


@pytest.mark.gpu
@pytest.mark.parametrize("T", [3, 700, 2100])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_moments_are_a_reference_and_its_sum(T, dtype):
    """m + ln(2) log2 s is the row's log of the sum of e^x, wherever its maximum lies: s as in expected(), log2 s (at most
    17 + 16) and its product off by 2^-22 of theirs, m exact, one rounding of none of them on the host."""
    x, tokens = rows(T, 20_011, dtype, 40)
    x[0] = 0
    x[0, -1] = 7  # (under what raises the reference by itself)
    x[1] += torch.linspace(0, 60, 20_011).to(dtype)
    moments = dart.torch_ops.token_logprobs(x.to(DEV), tokens.to(DEV), 2)[4].double().cpu()
    x = x.double()
    _, _, _, _, e = expected(x, tokens)
    got = moments[:, 0] + math.log(2) * moments[:, 1]
    assert bool(((got - x.logsumexp(-1)).abs() <= e + 2.0 ** -22 * moments[:, 1].abs()).all())
    assert bool((moments[:, 0] <= x.amax(-1)).all())


def _check_gradient(leaf_of, x, tokens, top, dtype):
    """The gradient of `leaf_of(x)`'s log probabilities, entropies and alternatives against the formula in 64 bits, with
    the tolerance of test_token_logprobs.test_gradients_against_the_formula."""
    gen, shape = torch.Generator().manual_seed(7), tokens.shape
    g, h, g_top = torch.randn(shape, generator=gen), torch.randn(shape, generator=gen), torch.randn(*shape, top, generator=gen)
    leaf = leaf_of(x).requires_grad_()
    out = dart.token_logprobs(leaf, tokens.to(DEV), top=top)
    got = torch.autograd.grad(out[:3], leaf, [t.to(DEV) for t in (g, h, g_top)])[0].double().cpu()
    assert got.shape == x.shape
    V, ids = x.shape[-1], out.top_tokens.cpu().view(tokens.numel(), top)
    x, got, tokens = x.double().reshape(-1, V), got.reshape(-1, V), tokens.reshape(-1)
    g, h, g_top = g.reshape(-1, 1).double(), h.reshape(-1, 1).double(), g_top.view(tokens.numel(), top).double()
    _, logp, entropy, z, e = expected(x, tokens)
    p, G = logp.exp(), g + g_top.sum(-1, keepdim=True)
    entropy, e, logp, z = entropy[:, None], e[:, None], logp.clamp_min(-1e4), z.clamp_min(-1e4)  # (p is 0 there)
    want = (-p * (G + h * (logp + entropy))).scatter_add_(1, tokens[:, None], g).scatter_add_(1, ids, g_top)
    size = p * ((2.0 ** -21 * (z.abs() / math.log(2) + 4) + 4 * e) * (G.abs() + h.abs() * (logp.abs() + entropy)) + 2 * e * h.abs())
    points = torch.zeros_like(want).scatter_add_(1, tokens[:, None], g.abs()).scatter_add_(1, ids, g_top.abs())
    limit = HALF_STEP[dtype] * want.abs() * (1 + 2.0 ** -8) + size \
        + 2.0 ** -18 * (points + p * (g.abs() + g_top.abs().sum(-1, keepdim=True))) + TINY[dtype]
    assert bool(((got - want).abs() <= limit).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,V,top", [(1030, 9001, 5), (2100, 6007, 20), (1100, 20_480, 0)])
def test_gradients_of_rows_that_a_thread_goes_through_in_steps(T, V, top, dtype):
    """From 1,024 rows on a row is one part, whose threads each take several chunks.  An odd size: rows begin at every
    offset within 16 bytes."""
    x, tokens = rows(T, V, dtype, 41 + V)
    _check_gradient(lambda x: x.to(DEV), x, tokens, top, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradients_of_rows_cut_out_of_longer_ones(dtype):
    """Logits and gradient begin at different offsets within 16 bytes; a mask, and a vocabulary that is padded."""
    T, V = 1030, 9001
    x, tokens = rows(T, V, dtype, 42)
    x[:, 7000:7100] = -math.inf
    x[5] = -math.inf
    x[5, :40] = 1
    tokens[tokens.ge(7000) & tokens.lt(7100)], tokens[5] = 3, 20

    def padded(x):
        wide = torch.full((T, V + 11), 50.0, dtype=dtype, device=DEV)
        return wide[:, 3:3 + V].copy_(x).detach()

    _check_gradient(padded, x, tokens, 6, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradients_of_all_tokens_but_the_last(dtype):
    """[B, T, V] logits whose last token is left out: the rows have two strides."""
    x, tokens = rows(4 * 270, 5003, dtype, 43)
    x, tokens = x.view(4, 270, 5003), tokens.view(4, 270)
    _check_gradient(lambda x: x.to(DEV), x, tokens, 3, dtype)
    more = torch.cat((x, x[:, :1] * 2), 1).to(DEV)
    _check_gradient(lambda x: more.detach()[:, :-1], x, tokens, 3, dtype)
    leaf = more.detach().requires_grad_()
    grad = torch.autograd.grad(dart.token_logprobs(leaf[:, :-1], tokens.to(DEV)).logprobs.sum(), leaf)[0]
    assert not grad[:, -1].any() and bool(grad[:, :-1].any(-1).all())
