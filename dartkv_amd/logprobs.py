"""What logits say of tokens: log probabilities, entropy and the most likely alternatives, with gradients.

``token_logprobs`` reads each row of logits once.  A serving program reports with it what it sampled and what else was
likely (also the continuations that a beam search goes on from, see ``BlockKVCache.fork``), scores prompts, and trains
on it; ``integrations.GraphDecodeStep`` calls it within its captured step.

No counterpart in the reference.
"""

from __future__ import annotations

from typing import NamedTuple

import torch
import torch.autograd.forward_ad as forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from .attention import _workspace
from .prompt import followed
from .rotate import DTYPES, no_tangents

MAX_TOP = 64


class TokenLogprobs(NamedTuple):
    """``logprobs`` and ``entropy`` [..] (fp32, nats), ``top_logprobs`` (fp32) and ``top_tokens`` (int64) [.., top]."""

    logprobs: torch.Tensor
    entropy: torch.Tensor
    top_logprobs: torch.Tensor
    top_tokens: torch.Tensor


def _checked(logits, tokens, top):
    if not isinstance(tokens, torch.Tensor):
        raise TypeError("tokens must be an int32 or int64 tensor")
    _lib.require_device(logits, tokens)
    if logits.dtype not in DTYPES:
        raise TypeError("token_logprobs takes bf16, fp16 and fp32 logits")
    if tokens.dtype not in (torch.int32, torch.int64):
        raise TypeError("tokens must be an int32 or int64 tensor")
    if logits.dim() < 1 or tokens.shape != logits.shape[:-1]:
        raise ValueError("logits must be [.., vocabulary] and tokens one for each row")
    if tokens.device != logits.device:
        raise ValueError("logits and tokens must be on the same device")
    V = logits.shape[-1]
    if V == 0 or V >= (1 << 31) - 64:
        raise ValueError("logits must have a vocabulary")
    if not 0 <= top <= min(MAX_TOP, V):
        raise ValueError(f"top must be from 0 to {MAX_TOP}, and at most the vocabulary")


def _forward(logits, tokens, top, stats):
    """[rows, V] logits and [rows] tokens: the four outputs, and the rows' statistics (None unless ``stats``)."""
    device, (rows, V) = logits.device, logits.shape
    key = ("logprobs", top, _lib.layouts(logits, tokens))
    known = _lib.template(key)
    if known is None:
        known = _lib.TokenLogprobsArgs()
        known.stride, known.rows, known.vocab, known.top = logits.stride(0), rows, V, top
        known.dtype, known.wide_tokens = _lib.dtype_code(logits.dtype), tokens.dtype == torch.int64
        known.workspace_bytes = _lib.load().dkv_token_logprobs_workspace_bytes(known)
        _lib.keep_template(key, known)
    logprobs, entropy = (torch.empty(rows, dtype=torch.float32, device=device) for _ in range(2))
    top_logprobs = torch.empty(rows, top, dtype=torch.float32, device=device)
    top_tokens = torch.empty(rows, top, dtype=torch.int64, device=device)
    moments = torch.empty(rows, 2, dtype=torch.float32, device=device) if stats else None
    if rows:
        a = _lib.TokenLogprobsArgs.from_buffer_copy(known)
        a.logits, a.tokens = logits.data_ptr(), tokens.data_ptr()
        a.logprobs, a.entropy, a.stats = logprobs.data_ptr(), entropy.data_ptr(), _lib.ptr(moments)
        a.top_logprobs, a.top_tokens = top_logprobs.data_ptr(), top_tokens.data_ptr()
        stream = _lib.stream_ptr(device)
        if a.workspace_bytes:
            workspace = _workspace(device, a.workspace_bytes, stream)
            a.workspace = workspace.data_ptr()
        _lib.launch(_lib.load().dkv_token_logprobs, a, device, "dkv_token_logprobs", stream)
    return logprobs, entropy, top_logprobs, top_tokens, moments


def _backward(logits, tokens, moments, entropy, top_tokens, grads):
    """The gradient of [rows, V] logits from those of logprobs, entropy and top_logprobs (None: 0)."""
    if getattr(forward_ad, "_current_level", 0) >= 0:
        no_tangents("the gradient of token_logprobs", logits, *grads)
    device, (rows, V) = logits.device, logits.shape
    out = torch.empty(rows, V, dtype=logits.dtype, device=device)
    if rows == 0:
        return out
    grads = [g if g is None or (g.dtype == torch.float32 and g.is_contiguous()) else g.to(torch.float32).contiguous()
             for g in grads]
    a, g = _lib.TokenLogprobsArgs(), _lib.TokenLogprobsGrads()
    a.logits, a.tokens, a.stats, a.entropy = logits.data_ptr(), tokens.data_ptr(), moments.data_ptr(), entropy.data_ptr()
    a.top_tokens = top_tokens.data_ptr()
    a.stride, a.rows, a.vocab, a.top = logits.stride(0), rows, V, top_tokens.shape[1]
    a.dtype, a.wide_tokens = _lib.dtype_code(logits.dtype), tokens.dtype == torch.int64
    g.logprobs, g.entropy, g.top_logprobs = (_lib.ptr(t) for t in grads)
    g.out, g.stride = out.data_ptr(), V
    lib, stream = _lib.load(), _lib.stream_ptr(device)
    _lib.launch(lambda args, s: lib.dkv_token_logprobs_backward(args, g, s), a, device, "dkv_token_logprobs_backward", stream)
    return out


def _rows(logits, tokens):
    """[rows, V] logits and [rows] tokens."""
    rows = logits.reshape(-1, logits.shape[-1])
    return rows if rows.stride(1) == 1 else rows.contiguous(), tokens.reshape(-1).contiguous()


def with_moments(logits, tokens, top):
    """``TokenLogprobs``' four, and the rows' moments [.., 2], which ``gradient`` takes: a reference m and log2 of the sum
    of e^(x - m)."""
    _checked(logits, tokens, top)
    no_tangents("token_logprobs", logits)
    shape = tokens.shape
    logprobs, entropy, top_logprobs, top_tokens, moments = _forward(*_rows(logits, tokens), top, True)
    return (logprobs.view(shape), entropy.view(shape), top_logprobs.view(*shape, top), top_tokens.view(*shape, top),
            moments.view(*shape, 2))


def gradient(logprobs, entropy, top_logprobs, logits, tokens, moments, row_entropy, top_tokens):
    """The gradient of logits [.., V] from those of their results; the rest as ``with_moments`` gave it."""
    top = top_tokens.shape[-1]
    _checked(logits, tokens, top)
    shape = tuple(tokens.shape)
    given = (logprobs, shape), (entropy, shape), (row_entropy, shape), (top_logprobs, (*shape, top)), \
        (top_tokens, (*shape, top)), (moments, (*shape, 2))
    if any(tuple(t.shape) != s or t.device != logits.device for t, s in given) or top_tokens.dtype != torch.int64:
        raise ValueError("the results' gradients, moments and alternatives must be those of the logits")
    rows, flat = _rows(logits, tokens)
    n = flat.numel()
    moments, row_entropy = (t.to(torch.float32).contiguous() for t in (moments, row_entropy))
    out = _backward(rows, flat, moments, row_entropy, top_tokens.contiguous().view(n, top),
                    (logprobs, entropy, top_logprobs))
    return out.view(logits.shape)


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, top):
        logprobs, entropy, top_logprobs, top_tokens, moments = _forward(logits, tokens, top, True)
        ctx.save_for_backward(logits, tokens, moments, entropy, top_tokens)
        ctx.mark_non_differentiable(top_tokens)
        ctx.set_materialize_grads(False)
        return logprobs, entropy, top_logprobs, top_tokens

    @staticmethod
    @once_differentiable
    def backward(ctx, logprobs, entropy, top_logprobs, _):
        logits, *rest = ctx.saved_tensors
        # (hooks of saved tensors, such as those that offload them, may give them back in another layout)
        if logits.stride(1) != 1:
            logits = logits.contiguous()
        if not all([t.is_contiguous() for t in rest]):
            rest = [t.contiguous() for t in rest]
        return _backward(logits, *rest, (logprobs, entropy, top_logprobs)), None, None


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, top: int = 0) -> TokenLogprobs:
    """Log probabilities of ``tokens`` [..] (int32 or int64) under ``logits`` [.., V] (bf16, fp16 or fp32), each row's
    entropy, and its ``top`` (up to 64) most likely tokens with theirs, in descending order, the lower one first among
    equals.  All in fp32, in nats.

    A negative token is of no interest: its log probability is 0, without a gradient; one behind the vocabulary has
    NaN.  Logits of -inf have probability 0; a row of nothing else has log probabilities -inf, entropy 0 and no
    gradient.  A NaN or an infinity makes the row's results NaN; a NaN is no alternative (-1 where too few others are).

    Rows of [rows, V] logits may have any stride and are read in place.  A last dimension that is not contiguous is
    copied, and so are more leading dimensions that do not fold into one, as ``logits[:, :-1]`` of a batch: the whole of
    the logits, kept for the backward pass.  Gradients of ``logits`` through the log probabilities, the entropy and the
    alternatives' log probabilities, not twice; a captured backward pass as for ``rotate_heads``.
    """
    top = int(top)
    _checked(logits, tokens, top)
    shape = tokens.shape
    rows, flat = _rows(logits, tokens)
    if followed(logits):
        no_tangents("token_logprobs", logits)
        out = _TokenLogprobs.apply(rows, flat, top)
    else:
        out = _forward(rows, flat, top, False)[:4]
    logprobs, entropy, top_logprobs, top_tokens = out
    if logits.dim() != 2:
        logprobs, entropy = logprobs.view(shape), entropy.view(shape)
        top_logprobs, top_tokens = top_logprobs.view(*shape, top), top_tokens.view(*shape, top)
    return TokenLogprobs(logprobs, entropy, top_logprobs, top_tokens)


__all__ = ["TokenLogprobs", "token_logprobs"]
