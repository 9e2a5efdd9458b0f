"""The HIP entry points as PyTorch operators: ``torch.ops.dartkv.*``.

Registered with ``torch.library.custom_op``, each operator is one dispatcher
node: ``torch.compile`` keeps it whole instead of tracing into ctypes, its
fake implementation gives output shapes and dtypes without touching the GPU
(meta and fake tensors), and ``torch.library.opcheck`` can test it.  Each one
runs the same C ABI call as the Python API beside it
(``quantization.quantize``, ``QuantizedTensor.dequantize``,
``mixed.quantize_key_mixed``, ``MixedQuantizedKey.dequantize``,
``attention.decode_attention``, ``prompt.prompt_attention``, ``rotate.rotate_heads``,
``logprobs.token_logprobs`` and the operators of ``blocks``); there is no second
implementation.

``decode_attention`` reads a ``DartKVCache``, which is not a tensor: the
operator takes an integer handle from ``cache_handle(cache)``, valid while the
cache lives.  The cache's packed pages are not operator inputs, so a compiled
graph must not move the operator across appends to that cache; appends run
Python control flow, which ends a compiled region anyway.
"""

from __future__ import annotations

import itertools
import weakref
from typing import Optional, Tuple

import torch

from . import attention as _attention
from . import blocks as _blocks
from . import logprobs as _logprobs
from . import mixed as _mixed
from . import prompt as _prompt
from . import quantization as _quantization
from . import rotate as _rotate
from .cache import DartKVCache

Tensor = torch.Tensor

_caches: "weakref.WeakValueDictionary[int, DartKVCache]" = weakref.WeakValueDictionary()
_handles: "weakref.WeakKeyDictionary[DartKVCache, int]" = weakref.WeakKeyDictionary()
_next_handle = itertools.count(1)


def cache_handle(cache: DartKVCache) -> int:
    """Integer naming ``cache`` for ``torch.ops.dartkv.decode_attention`` (valid while it lives).  Handles
    come from a counter and are never reused, so a graph that keeps the handle of a cache that has since
    been freed gets 'unknown handle' rather than another cache."""
    if not isinstance(cache, DartKVCache):
        raise TypeError("cache_handle expects a DartKVCache")
    handle = _handles.get(cache)
    if handle is None:
        handle = _handles[cache] = next(_next_handle)
        _caches[handle] = cache
    return handle


def _cache(handle: int) -> DartKVCache:
    cache = _caches.get(handle)
    if cache is None:
        raise ValueError("unknown DartKVCache handle; get one from dartkv_amd.torch_ops.cache_handle(cache)")
    return cache


def _row_layout(n: int, bits: int, group_size: int) -> Tuple[int, int]:
    """(groups, packed bytes) of one quantized row of n elements."""
    groups = -(-n // group_size)
    per_byte = 8 // bits
    packed = -(-groups * group_size // per_byte)
    return groups, packed


def _meta(data: Tensor, meta_dtype: Optional[torch.dtype]) -> torch.dtype:
    return _quantization._metadata_dtype(data, meta_dtype)


# ---- uniform rows (reference quantization.py:134-204) ----

@torch.library.custom_op("dartkv::quantize_rows", mutates_args=())
def quantize_rows(data: Tensor, bits: int, group_size: int,
                  meta_dtype: Optional[torch.dtype] = None) -> Tuple[Tensor, Tensor, Tensor]:
    """Codes [..., packed], scale and zero point [..., groups] of ``data`` quantized along its last dim."""
    q = _quantization.quantize(data, bits=bits, group_size=group_size, metadata_dtype=meta_dtype)
    return q.values, q.scale, q.zero_point


@quantize_rows.register_fake
def _(data, bits, group_size, meta_dtype=None):
    groups, packed = _row_layout(data.shape[-1], bits, group_size)
    meta = _meta(data, meta_dtype)
    outer = tuple(data.shape[:-1])
    return (data.new_empty(outer + (packed,), dtype=torch.uint8), data.new_empty(outer + (groups,), dtype=meta),
            data.new_empty(outer + (groups,), dtype=meta))


@torch.library.custom_op("dartkv::dequantize_rows", mutates_args=())
def dequantize_rows(values: Tensor, scale: Tensor, zero_point: Tensor, bits: int, group_size: int, n: int,
                    dtype: torch.dtype) -> Tensor:
    """Rows of ``quantize_rows`` back to [..., n] in ``dtype`` with the reference's rounding chain."""
    groups = scale.shape[-1]
    per_byte = 8 // bits
    q = _quantization.QuantizedTensor(
        values=values, scale=scale, zero_point=zero_point, original_shape=tuple(scale.shape[:-1]) + (n,),
        original_dim=n, padded_dim=groups * group_size, packed_dim=values.shape[-1] * per_byte,
        group_size=group_size, bits=bits, output_dtype=dtype, axis=scale.ndim - 1)
    return q.dequantize(dtype=dtype)


@dequantize_rows.register_fake
def _(values, scale, zero_point, bits, group_size, n, dtype):
    return scale.new_empty(tuple(scale.shape[:-1]) + (n,), dtype=dtype)


# ---- Dart keys (reference mixed.py:119-244) ----

@torch.library.custom_op("dartkv::quantize_key_mixed", mutates_args=())
def quantize_key_mixed(key_states: Tensor, group_size: int, promote_ratio: float, strategy: str,
                       meta_dtype: Optional[torch.dtype] = None,
                       channel_indices: Optional[Tensor] = None) -> Tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    """(low codes, high codes, channel indices, scale, zero point) of a key chunk [B, H, T, D]."""
    k = _mixed.quantize_key_mixed(key_states, group_size=group_size, promote_ratio=promote_ratio, strategy=strategy,
                                  metadata_dtype=meta_dtype, channel_indices=channel_indices)
    return k.low_values, k.high_values, k.channel_indices, k.scale, k.zero_point


@quantize_key_mixed.register_fake
def _(key_states, group_size, promote_ratio, strategy, meta_dtype=None, channel_indices=None):
    B, H, T, D = key_states.shape
    K = _mixed.promoted_count(D, promote_ratio)
    G = -(-T // group_size)
    nb = (group_size + 3) // 4
    meta = meta_dtype or (key_states.dtype if key_states.dtype in (torch.float16, torch.bfloat16) else torch.float32)
    u8 = torch.uint8
    return (key_states.new_empty((B, H, D, G, nb), dtype=u8), key_states.new_empty((B, H, K, G, nb if K else nb * 4),
                                                                                    dtype=u8),
            key_states.new_empty((B, H, K), dtype=torch.int32), key_states.new_empty((B, H, D, G), dtype=meta),
            key_states.new_empty((B, H, D, G), dtype=meta))


@torch.library.custom_op("dartkv::dequantize_key_mixed", mutates_args=())
def dequantize_key_mixed(low: Tensor, high: Tensor, channel_indices: Tensor, scale: Tensor, zero_point: Tensor,
                         tokens: int, group_size: int, dtype: torch.dtype) -> Tensor:
    """Keys [B, H, tokens, D] in ``dtype`` from the fields of ``quantize_key_mixed``."""
    B, H, D, G = scale.shape
    k = _mixed.MixedQuantizedKey(low_values=low, high_values=high, channel_indices=channel_indices, scale=scale,
                                 zero_point=zero_point, original_shape=(B, H, tokens, D), padded_tokens=G * group_size,
                                 group_size=group_size, low_bits=2, promote_bits=4, output_dtype=dtype)
    return k.dequantize(dtype=dtype)


@dequantize_key_mixed.register_fake
def _(low, high, channel_indices, scale, zero_point, tokens, group_size, dtype):
    B, H, D, _ = scale.shape
    return scale.new_empty((B, H, tokens, D), dtype=dtype)


# ---- decode (reference fused_attention.py:654-771, attention.py:32-87 for one token) ----

@torch.library.custom_op("dartkv::decode_attention", mutates_args=())
def decode_attention(query: Tensor, cache: int, scale: Optional[float] = None) -> Tensor:
    """One-token attention [B, Hq, 1, D] of ``query`` over the packed cache named by ``cache``."""
    return _attention.decode_attention(query, _cache(cache), scale=scale)


@decode_attention.register_fake
def _(query, cache, scale=None):
    B, Hq, D = query.shape[0], query.shape[1], query.shape[-1]
    return query.new_empty((B, Hq, 1, D))


# ---- prompts and block caches (no reference counterpart) ----

@torch.library.custom_op("dartkv::prompt_attention", mutates_args=())
def prompt_attention(query: Tensor, keys: Tensor, values: Tensor, query_starts: Optional[Tensor] = None,
                     key_starts: Optional[Tensor] = None, causal: bool = True, scale: Optional[float] = None) -> Tensor:
    """Attention over whole prompts, a batch [B, H, T, D] or packed [T, H, D] with starts."""
    return _prompt.prompt_attention(query, keys, values, query_starts, key_starts, causal=causal, scale=scale)


@prompt_attention.register_fake
def _(query, keys, values, query_starts=None, key_starts=None, causal=True, scale=None):
    return _prompt.new_output(query)


@torch.library.custom_op("dartkv::reserve_blocks", mutates_args=("table", "lengths", "free", "state"))
def reserve_blocks(table: Tensor, lengths: Tensor, free: Tensor, state: Tensor, tokens: Tensor, total: int,
                   block_size: int) -> Tuple[Tensor, Tensor]:
    """Slots [total] and starts [requests + 1] of the requests' new tokens; the tables' state moves on."""
    return _blocks.reserve_blocks(table, lengths, free, state, tokens, total, block_size=block_size)


@reserve_blocks.register_fake
def _(table, lengths, free, state, tokens, total, block_size):
    return lengths.new_empty((total,), dtype=torch.int64), lengths.new_empty((lengths.shape[0] + 1,))


@torch.library.custom_op("dartkv::release_blocks", mutates_args=("table", "lengths", "free", "state"))
def release_blocks(table: Tensor, lengths: Tensor, free: Tensor, state: Tensor, tokens: Optional[Tensor],
                   block_size: int) -> None:
    """Drop each request's last tokens (None: all)."""
    _blocks.release_blocks(table, lengths, free, state, tokens, block_size=block_size)


@release_blocks.register_fake
def _(table, lengths, free, state, tokens, block_size):
    return None


@torch.library.custom_op("dartkv::append_blocks",
                         mutates_args=("key_codes", "value_codes", "key_scale", "value_scale"))
def append_blocks(keys: Tensor, values: Tensor, slots: Tensor, key_codes: Tensor, value_codes: Tensor,
                  key_scale: Tensor, value_scale: Tensor) -> None:
    """New keys and values [T, H, D] into their slots of the e4m3 blocks."""
    _blocks.append_blocks(keys, values, slots, key_codes, value_codes, key_scale, value_scale)


@append_blocks.register_fake
def _(keys, values, slots, key_codes, value_codes, key_scale, value_scale):
    return None


# (an operator of its own: torch's custom operators need every argument that they change)
@torch.library.custom_op("dartkv::append_blocks_reported",
                         mutates_args=("key_codes", "value_codes", "key_scale", "value_scale", "nonfinite"))
def append_blocks_reported(keys: Tensor, values: Tensor, slots: Tensor, key_codes: Tensor, value_codes: Tensor,
                           key_scale: Tensor, value_scale: Tensor, nonfinite: Tensor) -> None:
    """``append_blocks``, and ``nonfinite`` (int32, one element) becomes 1 where a key or value is not finite."""
    _blocks.append_blocks(keys, values, slots, key_codes, value_codes, key_scale, value_scale, nonfinite=nonfinite)


@append_blocks_reported.register_fake
def _(keys, values, slots, key_codes, value_codes, key_scale, value_scale, nonfinite):
    return None


@torch.library.custom_op("dartkv::block_attention", mutates_args=())
def block_attention(query: Tensor, key_codes: Tensor, value_codes: Tensor, key_scale: Tensor, value_scale: Tensor,
                    table: Tensor, lengths: Tensor, starts: Optional[Tensor] = None, max_tokens: Optional[int] = None,
                    scale: Optional[float] = None) -> Tensor:
    """Attention [T, Hq, D] of each request's newest tokens over its blocks."""
    return _blocks.block_attention(query, key_codes, value_codes, key_scale, value_scale, table, lengths, starts,
                                   max_tokens=max_tokens, scale=scale)


@block_attention.register_fake
def _(query, key_codes, value_codes, key_scale, value_scale, table, lengths, starts=None, max_tokens=None, scale=None):
    return query.new_empty(query.shape)


# (operators of their own, as an operator's results are the same in number whatever its arguments)
@torch.library.custom_op("dartkv::reserve_shared_blocks", mutates_args=("table", "lengths", "free", "state", "shares"))
def reserve_shared_blocks(table: Tensor, lengths: Tensor, free: Tensor, state: Tensor, shares: Tensor, tokens: Tensor,
                          total: int, block_size: int) -> Tuple[Tensor, Tensor, Tensor, Tensor]:
    """``reserve_blocks`` of tables with forked requests: slots, starts, copies to be made, and positions."""
    positions = torch.empty(total, dtype=torch.int32, device=table.device)
    slots, starts, copies = _blocks.reserve_blocks(table, lengths, free, state, tokens, total, block_size=block_size,
                                                   shares=shares, positions=positions)
    return slots, starts, copies, positions


@reserve_shared_blocks.register_fake
def _(table, lengths, free, state, shares, tokens, total, block_size):
    return (lengths.new_empty((total,), dtype=torch.int64), lengths.new_empty((lengths.shape[0] + 1,)),
            lengths.new_empty((lengths.shape[0], 3)), lengths.new_empty((total,)))


@torch.library.custom_op("dartkv::release_shared_blocks", mutates_args=("table", "lengths", "free", "state", "shares"))
def release_shared_blocks(table: Tensor, lengths: Tensor, free: Tensor, state: Tensor, shares: Tensor,
                          tokens: Optional[Tensor], block_size: int) -> None:
    """``release_blocks`` of tables with forked requests."""
    _blocks.release_blocks(table, lengths, free, state, tokens, block_size=block_size, shares=shares)


@release_shared_blocks.register_fake
def _(table, lengths, free, state, shares, tokens, block_size):
    return None


@torch.library.custom_op("dartkv::fork_blocks", mutates_args=("table", "lengths", "free", "state", "shares"))
def fork_blocks(table: Tensor, lengths: Tensor, free: Tensor, state: Tensor, shares: Tensor, sources: Tensor,
                tokens: Optional[Tensor], block_size: int) -> None:
    """Requests become copies of others (-1: stay), of their first ``tokens`` (None: all)."""
    _blocks.fork_blocks(table, lengths, free, state, shares, sources, tokens, block_size=block_size)


@fork_blocks.register_fake
def _(table, lengths, free, state, shares, sources, tokens, block_size):
    return None


@torch.library.custom_op("dartkv::compact_blocks", mutates_args=("table", "lengths", "free", "state", "shares"))
def compact_blocks(table: Tensor, lengths: Tensor, free: Tensor, state: Tensor, shares: Tensor,
                   block_size: int) -> Tensor:
    """The blocks in use move to the lowest numbers; the copies [blocks // 2, 3] that have to be made."""
    return _blocks.compact_blocks(table, lengths, free, state, shares, block_size=block_size)


@compact_blocks.register_fake
def _(table, lengths, free, state, shares, block_size):
    return lengths.new_empty((free.shape[0] // 2, 3))


@torch.library.custom_op("dartkv::copy_blocks", mutates_args=("key_codes", "value_codes", "key_scale", "value_scale"))
def copy_blocks(copies: Tensor, key_codes: Tensor, value_codes: Tensor, key_scale: Tensor, value_scale: Tensor) -> None:
    """Blocks' first tokens and scales to other blocks, in every layer."""
    _blocks.copy_blocks(copies, key_codes, value_codes, key_scale, value_scale)


@copy_blocks.register_fake
def _(copies, key_codes, value_codes, key_scale, value_scale):
    return None


@torch.library.custom_op("dartkv::append_rotated_blocks",
                         mutates_args=("key_codes", "value_codes", "key_scale", "value_scale", "nonfinite"))
def append_rotated_blocks(query: Tensor, keys: Tensor, values: Tensor, cos: Tensor, sin: Tensor, positions: Tensor,
                          slots: Tensor, key_codes: Tensor, value_codes: Tensor, key_scale: Tensor,
                          value_scale: Tensor, nonfinite: Tensor, q_weight: Optional[Tensor] = None,
                          k_weight: Optional[Tensor] = None, eps: float = 1e-6, interleaved: bool = False) -> Tensor:
    """The rotated queries; keys, normed and rotated, and values go into their slots."""
    return _blocks.append_rotated_blocks(query, keys, values, cos, sin, positions, slots, key_codes, value_codes,
                                         key_scale, value_scale, q_weight=q_weight, k_weight=k_weight, eps=eps,
                                         interleaved=interleaved, nonfinite=nonfinite)


@append_rotated_blocks.register_fake
def _(query, keys, values, cos, sin, positions, slots, key_codes, value_codes, key_scale, value_scale, nonfinite,
      q_weight=None, k_weight=None, eps=1e-6, interleaved=False):
    return query.new_empty(query.shape)


# ---- norm and rotation, log probabilities: with gradients (no reference counterpart) ----

@torch.library.custom_op("dartkv::rotate_heads", mutates_args=())
def rotate_heads(query: Tensor, keys: Tensor, cos: Tensor, sin: Tensor, positions: Optional[Tensor] = None,
                 q_weight: Optional[Tensor] = None, k_weight: Optional[Tensor] = None, eps: float = 1e-6,
                 interleaved: bool = False) -> Tuple[Tensor, Tensor]:
    """RMS norm of each head and its rotation by the token's position."""
    with torch.no_grad():
        return _rotate.rotate_heads(query, keys, cos, sin, positions, q_weight=q_weight, k_weight=k_weight, eps=eps,
                                    interleaved=interleaved)


@rotate_heads.register_fake
def _(query, keys, cos, sin, positions=None, q_weight=None, k_weight=None, eps=1e-6, interleaved=False):
    return _rotate.new_rows(query), _rotate.new_rows(keys)


@torch.library.custom_op("dartkv::rotate_heads_backward", mutates_args=())
def rotate_heads_backward(q_grad: Tensor, k_grad: Tensor, query: Tensor, keys: Tensor, cos: Tensor, sin: Tensor,
                          positions: Optional[Tensor], q_weight: Optional[Tensor], k_weight: Optional[Tensor],
                          eps: float, interleaved: bool) -> Tuple[Tensor, Tensor, Tensor, Tensor]:
    """Gradients of query, keys and the weights (empty where there is no weight)."""
    dq, dk, *weights = _rotate.gradients(q_grad, k_grad, query, keys, cos, sin, positions, q_weight, k_weight, eps,
                                         interleaved)
    return dq, dk, *(query.new_empty(0) if w is None else w for w in weights)


@rotate_heads_backward.register_fake
def _(q_grad, k_grad, query, keys, cos, sin, positions, q_weight, k_weight, eps, interleaved):
    return (_rotate.new_rows(query), _rotate.new_rows(keys),
            *(query.new_empty(0) if w is None else w.new_empty(w.shape) for w in (q_weight, k_weight)))


def _rotate_setup(ctx, inputs, output):
    if any(ctx.needs_input_grad[2:4]):
        raise RuntimeError("rotate_heads has no gradients of cos and sin; detach them")
    query, keys, cos, sin, positions, q_weight, k_weight, ctx.eps, ctx.interleaved = inputs
    ctx.save_for_backward(query, keys, cos, sin, positions, q_weight, k_weight)


def _rotate_backward(ctx, q_grad, k_grad):
    query, keys, cos, sin, positions, q_weight, k_weight = ctx.saved_tensors
    dq, dk, dwq, dwk = torch.ops.dartkv.rotate_heads_backward(q_grad, k_grad, query, keys, cos, sin, positions, q_weight,
                                                              k_weight, ctx.eps, ctx.interleaved)
    return dq, dk, None, None, None, None if q_weight is None else dwq, None if k_weight is None else dwk, None, None


rotate_heads.register_autograd(_rotate_backward, setup_context=_rotate_setup)


@torch.library.custom_op("dartkv::token_logprobs", mutates_args=())
def token_logprobs(logits: Tensor, tokens: Tensor, top: int = 0) -> Tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    """``TokenLogprobs``' four, and what the gradient needs of each row: a reference m, which is not its maximum, and
    log2 of the sum of e^(x - m)."""
    return _logprobs.with_moments(logits, tokens, top)


@token_logprobs.register_fake
def _(logits, tokens, top=0):
    shape = tuple(tokens.shape)
    f32 = dict(dtype=torch.float32)
    return (logits.new_empty(shape, **f32), logits.new_empty(shape, **f32), logits.new_empty((*shape, top), **f32),
            logits.new_empty((*shape, top), dtype=torch.int64), logits.new_empty((*shape, 2), **f32))


@torch.library.custom_op("dartkv::token_logprobs_backward", mutates_args=())
def token_logprobs_backward(logprobs: Tensor, entropy: Tensor, top_logprobs: Tensor, logits: Tensor, tokens: Tensor,
                            moments: Tensor, row_entropy: Tensor, top_tokens: Tensor) -> Tensor:
    """The gradient of the logits from those of the log probabilities, the entropy and the alternatives."""
    return _logprobs.gradient(logprobs, entropy, top_logprobs, logits, tokens, moments, row_entropy, top_tokens)


@token_logprobs_backward.register_fake
def _(logprobs, entropy, top_logprobs, logits, tokens, moments, row_entropy, top_tokens):
    return logits.new_empty(logits.shape)


def _logprobs_setup(ctx, inputs, output):
    logits, tokens, _ = inputs
    _, entropy, _, top_tokens, moments = output
    ctx.save_for_backward(logits, tokens, moments, entropy, top_tokens)
    ctx.mark_non_differentiable(top_tokens, moments)


def _logprobs_backward(ctx, logprobs, entropy, top_logprobs, _, __):
    logits, tokens, moments, row_entropy, top_tokens = ctx.saved_tensors
    return torch.ops.dartkv.token_logprobs_backward(logprobs, entropy, top_logprobs, logits, tokens, moments, row_entropy,
                                                    top_tokens), None, None


token_logprobs.register_autograd(_logprobs_backward, setup_context=_logprobs_setup)


__all__ = ["append_blocks", "append_blocks_reported", "append_rotated_blocks", "block_attention", "cache_handle",
           "compact_blocks", "copy_blocks", "decode_attention", "dequantize_key_mixed", "dequantize_rows", "fork_blocks",
           "prompt_attention", "quantize_key_mixed", "quantize_rows", "release_blocks", "release_shared_blocks",
           "reserve_blocks", "reserve_shared_blocks", "rotate_heads", "rotate_heads_backward", "token_logprobs",
           "token_logprobs_backward"]
