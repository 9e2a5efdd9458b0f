"""Attention over whole prompts: causal, grouped heads, packed sequences of different lengths.

``prompt_attention`` is the step before a cache is decoded: the prompt's own queries, keys and values, in
bf16 or fp16, as a batch of one length or packed one after the other.  One HIP kernel (MFMA tiles with a running
softmax) reads each tensor once and holds no scores in memory.

The reference has no such kernel: its prefill runs the model's attention backend (reference
src/dart/integrations/qwen3.py:85-97).
"""

from __future__ import annotations

import math
from typing import Optional

import torch
import torch.autograd.forward_ad as forward_ad

from . import _lib
from .attention import _workspace

MAX_PROMPT_HEAD_DIM = 256


def followed(*tensors: torch.Tensor) -> bool:
    """Whether autograd would follow an operation on a tensor, backward or (which no_grad leaves on) forward."""
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        return True
    # (the level is -1 outside forward_ad.dual_level(), where no tensor has a tangent)
    return getattr(forward_ad, "_current_level", 0) >= 0 and any(forward_ad.unpack_dual(t).tangent is not None
                                                                 for t in tensors)


def no_gradients(name: str, *tensors: torch.Tensor) -> None:
    """Forward-only operators refuse tensors that autograd would follow."""
    if followed(*tensors):
        raise RuntimeError(f"{name} has no backward pass; call it under torch.no_grad(), or detach its "
                           "inputs (forward mode: unpack them)")


def scale_factor(scale: Optional[float], head_dim: int, name: str) -> float:
    if scale is None:
        return 1.0 / math.sqrt(head_dim)
    scale = float(scale)
    if not 1e-37 <= scale < 1e30:  # (its fp32 factor must not be 0: a hidden key's logit would be -inf * 0)
        raise ValueError(f"{name}: scale must be positive, from 1e-37 to 1e30")
    return scale


def int32_vector(t: torch.Tensor, what: str, device: torch.device) -> torch.Tensor:
    """``t`` as a contiguous int32 vector on ``device``; what 31 bits do not hold becomes the nearest that they do."""
    if not isinstance(t, torch.Tensor) or t.dim() != 1 or t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{what} must be a one-dimensional int32 or int64 tensor")
    if t.device != device:
        raise ValueError(f"{what} must be on {device}")
    if t.dtype == torch.int64:
        t = t.clamp(-(1 << 31), (1 << 31) - 1)
    return t.to(torch.int32).contiguous()


MAX_TOKEN_STRIDE = (1 << 23) - 1  # elements: the kernels' offsets within a tile have 31 bits


def aligned_rows(t: torch.Tensor, token_axis: int) -> torch.Tensor:
    """``t`` with contiguous, 16-byte aligned last-dimension rows (a copy where it has others)."""
    step = 16 // t.element_size()
    strides = t.stride()
    if strides[-1] != 1 or t.data_ptr() % 16 or any(s % step for s in strides[:-1]) \
            or strides[token_axis] > MAX_TOKEN_STRIDE:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def new_output(query: torch.Tensor) -> torch.Tensor:
    """The output of a call without ``out``: of the query's layout where that has rows of D, else contiguous."""
    out = torch.empty_like(query)
    if out.stride(-1) != 1 or any(s % 4 for s in out.stride()[:-1]):
        out = torch.empty(query.shape, dtype=query.dtype, device=query.device)
    return out


def check_output(out: torch.Tensor, query: torch.Tensor) -> None:
    """Refuse an ``out`` that the kernels cannot write: each row of D has to lie by itself."""
    if out.shape != query.shape or out.dtype != query.dtype or out.device != query.device or out.stride(-1) != 1 \
            or out.data_ptr() % 8 or any(s % 4 for s in out.stride()[:-1]):
        raise ValueError("out must be a tensor of the query's shape, dtype and device, with 8-byte aligned rows of D")
    if any(s == 0 and n > 1 for s, n in zip(out.stride(), out.shape)):
        raise ValueError("out must have rows of its own for every token and head")


def prompt_attention(query: torch.Tensor, keys: torch.Tensor, values: torch.Tensor,
                     query_starts: Optional[torch.Tensor] = None, key_starts: Optional[torch.Tensor] = None, *,
                     causal: bool = True, scale: Optional[float] = None,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(scale q k^T) v of whole prompts, query head h over KV head h // (Hq / Hkv).

    * A batch: ``query`` [B, Hq, Q, D], ``keys`` and ``values`` [B, Hkv, T, D].
    * Packed sequences: ``query`` [Tq, Hq, D], ``keys`` and ``values`` [Tk, Hkv, D] and ``query_starts`` [R + 1]
      (int32 or int64, on the device, ascending): sequence r is rows ``query_starts[r]`` to
      ``query_starts[r + 1]``.  ``key_starts`` (default: the same) where the keys are more than the queries.

    ``causal``: the last query token of a sequence sees all its nk keys, token i of nq the first
    ``i + 1 + nk - nq``; a row that sees no key is 0.  bf16 and fp16, head_dim a multiple of 8 up to 256, any
    strides (rows that are not 16-byte aligned are copied).  ``scale`` (1e-37 to 1e30) defaults to 1 / sqrt(D).
    Returns a tensor like ``query``, or ``out`` (contiguous rows of D).  Rows behind the last packed sequence and before
    the first are 0 in a new tensor and stay as they were in ``out``.  Keys a row does not see do not change it,
    whatever they hold.

    Softmax statistics and sums are fp32; the weights are rounded to the tensors' type for the second product (fp16:
    with 2^7 of its range in hand, so that weights down to 2^-21 of the largest keep all its bits).
    Forward only: tensors that require gradients are refused outside torch.no_grad(), forward-mode tangents always.
    """
    packed = query_starts is not None
    if packed and key_starts is None:
        key_starts = query_starts
    if not packed and key_starts is not None:
        raise ValueError("key_starts needs query_starts")
    fill = out is None
    scale = None if scale is None else float(scale)
    key = None
    if not packed or all(isinstance(t, torch.Tensor) and t.dtype == torch.int32 for t in (query_starts, key_starts)):
        key = ("prompt", bool(causal), scale, fill, packed,
               _lib.layouts(query, keys, values, *((query_starts, key_starts) if packed else ()),
                            *(() if fill else (out,))))
    known = _lib.template(key) if key is not None else None
    if known is not None and not (query.data_ptr() | keys.data_ptr() | values.data_ptr()) % 16 \
            and (fill or not out.data_ptr() % 8):
        no_gradients("prompt_attention", query, keys, values)
        if fill:
            out = new_output(query)
        a = _lib.PromptAttentionArgs.from_buffer_copy(known)
    else:
        a, query, keys, values, query_starts, key_starts, out, whole = _checked(query, keys, values, query_starts,
                                                                               key_starts, causal, scale, out)
        if a is None:
            return out
        if whole and key is not None:  # (no copy of an input was made)
            _lib.keep_template(key, a)
            a = _lib.PromptAttentionArgs.from_buffer_copy(a)
    a.query, a.keys, a.values, a.out = query.data_ptr(), keys.data_ptr(), values.data_ptr(), out.data_ptr()
    if packed:
        a.q_starts, a.k_starts = query_starts.data_ptr(), key_starts.data_ptr()
    stream = _lib.stream_ptr(query.device)
    if a.workspace_bytes:
        workspace = _workspace(query.device, a.workspace_bytes, stream)
        a.workspace = workspace.data_ptr()
    _lib.launch(_lib.load().dkv_prompt_attention, a, query.device, "dkv_prompt_attention", stream)
    return out


def _checked(query, keys, values, query_starts, key_starts, causal, scale, out):
    """The checks of a call and its arguments without pointers (None where there is nothing to compute)."""
    packed = query_starts is not None
    _lib.require_device(query, keys, values)
    if query.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError("prompt_attention takes bf16 and fp16 tensors")
    if keys.dtype != query.dtype or values.dtype != query.dtype:
        raise TypeError("query, keys and values must have one dtype")
    device = query.device
    if keys.device != device or values.device != device:
        raise ValueError("query, keys and values must be on the same device")
    dims = 3 if packed else 4
    if query.dim() != dims or keys.dim() != dims or values.dim() != dims:
        raise ValueError("query, keys and values must be [T, H, D] with query_starts, [B, H, T, D] without")
    if keys.shape != values.shape or query.shape[-1] != keys.shape[-1]:
        raise ValueError("query/key/value head_dim, and key/value shapes must be compatible")
    no_gradients("prompt_attention", query, keys, values)
    t_axis, h_axis = (0, 1) if packed else (2, 1)
    Hq, Hkv, D = query.shape[h_axis], keys.shape[h_axis], query.shape[-1]
    if Hkv == 0 or Hq == 0 or Hq % Hkv:
        raise ValueError("query heads must be divisible by KV heads")
    if D == 0 or D % 8 or D > MAX_PROMPT_HEAD_DIM:
        raise ValueError(f"head_dim must be a multiple of 8 up to {MAX_PROMPT_HEAD_DIM}")
    if not packed and query.shape[0] != keys.shape[0]:
        raise ValueError("query and keys must have one batch size")
    factor = scale_factor(scale, D, "prompt_attention")
    fill = out is None
    if out is None:
        out = new_output(query)
    else:
        check_output(out, query)
    given = (query, keys, values)
    query, keys, values = (aligned_rows(t, t_axis) for t in given)
    whole = all(a is b for a, b in zip(given, (query, keys, values)))

    a = _lib.PromptAttentionArgs()
    if packed:
        query_starts = int32_vector(query_starts, "query_starts", device)
        key_starts = int32_vector(key_starts, "key_starts", device)
        if query_starts.numel() < 2 or key_starts.numel() != query_starts.numel():
            raise ValueError("query_starts and key_starts must hold one more entry than there are sequences")
        a.requests = query_starts.numel() - 1
    else:
        a.requests = query.shape[0]
        a.q_sb, a.k_sb, a.v_sb, a.o_sb = query.stride(0), keys.stride(0), values.stride(0), out.stride(0)
    if a.requests == 0 or query.numel() == 0:
        a = None
        return a, query, keys, values, query_starts, key_starts, out, whole
    a.q_st, a.q_sh = query.stride(t_axis), query.stride(h_axis)
    a.k_st, a.k_sh = keys.stride(t_axis), keys.stride(h_axis)
    a.v_st, a.v_sh = values.stride(t_axis), values.stride(h_axis)
    a.o_st, a.o_sh = out.stride(t_axis), out.stride(h_axis)
    a.Hq, a.Hkv, a.D = Hq, Hkv, D
    a.q_tokens, a.k_tokens = query.shape[t_axis], keys.shape[t_axis]
    a.dtype = _lib.dtype_code(query.dtype)
    a.scale, a.causal, a.fill = factor, bool(causal), fill
    if packed:
        a.q_starts = query_starts.data_ptr()
    a.workspace_bytes = _lib.load().dkv_prompt_attention_workspace_bytes(a)
    return a, query, keys, values, query_starts, key_starts, out, whole


__all__ = ["prompt_attention"]
