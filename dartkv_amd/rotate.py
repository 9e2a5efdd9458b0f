"""Norm and rotation of query and key heads in one pass, with gradients.

``rotate_heads`` stands between a layer's projections and its attention (``prompt_attention``, or ``append_blocks``
and ``block_attention``; ``append_rotated_blocks`` does it within the append): RMS norm of each head, as models with
norms of queries and keys have it, and the rotary embedding by the token's position.

The reference calls the model's modules for both (reference src/dart/integrations/qwen3.py:48-53).
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
import torch.autograd.forward_ad as forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from .attention import _workspace
from .prompt import aligned_rows, followed

MAX_ROTATE_HEAD_DIM = 256
DTYPES = (torch.bfloat16, torch.float16, torch.float32)
_MAX_BACKWARD = 32  # arguments of backward passes that are kept for a layout of the forward


def no_tangents(name: str, *tensors: Optional[torch.Tensor]) -> None:
    """Operators with a backward pass alone, and their backward passes, refuse forward-mode tangents."""
    if getattr(forward_ad, "_current_level", 0) >= 0 and any(
            t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{name} has no forward-mode derivative; unpack its inputs")


def new_rows(like: torch.Tensor) -> torch.Tensor:
    """A tensor like ``like``, in its layout where that has rows of the last dimension, else contiguous."""
    out = torch.empty_like(like)
    if out.stride(-1) != 1 or any(s * out.element_size() % 16 for s in out.stride()[:-1]):
        out = torch.empty(like.shape, dtype=like.dtype, device=like.device)
    return out


def check_weights(q_weight, k_weight, D, device) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor]]:
    given = [w for w in (q_weight, k_weight) if w is not None]
    for w in given:
        if w.dtype not in DTYPES or w.dtype != given[0].dtype:
            raise TypeError("q_weight and k_weight must be bf16, fp16 or fp32, and of one dtype")
        if w.shape != (D,) or w.device != device:
            raise ValueError("q_weight and k_weight must be [head_dim] tensors on the same device")
    return tuple(w if w is None or (w.is_contiguous() and w.data_ptr() % 16 == 0)
                 else w.clone(memory_format=torch.contiguous_format) for w in (q_weight, k_weight))


def check_angles(cos, sin, positions, tokens: Tuple[int, ...], D: int, device):
    """cos and sin with one layout and aligned rows, the positions as a contiguous vector, and the strides of a batch
    and a token.  ``tokens``: (T,) of packed queries, (B, T) of a batch."""
    if cos.dtype not in DTYPES or sin.dtype != cos.dtype:
        raise TypeError("cos and sin must be bf16, fp16 or fp32, and of one dtype")
    if cos.shape != sin.shape or cos.dim() < 2 or cos.device != device or sin.device != device:
        raise ValueError("cos and sin must have one shape [.., angles], on the same device")
    if 2 * cos.shape[-1] > D:
        raise ValueError("cos and sin have more angles than head_dim has pairs")
    if positions is not None:
        if positions.dtype not in (torch.int32, torch.int64):
            raise TypeError("positions must be an int32 or int64 tensor")
        if positions.shape != tokens or positions.device != device:
            raise ValueError(f"positions must hold one position for each token, {list(tokens)}")
        if cos.dim() != 2:
            raise ValueError("with positions, cos and sin are tables [positions, angles]")
        positions = positions.contiguous()
    elif tuple(cos.shape[:-1]) not in ((tokens,) if len(tokens) == 1 else (tokens, tokens[1:], (1, tokens[1]))):
        raise ValueError("without positions, cos and sin hold the angles of each token")
    half = cos.shape[-1]
    vector = 8 if half % 8 == 0 else 2 if half % 2 == 0 else 1
    step = min(16, vector * cos.element_size())

    def rows(t):
        return t.stride(-1) == 1 and t.data_ptr() % step == 0 and not any(
            s * t.element_size() % step for s in t.stride()[:-1])

    if half and (cos.stride() != sin.stride() or not rows(cos) or not rows(sin)):
        cos, sin = (t.clone(memory_format=torch.contiguous_format) for t in (cos, sin))
    c_st = cos.stride(-2)
    c_sb = cos.stride(0) if cos.dim() == 3 and cos.shape[0] > 1 else 0
    return cos, sin, positions, c_sb, c_st


def set_angles(a, cos, sin, positions, c_sb, c_st, interleaved, eps) -> None:
    a.c_sb, a.c_st, a.table_rows = c_sb, c_st, cos.shape[0]
    a.wide_positions = positions is not None and positions.dtype == torch.int64
    a.half, a.interleaved = cos.shape[-1], bool(interleaved)
    a.angle_dtype, a.eps = _lib.dtype_code(cos.dtype), float(eps)


def _checked(query, keys, cos, sin, positions, q_weight, k_weight, eps, interleaved):
    """The checks of a call: its arguments without pointers, and the tensors with aligned rows."""
    _lib.require_device(query, keys, cos, sin, positions, q_weight, k_weight)
    device = query.device
    if query.dtype not in DTYPES:
        raise TypeError("rotate_heads takes bf16, fp16 and fp32 queries and keys")
    if keys.dtype != query.dtype:
        raise TypeError("query and keys must have one dtype")
    if keys.device != device:
        raise ValueError("the tensors must be on the same device")
    if query.dim() not in (3, 4) or keys.dim() != query.dim():
        raise ValueError("query and keys must be [T, H, D], or [B, H, T, D]")
    t_axis, h_axis = (0, 1) if query.dim() == 3 else (2, 1)
    tokens = query.shape[:1] if query.dim() == 3 else (query.shape[0], query.shape[2])
    D = query.shape[-1]
    if keys.shape[-1] != D or keys.shape[0] != query.shape[0] or keys.shape[t_axis] != query.shape[t_axis]:
        raise ValueError("query and keys must have the same tokens and head_dim")
    if query.shape[h_axis] == 0 or keys.shape[h_axis] == 0:
        raise ValueError("query and keys must have heads")
    if D == 0 or D % 8 or D > MAX_ROTATE_HEAD_DIM:
        raise ValueError(f"head_dim must be a multiple of 8 up to {MAX_ROTATE_HEAD_DIM}")
    if not 0 <= eps < 1e30:
        raise ValueError("eps must not be negative")
    q_weight, k_weight = check_weights(q_weight, k_weight, D, device)
    cos, sin, positions, c_sb, c_st = check_angles(cos, sin, positions, tuple(tokens), D, device)
    query, keys = aligned_rows(query, t_axis), aligned_rows(keys, t_axis)
    a = _lib.RotateHeadsArgs()
    a.batch, a.tokens = (1, tokens[0]) if query.dim() == 3 else tokens
    a.Hq, a.Hkv, a.D = query.shape[h_axis], keys.shape[h_axis], D
    a.dtype = _lib.dtype_code(query.dtype)
    a.weight_dtype = _lib.dtype_code(next((w.dtype for w in (q_weight, k_weight) if w is not None), query.dtype))
    set_angles(a, cos, sin, positions, c_sb, c_st, interleaved, eps)
    _strides(a, "q", query), _strides(a, "k", keys)
    return a, query, keys, cos, sin, positions, q_weight, k_weight


def _strides(a, name: str, t: torch.Tensor) -> None:
    sb, sh, st = t.stride()[:3] if t.dim() == 4 else (0, t.stride(1), t.stride(0))
    for field, stride in (("sb", sb), ("st", st), ("sh", sh)):
        setattr(a, f"{name}_{field}", stride)


def _point(a, query, keys, cos, sin, positions, q_weight, k_weight) -> None:
    a.query, a.keys, a.cos, a.sin = query.data_ptr(), keys.data_ptr(), cos.data_ptr(), sin.data_ptr()
    a.positions, a.q_weight, a.k_weight = _lib.ptr(positions), _lib.ptr(q_weight), _lib.ptr(k_weight)


def _forward(query, keys, cos, sin, positions, q_weight, k_weight, eps, interleaved):
    """The outputs, and what a backward pass takes of the call: its arguments, its tensors with aligned rows, and the
    arguments that are kept for its layouts (None where rows had to be copied)."""
    given = (query, keys, cos, sin, positions, q_weight, k_weight)
    key = ("rotate", eps, interleaved, positions is None, q_weight is None, k_weight is None,
           _lib.layouts(*[t for t in given if t is not None]))
    known = _lib.template(key)
    if known is not None and not (query.data_ptr() | keys.data_ptr() | cos.data_ptr() | sin.data_ptr()
                                  | _lib.ptr(q_weight) | _lib.ptr(k_weight)) % 16:
        a, tensors = _lib.RotateHeadsArgs.from_buffer_copy(known), given
        q_out, k_out = (torch.empty_like(query), torch.empty_like(keys)) if known.alike else (new_rows(query), new_rows(keys))
    else:
        a, *tensors = _checked(*given, eps, interleaved)
        q_out, k_out = new_rows(query), new_rows(keys)
        _strides(a, "qo", q_out), _strides(a, "ko", k_out)
        if all(x is y for x, y in zip(given, tensors)):
            a.alike = all(x.stride() == torch.empty_like(y).stride() for x, y in ((q_out, query), (k_out, keys)))
            a.rows, a.backward = _rows_of(*tensors[:4]), {}  # (of backward passes, by the gradients' layouts)
            _lib.keep_template(key, a)
            known, a = a, _lib.RotateHeadsArgs.from_buffer_copy(a)
        else:
            known = None
    if a.tokens and a.batch:
        _point(a, *tensors)
        a.q_out, a.k_out = q_out.data_ptr(), k_out.data_ptr()
        _lib.launch(_lib.load().dkv_rotate_heads, a, query.device, "dkv_rotate_heads")
    return q_out, k_out, a, tensors, known


def _backward(a, tensors, q_grad, k_grad, wanted, like=None, kept=None):
    """Gradients of query, keys and the weights (None where there is none, or ``wanted`` says no).  ``kept``: the arguments
    that are kept for the forward's layouts, with those of its backward passes."""
    query, keys, cos, sin, positions, q_weight, k_weight = tensors
    if getattr(forward_ad, "_current_level", 0) >= 0:
        no_tangents("the gradient of rotate_heads", q_grad, k_grad, query, keys, cos, sin, q_weight, k_weight)
    if kept is not None and kept.alike:
        dq, dk = torch.empty_like(query), torch.empty_like(keys)
    else:
        dq, dk = (new_rows(t) for t in like or (query, keys))
    weights = [w.new_empty(w.shape) if w is not None and want else None
               for w, want in zip((q_weight, k_weight), wanted)]
    if not a.tokens or not a.batch:
        return dq, dk, *(w if w is None else w.zero_() for w in weights)
    key = None if kept is None else (wanted, _lib.layouts(q_grad, k_grad))
    known = None if kept is None else kept.backward.get(key)
    if known is None or (q_grad.data_ptr() | k_grad.data_ptr()) % 16:
        t_axis = 0 if query.dim() == 3 else 2
        given = q_grad, k_grad
        q_grad, k_grad = aligned_rows(q_grad.to(query.dtype), t_axis), aligned_rows(k_grad.to(keys.dtype), t_axis)
        known = _lib.RotateHeadsArgs.from_buffer_copy(a)
        for name, t in (("qg", q_grad), ("kg", k_grad), ("qo", dq), ("ko", dk)):
            _strides(known, name, t)
        known.workspace_bytes = 0
        if any(w is not None for w in weights):
            known.workspace_bytes = _lib.load().dkv_rotate_heads_backward_workspace_bytes(known)
        if kept is not None and q_grad is given[0] and k_grad is given[1]:
            if len(kept.backward) >= _MAX_BACKWARD:
                kept.backward.clear()
            kept.backward[key] = known
    a = _lib.RotateHeadsArgs.from_buffer_copy(known)
    _point(a, *tensors)
    a.q_grad, a.k_grad, a.q_out, a.k_out = q_grad.data_ptr(), k_grad.data_ptr(), dq.data_ptr(), dk.data_ptr()
    a.q_weight_grad, a.k_weight_grad = _lib.ptr(weights[0]), _lib.ptr(weights[1])
    stream = _lib.stream_ptr(query.device)
    if a.workspace_bytes:
        workspace = _workspace(query.device, a.workspace_bytes, stream)
        a.workspace = workspace.data_ptr()
    _lib.launch(_lib.load().dkv_rotate_heads_backward, a, query.device, "dkv_rotate_heads_backward", stream)
    return dq, dk, *weights


def gradients(q_grad, k_grad, query, keys, cos, sin, positions, q_weight, k_weight, eps, interleaved):
    """Gradients of query, keys, q_weight and k_weight (None without one) from those of the outputs."""
    a, *tensors = _checked(query, keys, cos, sin, positions, q_weight, k_weight, eps, interleaved)
    if q_grad.shape != query.shape or k_grad.shape != keys.shape:
        raise ValueError("q_grad and k_grad must have the shapes of query and keys")
    _lib.require_device(q_grad, k_grad)
    return _backward(a, tensors, q_grad, k_grad, (True, True), (query, keys))


def _rows_of(query, keys, cos, sin) -> tuple:
    """What a call's arguments hold of its tensors' layouts, but for their sizes."""
    return query.stride(), keys.stride(), cos.stride(), sin.stride(), query.dtype, cos.dtype


class _RotateHeads(torch.autograd.Function):
    @staticmethod
    def forward(ctx, query, keys, q_weight, k_weight, cos, sin, positions, eps, interleaved):
        q_out, k_out, ctx.args, tensors, ctx.kept = _forward(query, keys, cos, sin, positions, q_weight, k_weight, eps,
                                                             interleaved)
        ctx.rows = _rows_of(*tensors[:4]) if ctx.kept is None else ctx.kept.rows
        ctx.save_for_backward(*tensors)
        return q_out, k_out

    @staticmethod
    @once_differentiable
    def backward(ctx, q_grad, k_grad):
        need, args, kept, tensors = ctx.needs_input_grad, ctx.args, ctx.kept, ctx.saved_tensors
        query, keys, cos, sin, *vectors = tensors  # (vectors: positions and weights)
        # (hooks of saved tensors, such as those that offload them, may give them back in another layout)
        if _rows_of(query, keys, cos, sin) != ctx.rows or not all([t is None or t.is_contiguous() for t in vectors]) \
                or (query.data_ptr() | keys.data_ptr() | cos.data_ptr() | sin.data_ptr()
                    | _lib.ptr(vectors[1]) | _lib.ptr(vectors[2])) % 16:
            (args, *tensors), kept = _checked(*tensors, args.eps, bool(args.interleaved)), None
        dq, dk, dwq, dwk = _backward(args, tensors, q_grad, k_grad, need[2:4], kept=kept)
        return dq if need[0] else None, dk if need[1] else None, dwq, dwk, None, None, None, None, None


def rotate_heads(query: torch.Tensor, keys: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                 positions: Optional[torch.Tensor] = None, *, q_weight: Optional[torch.Tensor] = None,
                 k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                 interleaved: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """RMS norm of each query and key head, then the rotation by its token's position: returns (query, keys).

    ``query`` and ``keys``: packed tokens [T, H, D], or a batch [B, H, T, D] (bf16, fp16 or fp32, head_dim a multiple
    of 8 up to 256, any strides; views of one projection's output need no copy).  ``q_weight`` and ``k_weight`` [D] (any
    of these types, both the same): the norms' weights, x / sqrt(mean(x^2) + eps) * weight; None: no norm.

    The first ``2 * angles`` channels turn, channel i with i + angles, or with ``interleaved`` 2 i with 2 i + 1:
    (a cos - b sin, b cos + a sin); those behind stay.  ``cos`` and ``sin``: with ``positions`` (int32 or int64, [T] or
    [B, T]) tables [positions, angles]; without, each token's own angles, [T, angles], of a batch [B, T, angles] or
    [1, T, angles] too.  A position behind the table makes the turned channels NaN; a negative one is of no token: its
    rows are 0 and have no part in the gradients.

    Computed in fp32 and rounded once; the outputs have the inputs' layout where it has whole rows.  Gradients: of
    query, keys and the weights, with sums in one order (the same result every time); not of cos and sin, and not
    twice.  A backward pass may be captured in a HIP graph with its forward; as for every operation of autograd, no
    eager graph of the same leaves may be alive then.
    """
    if positions is not None and not isinstance(positions, torch.Tensor):
        raise TypeError("positions must be an int32 or int64 tensor")
    given = [t for t in (query, keys, cos, sin, q_weight, k_weight) if t is not None]
    if followed(*given):
        no_tangents("rotate_heads", *given)
        if cos.requires_grad or sin.requires_grad:
            raise RuntimeError("rotate_heads has no gradients of cos and sin; detach them")
        return _RotateHeads.apply(query, keys, q_weight, k_weight, cos, sin, positions, float(eps), bool(interleaved))
    return _forward(query, keys, cos, sin, positions, q_weight, k_weight, float(eps), bool(interleaved))[:2]


__all__ = ["rotate_heads"]
