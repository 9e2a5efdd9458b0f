"""A cache in 8 bits for requests of different lengths: blocks of tokens, found through tables built on the GPU.

``DartKVCache`` holds sequences of one length.  A program that serves requests as they come has requests of
different lengths that begin and end at different times; here each holds blocks of ``block_size`` tokens out of one
pool, in e4m3 with one power-of-two scale per block and KV head:

* ``reserve_blocks`` / ``release_blocks``: block tables and slot maps from the requests' lengths;
* ``fork_blocks``: rows that become copies of others, by holding the same blocks (``shares``); a row that writes into a
  block of others gets a copy of its own when it reserves, whose contents ``copy_blocks`` copies;
* ``compact_blocks``: the blocks in use move to the lowest numbers;
* ``append_blocks``: new keys and values into their slots, and ``append_rotated_blocks`` with the norm and the rotation
  of queries and keys before;
* ``block_attention``: attention of each request's newest tokens over its blocks;
* ``BlockKVCache``: the tensors of all that for a model's layers, and the calls on them.

Everything runs on the GPU without host synchronization, so a decode step (reserve, append, attention) can be
captured in a HIP graph and replayed while the requests grow.  The reference has no counterpart.
"""

from __future__ import annotations

import itertools
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib
from .attention import _workspace
from .prompt import aligned_rows, check_output, int32_vector, no_gradients, scale_factor
from .rotate import check_angles, check_weights, set_angles

BLOCK_SIZES = (16, 32, 64, 128, 256)
MAX_BLOCK_HEAD_DIM = 256
MAX_REQUESTS = 8190
CODE_DTYPE = torch.float8_e4m3fn

_STATUS = ((1, "too few free blocks"), (2, "a request needs more than max_blocks blocks"),
           (4, "a negative token count"), (8, "more new tokens than total"),
           (16, "a source that is not a request"))


def _check_state(table, lengths, free, state, block_size) -> torch.device:
    _lib.require_device(table, lengths, free, state)
    if block_size not in BLOCK_SIZES:
        raise ValueError(f"block_size must be one of {BLOCK_SIZES}")
    device = table.device
    for t, what, dim in ((table, "table", 2), (lengths, "lengths", 1), (free, "free", 1), (state, "state", 1)):
        if t.dtype != torch.int32 or t.dim() != dim or not t.is_contiguous():
            raise TypeError(f"{what} must be a contiguous int32 tensor of {dim} dimension(s)")
        if t.device != device:
            raise ValueError("table, lengths, free and state must be on the same device")
    if lengths.numel() != table.shape[0] or state.numel() != 4 or table.numel() == 0 or free.numel() == 0:
        raise ValueError("table must be [requests, max_blocks], lengths [requests], free [blocks], state [4]")
    if table.shape[0] > MAX_REQUESTS:
        raise ValueError(f"at most {MAX_REQUESTS} requests")
    return device


def _check_shares(shares, free) -> None:
    if not isinstance(shares, torch.Tensor) or shares.dtype != torch.int32 or not shares.is_contiguous():
        raise TypeError("shares must be a contiguous int32 tensor of 1 dimension(s)")
    if shares.shape != free.shape or shares.device != free.device:
        raise ValueError("shares must be [blocks], on the tables' device")


def _tables_args(name, table, lengths, free, state, tokens, block_size, shares=None):
    """Checked arguments of a call on the tables' state, and the counts as an int32 vector."""
    if shares is None:
        key = (name, block_size, _lib.layouts(table, lengths, free, state, *(() if tokens is None else (tokens,))))
    else:
        key = (name, block_size, tokens is None,
               _lib.layouts(table, lengths, free, state, shares, *(() if tokens is None else (tokens,))))
    known = _lib.template(key)
    if known is None or (shares is not None and shares.data_ptr() % 16):
        device = _check_state(table, lengths, free, state, block_size)
        if shares is not None:
            _check_shares(shares, free)
        a = _lib.BlockTablesArgs()
        a.requests, a.max_blocks, a.blocks, a.block_size = table.shape[0], table.shape[1], free.shape[0], block_size
        if shares is not None and name != "reserve":
            a.workspace_bytes = _lib.load().dkv_share_workspace_bytes(a)
        if tokens is not None:
            checked = _counts(tokens, lengths, device)
            if checked is tokens:
                _lib.keep_template(key, a)
            tokens = checked
        else:
            _lib.keep_template(key, a)
        known = a
    a = _lib.BlockTablesArgs.from_buffer_copy(known)
    a.table, a.lengths, a.free, a.state = table.data_ptr(), lengths.data_ptr(), free.data_ptr(), state.data_ptr()
    if tokens is not None:
        a.tokens = tokens.data_ptr()
    if shares is not None:
        a.shares = shares.data_ptr()
    return a, tokens


def _launch_shared(function, a, device, where) -> None:
    """A call whose launches pass their records through a workspace."""
    stream = _lib.stream_ptr(device)
    if a.workspace_bytes:
        workspace = _workspace(device, a.workspace_bytes, stream)
        a.workspace = workspace.data_ptr()
    _lib.launch(function, a, device, where, stream)


def _counts(tokens, lengths, device) -> torch.Tensor:
    tokens = int32_vector(tokens, "tokens", device)
    if tokens.numel() != lengths.numel():
        raise ValueError("tokens must hold one count per request")
    return tokens


def reserve_blocks(table: torch.Tensor, lengths: torch.Tensor, free: torch.Tensor, state: torch.Tensor,
                   tokens: torch.Tensor, total: int, *, block_size: int, shares: Optional[torch.Tensor] = None,
                   positions: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, ...]:
    """Room for ``tokens[r]`` new tokens behind each request's ``lengths[r]``: returns (slots, starts), and with
    ``shares`` (slots, starts, copies).

    ``table`` [requests, max_blocks], ``lengths`` [requests], ``free`` [blocks] and ``state`` [4] (int32, on the
    device) are the tables' state and are updated in place: ``free[:state[0]]`` is the stack of free blocks, of
    which requests take blocks from the top, in their order.  ``tokens``: one count per request, on the device.
    ``total``: how many tokens the caller's packed tensors hold, at least the counts' sum.  ``slots`` [total]
    (int64) is block * block_size + offset of each packed token, -1 behind the last; ``starts`` [requests + 1]
    (int32) each request's first place.

    ``shares`` [blocks] (int32), where requests were forked: a request that gets tokens in a block that others hold
    takes a block for a copy of it first; of the writers of one call that are all its holders the last keeps it.
    ``copies`` [requests, 3] (int32) holds (block, copy, tokens) of each, -1 behind the last: ``copy_blocks`` has to
    make them before the tokens are appended.  ``positions`` [total] (int32) gets each packed token's position in its
    request, -1 behind the last.

    Nothing is read back: a call that cannot be met (too few free blocks, more than max_blocks, a negative count,
    more tokens than total) changes nothing but ``state[1]``, and its slots are -1 and its starts 0, so that
    appends and attention of that call do nothing (``BlockKVCache.check`` raises).
    """
    if not isinstance(tokens, torch.Tensor):
        raise TypeError("tokens must be a one-dimensional int32 or int64 tensor")
    a, tokens = _tables_args("reserve", table, lengths, free, state, tokens, block_size, shares)
    total = int(total)
    if not 0 <= total < 1 << 31:
        raise ValueError("total must not be negative")
    device = table.device
    if positions is not None:
        if positions.dtype != torch.int32 or positions.shape != (total,) or positions.device != device \
                or not positions.is_contiguous() or positions.data_ptr() % 16:
            raise ValueError("positions must be an aligned contiguous int32 [total] tensor on the tables' device")
        a.positions = positions.data_ptr()
    slots = torch.empty(total, dtype=torch.int64, device=device)
    starts = torch.empty(a.requests + 1, dtype=torch.int32, device=device)
    a.slots, a.starts, a.total = slots.data_ptr(), starts.data_ptr(), total
    if shares is None:
        _lib.launch(_lib.load().dkv_reserve_blocks, a, device, "dkv_reserve_blocks")
        return slots, starts
    copies = torch.empty(a.requests, 3, dtype=torch.int32, device=device)
    a.copies = copies.data_ptr()
    _lib.launch(_lib.load().dkv_reserve_blocks, a, device, "dkv_reserve_blocks")
    return slots, starts, copies


def release_blocks(table: torch.Tensor, lengths: torch.Tensor, free: torch.Tensor, state: torch.Tensor,
                   tokens: Optional[torch.Tensor] = None, *, block_size: int,
                   shares: Optional[torch.Tensor] = None) -> None:
    """Drop the last ``tokens[r]`` tokens of each request (None: all of them; more than it has: all it has) and
    return the blocks in which none is left to the free stack.  The exact inverse of ``reserve_blocks`` with the
    same counts: rejected draft tokens are given back as they were taken.  A block that keeps tokens keeps its scale:
    where a dropped token had raised it, those that come later are as coarse as that left it, until the block begins
    anew.

    ``shares`` [blocks] (int32), where requests were forked: a block returns when no request holds it any more, and those
    of a call return in the order of their numbers, the lowest on top of the stack."""
    if tokens is not None and not isinstance(tokens, torch.Tensor):
        raise TypeError("tokens must be a one-dimensional int32 or int64 tensor")
    a, tokens = _tables_args("release", table, lengths, free, state, tokens, block_size, shares)
    if shares is None:
        _lib.launch(_lib.load().dkv_release_blocks, a, table.device, "dkv_release_blocks")
    else:
        _launch_shared(_lib.load().dkv_release_blocks, a, table.device, "dkv_release_blocks")


def fork_blocks(table: torch.Tensor, lengths: torch.Tensor, free: torch.Tensor, state: torch.Tensor,
                shares: torch.Tensor, sources: torch.Tensor, tokens: Optional[torch.Tensor] = None, *,
                block_size: int) -> None:
    """Make request r a copy of what request ``sources[r]`` was before the call, or of its first ``tokens[r]`` tokens
    (None, or more than it has: all); -1 leaves a request as it is.  All requests change at once, so beams go on from
    each other in any order.  What they held before returns to the stack where no request holds it any more, the lowest
    number on top.

    No block is copied: both requests hold it, and ``shares`` [blocks] (int32, zeros at the start) counts the holders
    beside one.  From then on every call on these tables has to be given ``shares``.  A source that is not a request, or
    a negative count, leaves its request as it was and sets ``state[1]`` (``BlockKVCache.check`` raises)."""
    if not isinstance(sources, torch.Tensor) or not (tokens is None or isinstance(tokens, torch.Tensor)):
        raise TypeError("sources and tokens must be one-dimensional int32 or int64 tensors")
    if not isinstance(shares, torch.Tensor):
        raise TypeError("shares must be a contiguous int32 tensor of 1 dimension(s)")
    a, tokens = _tables_args("fork", table, lengths, free, state, tokens, block_size, shares)
    sources = int32_vector(sources, "sources", table.device)
    if sources.numel() != lengths.numel():
        raise ValueError("sources must hold one request per request")
    a.sources = sources.data_ptr()
    _launch_shared(_lib.load().dkv_fork_blocks, a, table.device, "dkv_fork_blocks")


def compact_blocks(table: torch.Tensor, lengths: torch.Tensor, free: torch.Tensor, state: torch.Tensor,
                   shares: Optional[torch.Tensor] = None, *, block_size: int) -> torch.Tensor:
    """Move the blocks in use to the lowest numbers, so that the free ones are the highest and the pool behind them can
    be used otherwise: of n used blocks those numbered n and above go to the free numbers below n, in ascending order.
    Tables, stack and shares follow; returns the ``copies`` [blocks // 2, 3] (block, new number, block_size), -1 behind
    the last, which ``copy_blocks`` has to make in every layer.  At most 2^20 blocks.  Slots given before are no longer
    valid."""
    a, _ = _tables_args("compact", table, lengths, free, state, None, block_size, shares)
    a.workspace_bytes = _lib.load().dkv_share_workspace_bytes(a)
    copies = torch.empty(a.blocks // 2, 3, dtype=torch.int32, device=table.device)
    a.copies = copies.data_ptr()
    _launch_shared(_lib.load().dkv_compact_blocks, a, table.device, "dkv_compact_blocks")
    return copies


def copy_blocks(copies: torch.Tensor, key_codes: torch.Tensor, value_codes: torch.Tensor, key_scale: torch.Tensor,
                value_scale: torch.Tensor) -> None:
    """For each (block, target, tokens) of ``copies`` [n, 3] (int32): the block's first ``tokens`` tokens and its scales
    to the block ``target``, in every layer of ``key_codes``, ``value_codes`` [layers, blocks, heads, block_size,
    head_dim] (e4m3) and ``key_scale``, ``value_scale`` [layers, blocks, heads] (or without layers).  Entries with a
    number outside the blocks are skipped.  No target may be another entry's source or target (the order of copies is
    not defined, and nothing checks it on the device)."""
    key = ("copy", _lib.layouts(copies, key_codes, value_codes, key_scale, value_scale))
    a = _lib.template(key)
    if a is None or (key_codes.data_ptr() | value_codes.data_ptr()) % 16:
        a = _checked_copy(copies, key_codes, value_codes, key_scale, value_scale)
        _lib.keep_template(key, a)
    if a.count == 0:
        return
    a = _lib.CopyBlocksArgs.from_buffer_copy(a)
    a.copies, a.key_codes, a.value_codes = copies.data_ptr(), key_codes.data_ptr(), value_codes.data_ptr()
    a.key_scale, a.value_scale = key_scale.data_ptr(), value_scale.data_ptr()
    _lib.launch(_lib.load().dkv_copy_blocks, a, copies.device, "dkv_copy_blocks")


def _checked_copy(copies, key_codes, value_codes, key_scale, value_scale):
    _lib.require_device(copies, key_codes, value_codes, key_scale, value_scale)
    if copies.dtype != torch.int32 or copies.dim() != 2 or copies.shape[1] != 3 or not copies.is_contiguous():
        raise TypeError("copies must be a contiguous int32 [n, 3] tensor")
    pools = key_codes, value_codes, key_scale, value_scale
    if key_codes.dim() == 4:
        pools = [t.unsqueeze(0) for t in pools]
    if any(t.dim() != dim for t, dim in zip(pools, (5, 5, 3, 3))) or len({t.shape[0] for t in pools}) != 1 \
            or pools[0].shape[0] == 0:
        raise ValueError("key_codes and value_codes must be [layers, blocks, heads, block_size, head_dim], key_scale and "
                         "value_scale [layers, blocks, heads], or all without layers")
    if pools[0].shape != pools[1].shape:
        raise ValueError("key_codes and value_codes must have one shape")
    _check_pool(*(t[0] for t in pools), copies.device)
    layers, blocks, heads, block_size, D = pools[0].shape
    if D == 0 or D % 16 or D > MAX_BLOCK_HEAD_DIM:
        raise ValueError(f"head_dim must be a multiple of 16 up to {MAX_BLOCK_HEAD_DIM}")
    if any(t.data_ptr() % 16 or t.stride(0) % 16 for t in pools[:2]):
        raise ValueError("key_codes and value_codes must have 16-byte aligned layers")
    a = _lib.CopyBlocksArgs()
    a.count, a.layers, a.blocks, a.H, a.block_size, a.D = copies.shape[0], layers, blocks, heads, block_size, D
    a.key_stride, a.value_stride, a.key_scale_stride, a.value_scale_stride = (t.stride(0) for t in pools)
    return a


def _check_pool(key_codes, value_codes, key_scale, value_scale, device):
    if key_codes.dim() != 4 or key_codes.shape != value_codes.shape:
        raise ValueError("key_codes and value_codes must be [blocks, heads, block_size, head_dim]")
    blocks, heads, block_size, _ = key_codes.shape
    for t in (key_codes, value_codes):
        if t.dtype != CODE_DTYPE or not t.is_contiguous():
            raise TypeError("key_codes and value_codes must be contiguous float8_e4m3fn tensors")
    for t in (key_scale, value_scale):
        if t.dtype != torch.float32 or not t.is_contiguous():
            raise TypeError("key_scale and value_scale must be contiguous float32 tensors")
        if t.shape != (blocks, heads):
            raise ValueError("key_scale and value_scale must be [blocks, heads]")
    if any(t.device != device for t in (key_codes, value_codes, key_scale, value_scale)):
        raise ValueError("the tensors must be on the same device")
    if block_size not in BLOCK_SIZES:
        raise ValueError(f"block_size must be one of {BLOCK_SIZES}")
    if blocks == 0 or heads == 0:
        raise ValueError("key_codes must hold blocks and heads")


def append_blocks(keys: torch.Tensor, values: torch.Tensor, slots: torch.Tensor, key_codes: torch.Tensor,
                  value_codes: torch.Tensor, key_scale: torch.Tensor, value_scale: torch.Tensor, *,
                  nonfinite: Optional[torch.Tensor] = None) -> None:
    """Write new ``keys`` and ``values`` [T, heads, head_dim] (bf16, fp16 or fp32) to ``slots`` [T], as
    ``reserve_blocks`` gives them, of the blocks ``key_codes``, ``value_codes`` [blocks, heads, block_size,
    head_dim] (e4m3) with scales ``key_scale``, ``value_scale`` [blocks, heads].

    A block's scale is the least power of two (2^-120 at least) that brings its tokens so far under e4m3's 448;
    codes are value / scale, rounded half to even.  A token at offset 0 begins its block anew.  When later tokens
    raise the scale, the codes before them are rounded to it.  Slots are used once each, a block's next to each
    other and ascending; -1 (and any slot outside the blocks) writes nothing.  NaN and infinities become NaN, do
    not count for the scale, and set ``nonfinite`` (an int32 scalar tensor) to 1.  head_dim: a multiple of 16 up to
    256.  Keys and values that require gradients are refused outside torch.no_grad(), forward-mode tangents always.
    """
    no_gradients("append_blocks", keys, values)
    key = ("append", _lib.layouts(keys, values, slots, key_codes, value_codes, key_scale, value_scale))
    known = _lib.template(key)
    if known is None or (keys.data_ptr() | values.data_ptr()) % 16:
        a, keys, values, slots, whole = _checked_append(keys, values, slots, key_codes, value_codes, key_scale, value_scale)
        if whole:
            _lib.keep_template(key, a)
    else:
        a = known
    device = keys.device
    if nonfinite is not None and (nonfinite.dtype != torch.int32 or nonfinite.numel() != 1
                                  or nonfinite.device != device):
        raise TypeError("nonfinite must be an int32 tensor of one element on the same device")
    if a.tokens == 0:
        return
    a = _lib.AppendBlocksArgs.from_buffer_copy(a)
    a.keys, a.values, a.slots = keys.data_ptr(), values.data_ptr(), slots.data_ptr()
    a.key_codes, a.value_codes = key_codes.data_ptr(), value_codes.data_ptr()
    a.key_scale, a.value_scale = key_scale.data_ptr(), value_scale.data_ptr()
    a.nonfinite = 0 if nonfinite is None else nonfinite.data_ptr()
    _lib.launch(_lib.load().dkv_append_blocks, a, device, "dkv_append_blocks")


def _checked_append(keys, values, slots, key_codes, value_codes, key_scale, value_scale):
    _lib.require_device(keys, values, slots, key_codes, value_codes, key_scale, value_scale)
    device = keys.device
    if keys.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise TypeError("append_blocks takes bf16, fp16 and fp32 keys and values")
    if values.dtype != keys.dtype:
        raise TypeError("keys and values must have one dtype")
    if keys.dim() != 3 or keys.shape != values.shape:
        raise ValueError("keys and values must be [tokens, heads, head_dim]")
    _check_pool(key_codes, value_codes, key_scale, value_scale, device)
    T, H, D = keys.shape
    if (H, D) != (key_codes.shape[1], key_codes.shape[3]):
        raise ValueError("keys and values must have the cache's heads and head_dim")
    if D == 0 or D % 16 or D > MAX_BLOCK_HEAD_DIM:
        raise ValueError(f"head_dim must be a multiple of 16 up to {MAX_BLOCK_HEAD_DIM}")
    if slots.dtype != torch.int64 or slots.shape != (T,):
        raise TypeError("slots must be an int64 tensor with one entry per token")
    if values.device != device or slots.device != device:
        raise ValueError("the tensors must be on the same device")
    given = (keys, values, slots)
    keys, values, slots = aligned_rows(keys, 0), aligned_rows(values, 0), slots.contiguous()
    a = _lib.AppendBlocksArgs()
    a.dtype = _lib.dtype_code(keys.dtype)
    a.k_st, a.k_sh, a.v_st, a.v_sh = keys.stride(0), keys.stride(1), values.stride(0), values.stride(1)
    a.tokens, a.H, a.D = T, H, D
    a.blocks, a.block_size = key_codes.shape[0], key_codes.shape[2]
    return a, keys, values, slots, all(x is y for x, y in zip(given, (keys, values, slots)))


def append_rotated_blocks(query: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, cos: torch.Tensor,
                          sin: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor, key_codes: torch.Tensor,
                          value_codes: torch.Tensor, key_scale: torch.Tensor, value_scale: torch.Tensor, *,
                          q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
                          eps: float = 1e-6, interleaved: bool = False,
                          nonfinite: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``rotate_heads`` of ``query`` [T, Hq, head_dim] and ``keys`` [T, heads, head_dim], and ``append_blocks`` of those
    keys with ``values``, in one launch: returns the queries.

    Arguments as there, with ``positions`` [T] (as ``reserve_blocks`` gives them, the same for all layers) and tables
    ``cos``, ``sin`` [positions, angles], whose angles have to be a multiple of 8.  The keys are rounded to their type
    before they become codes, as between the two calls.  Nothing has a gradient: tensors that require gradients are
    refused outside torch.no_grad(), forward-mode tangents always."""
    if not isinstance(positions, torch.Tensor):
        raise TypeError("positions must be an int32 or int64 tensor")
    given = [t for t in (query, keys, values, cos, sin, q_weight, k_weight) if t is not None]
    no_gradients("append_rotated_blocks", *given)
    tensors = (query, keys, values, cos, sin, positions, slots, key_codes, value_codes, key_scale, value_scale, q_weight,
               k_weight)
    key = ("append_rotated", float(eps), bool(interleaved), q_weight is None, k_weight is None,
           _lib.layouts(*(t for t in tensors if t is not None)))
    known = _lib.template(key)
    if known is None or (query.data_ptr() | keys.data_ptr() | values.data_ptr() | cos.data_ptr() | sin.data_ptr()
                         | _lib.ptr(q_weight) | _lib.ptr(k_weight)) % 16:
        known, checked = _checked_rotated(*tensors, eps, interleaved)
        if all(x is y for x, y in zip(tensors, checked)):
            _lib.keep_template(key, known)
        query, keys, values, cos, sin, positions, slots, *_, q_weight, k_weight = checked
    device = query.device
    if nonfinite is not None and (nonfinite.dtype != torch.int32 or nonfinite.numel() != 1
                                  or nonfinite.device != device):
        raise TypeError("nonfinite must be an int32 tensor of one element on the same device")
    out = torch.empty(query.shape, dtype=query.dtype, device=device)
    if query.shape[0] == 0:
        return out
    a, r = (type(x).from_buffer_copy(x) for x in known)
    a.keys, a.values, a.slots = keys.data_ptr(), values.data_ptr(), slots.data_ptr()
    a.key_codes, a.value_codes = key_codes.data_ptr(), value_codes.data_ptr()
    a.key_scale, a.value_scale = key_scale.data_ptr(), value_scale.data_ptr()
    a.nonfinite = _lib.ptr(nonfinite)
    r.query, r.q_out, r.cos, r.sin, r.positions = (t.data_ptr() for t in (query, out, cos, sin, positions))
    r.q_weight, r.k_weight = _lib.ptr(q_weight), _lib.ptr(k_weight)
    lib = _lib.load()
    _lib.launch(lambda args, stream: lib.dkv_append_rotated_blocks(args, r, stream), a, device, "dkv_append_rotated_blocks")
    return out


def _checked_rotated(query, keys, values, cos, sin, positions, slots, key_codes, value_codes, key_scale, value_scale,
                     q_weight, k_weight, eps, interleaved):
    _lib.require_device(query, cos, sin, positions, q_weight, k_weight)
    a, keys, values, slots, _ = _checked_append(keys, values, slots, key_codes, value_codes, key_scale, value_scale)
    device, D = keys.device, a.D
    if query.dtype != keys.dtype:
        raise TypeError("query and keys must have one dtype")
    if query.dim() != 3 or query.shape[0] != a.tokens or query.shape[1] == 0 or query.shape[2] != D:
        raise ValueError("query must be [tokens, heads, head_dim], of the keys' tokens and head_dim")
    if query.device != device:
        raise ValueError("the tensors must be on the same device")
    if cos.shape[-1] % 8:
        raise ValueError("append_rotated_blocks takes angles in multiples of 8; else use rotate_heads and append_blocks")
    if not 0 <= eps < 1e30:
        raise ValueError("eps must not be negative")
    q_weight, k_weight = check_weights(q_weight, k_weight, D, device)
    cos, sin, positions, c_sb, c_st = check_angles(cos, sin, positions, (a.tokens,), D, device)
    query = aligned_rows(query, 0)
    r = _lib.RotateHeadsArgs()
    r.batch, r.tokens, r.Hq, r.Hkv, r.D = 1, a.tokens, query.shape[1], a.H, D
    r.q_st, r.q_sh, r.qo_st, r.qo_sh = query.stride(0), query.stride(1), query.shape[1] * D, D
    r.dtype = a.dtype
    r.weight_dtype = _lib.dtype_code(next((w.dtype for w in (q_weight, k_weight) if w is not None), query.dtype))
    set_angles(r, cos, sin, positions, c_sb, c_st, interleaved, eps)
    return (a, r), (query, keys, values, cos, sin, positions, slots, key_codes, value_codes, key_scale, value_scale,
                    q_weight, k_weight)


def block_attention(query: torch.Tensor, key_codes: torch.Tensor, value_codes: torch.Tensor, key_scale: torch.Tensor,
                    value_scale: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor,
                    starts: Optional[torch.Tensor] = None, *, max_tokens: Optional[int] = None,
                    scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of each request's newest tokens over its blocks, their own keys and values among them.

    ``query`` [T, Hq, D] (bf16 or fp16) holds the requests' new tokens one after the other, request r's in rows
    ``starts[r]`` to ``starts[r + 1]`` (``reserve_blocks``; None: one token each); the last is at position
    ``lengths[r] - 1``, so token i of n sees the first ``lengths[r] - n + 1 + i`` keys, and a row that sees none is
    0.  ``max_tokens``: no request has more new tokens in this call; where that is at most 64 rows (tokens times
    query heads per KV head) the kernel for few rows does all of it, and the output rows of a request that has
    more after all are undefined.  Default: T (without starts 1).
    ``table`` [requests, max_blocks] and ``lengths`` [requests] (int32), the codes and scales as ``append_blocks``
    writes them: the scales have to be powers of two (of others the kernels use different parts; nothing checks that
    on the device).  Bytes of a block behind its request's length are not used.  A table entry outside the blocks
    makes the rows that see it NaN.  Returns a tensor like ``query``, or ``out``; rows behind the last request and
    before the first are 0 in a new tensor and stay as they were in ``out``.  ``scale`` (1e-37 to 1e30) defaults to
    1 / sqrt(D).

    Statistics and sums are fp32; the weights keep 16 bits for the second product, but for a bf16 query's requests of
    more rows than the kernel for few takes, where they are rounded to bf16.  Forward only: a query that requires
    gradients is refused outside torch.no_grad(), forward-mode tangents always.
    """
    fill = out is None
    scale = None if scale is None else float(scale)
    max_tokens = None if max_tokens is None else int(max_tokens)
    key = None
    if starts is None or (isinstance(starts, torch.Tensor) and starts.dtype == torch.int32):
        key = ("attend", max_tokens, scale, fill,
               _lib.layouts(query, key_codes, value_codes, key_scale, value_scale, table, lengths,
                            *(() if starts is None else (starts,)), *(() if fill else (out,))), starts is None)
    known = _lib.template(key) if key is not None else None
    if known is not None and not query.data_ptr() % 16 and (fill or not out.data_ptr() % 8):
        no_gradients("block_attention", query)
        a = known
    else:
        a, query, starts, whole = _checked_attention(query, key_codes, value_codes, key_scale, value_scale, table,
                                                     lengths, starts, max_tokens, scale, out)
        if whole and key is not None:
            _lib.keep_template(key, a)
    device = query.device
    if fill:
        out = torch.empty(query.shape, dtype=query.dtype, device=device)
    if a.tokens == 0:
        return out
    stream = _lib.stream_ptr(device)
    a = _lib.BlockAttentionArgs.from_buffer_copy(a)
    workspace = _workspace(device, a.workspace_bytes, stream)
    a.query, a.out, a.workspace = query.data_ptr(), out.data_ptr(), workspace.data_ptr()
    if starts is not None:
        a.starts = starts.data_ptr()
    a.table, a.lengths = table.data_ptr(), lengths.data_ptr()
    a.key_codes, a.value_codes = key_codes.data_ptr(), value_codes.data_ptr()
    a.key_scale, a.value_scale = key_scale.data_ptr(), value_scale.data_ptr()
    _lib.launch(_lib.load().dkv_block_attention, a, device, "dkv_block_attention", stream)
    return out


def _checked_attention(query, key_codes, value_codes, key_scale, value_scale, table, lengths, starts, max_tokens, scale,
                       out):
    _lib.require_device(query, key_codes, value_codes, key_scale, value_scale, table, lengths)
    device = query.device
    if query.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError("block_attention takes bf16 and fp16 queries")
    if query.dim() != 3:
        raise ValueError("query must have shape [tokens, heads, head_dim]")
    _check_pool(key_codes, value_codes, key_scale, value_scale, device)
    no_gradients("block_attention", query)
    T, Hq, D = query.shape
    blocks, Hkv, block_size, _ = key_codes.shape
    if D != key_codes.shape[3] or D == 0 or D % 16 or D > MAX_BLOCK_HEAD_DIM:
        raise ValueError(f"query and cache must have one head_dim, a multiple of 16 up to {MAX_BLOCK_HEAD_DIM}")
    if Hq == 0 or Hq % Hkv:
        raise ValueError("query heads must be divisible by cache KV heads")
    if table.dtype != torch.int32 or table.dim() != 2 or not table.is_contiguous() or table.numel() == 0:
        raise TypeError("table must be a contiguous int32 [requests, max_blocks] tensor")
    if lengths.dtype != torch.int32 or lengths.shape != (table.shape[0],) or not lengths.is_contiguous():
        raise TypeError("lengths must be a contiguous int32 [requests] tensor")
    if table.device != device or lengths.device != device:
        raise ValueError("the tensors must be on the same device")
    given = (query, starts)
    if starts is None:
        if T != table.shape[0]:
            raise ValueError("without starts the query holds one token per request")
        most = 1
    else:
        starts = int32_vector(starts, "starts", device)
        if starts.numel() != table.shape[0] + 1:
            raise ValueError("starts must hold one more entry than there are requests")
        most = max(1, T)
    if max_tokens is not None:
        if max_tokens < 1:
            raise ValueError("max_tokens must be positive")
        most = min(most, int(max_tokens))
    factor = scale_factor(scale, D, "block_attention")
    fill = out is None
    if not fill:
        check_output(out, query)
    query = aligned_rows(query, 0)
    a = _lib.BlockAttentionArgs()
    a.dtype = _lib.dtype_code(query.dtype)
    a.q_st, a.q_sh = query.stride(0), query.stride(1)
    a.o_st, a.o_sh = (Hq * D, D) if fill else out.stride()[:2]
    a.tokens = T
    a.requests, a.max_blocks = table.shape
    a.blocks, a.block_size = blocks, block_size
    a.Hq, a.Hkv, a.D = Hq, Hkv, D
    a.scale, a.max_tokens, a.fill = factor, most, fill
    a.workspace_bytes = _lib.load().dkv_block_attention_workspace_bytes(a)
    return a, query, starts, query is given[0] and starts is given[1]


_steps = itertools.count(1)  # one line of steps for all caches, so that none takes another's plan


class BlockPlan(NamedTuple):
    """Where a step's new tokens go: ``reserve_blocks``' slots and starts, the most tokens of a request, the
    step of one cache that they belong to, and the tokens' positions where they were asked for."""

    slots: torch.Tensor
    starts: torch.Tensor
    max_tokens: int
    step: int
    positions: Optional[torch.Tensor] = None


class BlockKVCache:
    """The block tables of ``requests`` rows and, for each of ``layers`` layers, ``blocks`` e4m3 blocks.

    A step of a serving loop: ``plan = cache.reserve(tokens, total)`` once, then per layer ``cache.append(layer,
    keys, values, plan)`` and ``cache.attention(layer, query, plan)``.  ``release`` gives back a request's last
    tokens, or all of them.  Nothing synchronizes; ``check`` reads the status once and raises.

    ``max_blocks``: the most blocks of a request (default: all).  Attention of chunks plans its parts and workspace for
    requests of that length, so a bound that the program knows is worth giving.

    A plan of an earlier step, or of another cache, is refused.  Replays of a captured step move the requests on
    without this object's knowledge: after one, no plan made outside the graph before it may be used.
    """

    def __init__(self, requests: int, blocks: int, kv_heads: int, head_dim: int, *, layers: int = 1,
                 block_size: int = 64, max_blocks: Optional[int] = None, sharing: bool = False, device="cuda") -> None:
        if block_size not in BLOCK_SIZES:
            raise ValueError(f"block_size must be one of {BLOCK_SIZES}")
        if min(requests, blocks, kv_heads, layers) < 1 or requests > MAX_REQUESTS:
            raise ValueError(f"requests (at most {MAX_REQUESTS}), blocks, kv_heads and layers must be positive")
        if head_dim < 16 or head_dim % 16 or head_dim > MAX_BLOCK_HEAD_DIM:
            raise ValueError(f"head_dim must be a multiple of 16 up to {MAX_BLOCK_HEAD_DIM}")
        max_blocks = blocks if max_blocks is None else max_blocks
        if max_blocks < 1:
            raise ValueError("max_blocks must be positive")
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError("BlockKVCache lives on a ROCm GPU (dartkv_amd has no CPU path)")
        self.block_size = block_size
        shape = (layers, blocks, kv_heads, block_size, head_dim)
        # (zeros: fp8 tensors have no fill of their own)
        self.key_codes = torch.zeros(shape, dtype=torch.uint8, device=device).view(CODE_DTYPE)
        self.value_codes = torch.zeros(shape, dtype=torch.uint8, device=device).view(CODE_DTYPE)
        self.key_scale = torch.ones(shape[:3], dtype=torch.float32, device=device)
        self.value_scale = torch.ones(shape[:3], dtype=torch.float32, device=device)
        self.table = torch.full((requests, max_blocks), -1, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(requests, dtype=torch.int32, device=device)
        self.free = torch.arange(blocks - 1, -1, -1, dtype=torch.int32, device=device)
        self.state = torch.tensor([blocks, 0, 0, 0], dtype=torch.int32, device=device)
        self.shares = torch.zeros(blocks, dtype=torch.int32, device=device) if sharing else None
        self.nonfinite = torch.zeros(1, dtype=torch.int32, device=device)
        self._step = next(_steps)

    def _check_plan(self, plan: BlockPlan) -> None:
        if plan.step != self._step:
            raise ValueError("the plan is of an earlier reserve, whose requests' lengths have moved on, or of another cache")

    @property
    def _tables(self) -> Tuple[torch.Tensor, ...]:
        return self.table, self.lengths, self.free, self.state

    @property
    def _pools(self) -> Tuple[torch.Tensor, ...]:
        return self.key_codes, self.value_codes, self.key_scale, self.value_scale

    def reserve(self, tokens: torch.Tensor, total: int, *, max_tokens: Optional[int] = None,
                positions: bool = False) -> BlockPlan:
        """Room for ``tokens[r]`` new tokens of each request (``reserve_blocks``).  ``max_tokens``: the most of
        them, where the caller knows it (default ``total``); ``attention`` leaves the rows of a request with more
        undefined.  A decode step without it also launches the kernel for chunks, which finds nothing to do.
        ``positions``: the plan has the tokens' positions, for ``append_rotated``."""
        places = torch.empty(int(total), dtype=torch.int32, device=self.table.device) if positions else None
        slots, starts, *copies = reserve_blocks(*self._tables, tokens, total, block_size=self.block_size,
                                                shares=self.shares, positions=places)
        for more in copies:
            copy_blocks(more, *self._pools)
        self._step = next(_steps)
        return BlockPlan(slots, starts, max(1, total if max_tokens is None else max_tokens), self._step, places)

    def release(self, tokens: Optional[torch.Tensor] = None) -> None:
        """Drop each request's last ``tokens[r]`` tokens, or everything (``release_blocks``)."""
        release_blocks(*self._tables, tokens, block_size=self.block_size, shares=self.shares)
        self._step = next(_steps)

    def fork(self, sources: torch.Tensor, tokens: Optional[torch.Tensor] = None) -> None:
        """Make each request r a copy of request ``sources[r]`` as it is now, or of its first ``tokens[r]`` tokens; -1
        leaves it as it is (``fork_blocks``).  The cache has to be made with ``sharing``."""
        if self.shares is None:
            raise ValueError("the cache was made without sharing")
        fork_blocks(*self._tables, self.shares, sources, tokens, block_size=self.block_size)
        self._step = next(_steps)

    def compact(self) -> torch.Tensor:
        """Move the blocks in use to the lowest numbers, in all layers (``compact_blocks``): those from
        ``blocks - state[0]`` on are free afterwards.  Returns the copies that were made."""
        copies = compact_blocks(*self._tables, self.shares, block_size=self.block_size)
        copy_blocks(copies, *self._pools)
        self._step = next(_steps)
        return copies

    def append(self, layer: int, keys: torch.Tensor, values: torch.Tensor, plan: BlockPlan) -> None:
        """The step's new ``keys`` and ``values`` [T, kv_heads, head_dim] of one layer (``append_blocks``)."""
        self._check_plan(plan)
        append_blocks(keys, values, plan.slots, self.key_codes[layer], self.value_codes[layer], self.key_scale[layer],
                      self.value_scale[layer], nonfinite=self.nonfinite)

    def append_rotated(self, layer: int, query: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, cos: torch.Tensor,
                       sin: torch.Tensor, plan: BlockPlan, *, q_weight: Optional[torch.Tensor] = None,
                       k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                       interleaved: bool = False) -> torch.Tensor:
        """``append`` of keys that are normed and turned by their positions on the way, and the queries likewise: returns
        these (``append_rotated_blocks``).  The plan has to be made with ``positions``."""
        self._check_plan(plan)
        if plan.positions is None:
            raise ValueError("the plan has no positions; reserve with positions=True")
        return append_rotated_blocks(query, keys, values, cos, sin, plan.positions, plan.slots, self.key_codes[layer],
                                     self.value_codes[layer], self.key_scale[layer], self.value_scale[layer],
                                     q_weight=q_weight, k_weight=k_weight, eps=eps, interleaved=interleaved,
                                     nonfinite=self.nonfinite)

    def attention(self, layer: int, query: torch.Tensor, plan: BlockPlan, *, scale: Optional[float] = None,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of the step's ``query`` [T, heads, head_dim] over one layer's blocks (``block_attention``),
        after the layer's ``append`` and before the next ``reserve`` or ``release``."""
        self._check_plan(plan)
        return block_attention(query, self.key_codes[layer], self.value_codes[layer], self.key_scale[layer],
                               self.value_scale[layer], self.table, self.lengths, plan.starts,
                               max_tokens=plan.max_tokens, scale=scale, out=out)

    def check(self) -> None:
        """Raise what the calls so far could not do (one host synchronization), and clear it."""
        status, nonfinite = int(self.state[1]), int(self.nonfinite)
        if status:
            self.state[1] = 0
            raise RuntimeError("block cache: " + ", ".join(text for bit, text in _STATUS if status & bit))
        if nonfinite:
            self.nonfinite.zero_()
            raise ValueError("append_blocks requires finite keys and values")


__all__ = ["BlockKVCache", "BlockPlan", "append_blocks", "append_rotated_blocks", "block_attention", "compact_blocks",
           "copy_blocks", "fork_blocks", "release_blocks", "reserve_blocks"]
