"""A cache in 8 bits for requests of different lengths: blocks of tokens, found through tables built on the GPU.

``DartKVCache`` holds sequences of one length.  A program that serves requests as they come has requests of
different lengths that begin and end at different times; here each holds blocks of ``block_size`` tokens out of one
pool, in e4m3 with one power-of-two scale per block and KV head:

* ``reserve_blocks`` / ``release_blocks``: block tables and slot maps from the requests' lengths;
* ``append_blocks``: new keys and values into their slots;
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

BLOCK_SIZES = (16, 32, 64, 128, 256)
MAX_BLOCK_HEAD_DIM = 256
MAX_REQUESTS = 8190
CODE_DTYPE = torch.float8_e4m3fn

_STATUS = ((1, "too few free blocks"), (2, "a request needs more than max_blocks blocks"),
           (4, "a negative token count"), (8, "more new tokens than total"))


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


def _tables_args(name, table, lengths, free, state, tokens, block_size):
    """Checked arguments of a call on the tables' state, and the counts as an int32 vector."""
    key = (name, block_size, _lib.layouts(table, lengths, free, state, *(() if tokens is None else (tokens,))))
    known = _lib.template(key)
    if known is None:
        device = _check_state(table, lengths, free, state, block_size)
        a = _lib.BlockTablesArgs()
        a.requests, a.max_blocks, a.blocks, a.block_size = table.shape[0], table.shape[1], free.shape[0], block_size
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
    return a, tokens


def _counts(tokens, lengths, device) -> torch.Tensor:
    tokens = int32_vector(tokens, "tokens", device)
    if tokens.numel() != lengths.numel():
        raise ValueError("tokens must hold one count per request")
    return tokens


def reserve_blocks(table: torch.Tensor, lengths: torch.Tensor, free: torch.Tensor, state: torch.Tensor,
                   tokens: torch.Tensor, total: int, *, block_size: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """Room for ``tokens[r]`` new tokens behind each request's ``lengths[r]``: returns (slots, starts).

    ``table`` [requests, max_blocks], ``lengths`` [requests], ``free`` [blocks] and ``state`` [4] (int32, on the
    device) are the tables' state and are updated in place: ``free[:state[0]]`` is the stack of free blocks, of
    which requests take blocks from the top, in their order.  ``tokens``: one count per request, on the device.
    ``total``: how many tokens the caller's packed tensors hold, at least the counts' sum.  ``slots`` [total]
    (int64) is block * block_size + offset of each packed token, -1 behind the last; ``starts`` [requests + 1]
    (int32) each request's first place.

    Nothing is read back: a call that cannot be met (too few free blocks, more than max_blocks, a negative count,
    more tokens than total) changes nothing but ``state[1]``, and its slots are -1 and its starts 0, so that
    appends and attention of that call do nothing (``BlockKVCache.check`` raises).
    """
    if not isinstance(tokens, torch.Tensor):
        raise TypeError("tokens must be a one-dimensional int32 or int64 tensor")
    a, tokens = _tables_args("reserve", table, lengths, free, state, tokens, block_size)
    total = int(total)
    if not 0 <= total < 1 << 31:
        raise ValueError("total must not be negative")
    device = table.device
    slots = torch.empty(total, dtype=torch.int64, device=device)
    starts = torch.empty(a.requests + 1, dtype=torch.int32, device=device)
    a.slots, a.starts, a.total = slots.data_ptr(), starts.data_ptr(), total
    _lib.launch(_lib.load().dkv_reserve_blocks, a, device, "dkv_reserve_blocks")
    return slots, starts


def release_blocks(table: torch.Tensor, lengths: torch.Tensor, free: torch.Tensor, state: torch.Tensor,
                   tokens: Optional[torch.Tensor] = None, *, block_size: int) -> None:
    """Drop the last ``tokens[r]`` tokens of each request (None: all of them; more than it has: all it has) and
    return the blocks in which none is left to the free stack.  The exact inverse of ``reserve_blocks`` with the
    same counts: rejected draft tokens are given back as they were taken.  A block that keeps tokens keeps its scale:
    where a dropped token had raised it, those that come later are as coarse as that left it, until the block begins
    anew."""
    if tokens is not None and not isinstance(tokens, torch.Tensor):
        raise TypeError("tokens must be a one-dimensional int32 or int64 tensor")
    a, tokens = _tables_args("release", table, lengths, free, state, tokens, block_size)
    _lib.launch(_lib.load().dkv_release_blocks, a, table.device, "dkv_release_blocks")


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
    """Where a step's new tokens go: ``reserve_blocks``' slots and starts, the most tokens of a request, and the
    step of one cache that they belong to."""

    slots: torch.Tensor
    starts: torch.Tensor
    max_tokens: int
    step: int


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
                 block_size: int = 64, max_blocks: Optional[int] = None, device="cuda") -> None:
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
        self.nonfinite = torch.zeros(1, dtype=torch.int32, device=device)
        self._step = next(_steps)

    def _check_plan(self, plan: BlockPlan) -> None:
        if plan.step != self._step:
            raise ValueError("the plan is of an earlier reserve, whose requests' lengths have moved on, or of another cache")

    def reserve(self, tokens: torch.Tensor, total: int, *, max_tokens: Optional[int] = None) -> BlockPlan:
        """Room for ``tokens[r]`` new tokens of each request (``reserve_blocks``).  ``max_tokens``: the most of
        them, where the caller knows it (default ``total``); ``attention`` leaves the rows of a request with more
        undefined.  A decode step without it also launches the kernel for chunks, which finds nothing to do."""
        slots, starts = reserve_blocks(self.table, self.lengths, self.free, self.state, tokens, total,
                                       block_size=self.block_size)
        self._step = next(_steps)
        return BlockPlan(slots, starts, max(1, total if max_tokens is None else max_tokens), self._step)

    def release(self, tokens: Optional[torch.Tensor] = None) -> None:
        """Drop each request's last ``tokens[r]`` tokens, or everything (``release_blocks``)."""
        release_blocks(self.table, self.lengths, self.free, self.state, tokens, block_size=self.block_size)
        self._step = next(_steps)

    def append(self, layer: int, keys: torch.Tensor, values: torch.Tensor, plan: BlockPlan) -> None:
        """The step's new ``keys`` and ``values`` [T, kv_heads, head_dim] of one layer (``append_blocks``)."""
        self._check_plan(plan)
        append_blocks(keys, values, plan.slots, self.key_codes[layer], self.value_codes[layer], self.key_scale[layer],
                      self.value_scale[layer], nonfinite=self.nonfinite)

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


__all__ = ["BlockKVCache", "BlockPlan", "append_blocks", "block_attention", "release_blocks", "reserve_blocks"]
