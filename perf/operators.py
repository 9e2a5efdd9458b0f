"""The operators that serve requests of different lengths: what each computes, in plain torch, and the
calls that a program makes of the framework's own.

Four kinds of work:

* ``prompt``: causal attention of whole prompts, packed one after the other or as a batch, grouped heads;
* ``attend``: attention of each request's new tokens over its cache, held in e4m3 blocks of tokens with
  one scale per block and KV head, found through a block table;
* ``append``: new keys and values into those blocks, scales and codes;
* ``tables``: the block tables and slot maps, from the requests' lengths: rows give tokens back and
  take as many again, so a pass leaves the state as it found it.

Keys are N(0, 1) with a sixteenth of the channels of each KV head scaled by 10, values and queries N(0, 1).
"""

import itertools
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0
MIN_EXPONENT, MAX_EXPONENT = -120, 121  # of a block's scale


def _case(name, kind, R, lo, hi, **over):
    """R requests whose lengths are spread over [lo, hi]; ``new``: the most new tokens of a request."""
    case = dict(name=name, kind=kind, R=R, lo=lo, hi=hi, H=8, G=4, D=128, dtype="bf16", bs=64, new=1, batch=False,
                shape=1)
    case.update(over)
    return case


def listed():
    return [
        # one short chat prompt, a [B, H, T, D] batch of one: what the model adapter's prefill hands over
        _case("prompt_single", "prompt", 1, 1024, 1024, batch=True),
        # a packed batch of ragged prompts, as a scheduler admits them
        _case("prompt_packed", "prompt", 16, 64, 4096),
        # one long prompt
        _case("prompt_long", "prompt", 1, 16384, 16384),
        # a small model's heads in fp16, six query heads per KV head, odd lengths
        _case("prompt_head64", "prompt", 5, 501, 3001, D=64, G=6, dtype="fp16"),
        # one interactive request, one new token: latency
        _case("attend_single", "attend", 1, 4000, 4000),
        # long contexts at full batch, ragged, one token each: the bandwidth case
        _case("attend_batch", "attend", 64, 2048, 32768),
        # speculative decoding: four drafted tokens, eight query heads per KV head, fp16, large blocks
        _case("attend_draft", "attend", 16, 500, 8000, G=8, dtype="fp16", bs=128, new=4),
        # chunks of prompts beside single tokens in one call (continuous batching)
        _case("attend_chunk", "attend", 8, 1000, 8192, new=512),
        # a decode step's new tokens, one for each of a full batch, partly filled blocks
        _case("append_step", "append", 64, 100, 2000),
        # packed prompts written at once
        _case("append_prompts", "append", 16, 1000, 8192, new=8192),
        # a decode step of a full batch: one slot for each request
        _case("tables_step", "tables", 256, 1, 8000, bs=16),
        # finished requests make room, and prompts of several thousand tokens take it
        _case("tables_prompts", "tables", 128, 1, 8192, new=8192),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed ranges, sizes spread over their logarithm."""
    kind = rng.choice(["prompt", "prompt", "attend", "attend", "append", "tables"])
    hi = _log_int(rng, 16, {"prompt": 8192, "attend": 32768, "append": 16384, "tables": 16384}[kind])
    lo = max(1, int(hi * rng.choice([0.02, 0.3, 1.0])))
    H = rng.choice([1, 2, 4, 8])
    D = rng.choice([64, 128, 128, 80, 256])
    over = dict(H=H, G=rng.randint(1, 8), D=D, dtype=rng.choice(["bf16", "bf16", "fp16"]),
                bs=rng.choice([16, 32, 64, 64, 128]), shape=rng.randint(1, 1 << 20))
    heads = H * over["G"]
    if kind == "prompt":
        R = _log_int(rng, 1, max(1, min(64, (1 << 39) // (D * heads * hi * hi))))
        over["batch"] = lo == hi and rng.random() < 0.5
    elif kind == "attend":
        R = _log_int(rng, 1, max(1, min(128, (1 << 30) // (H * hi * D))))
        new = rng.choice([1, 1, 2, 5, 64, 700])
        over["new"] = max(1, min(new, hi, (1 << 31) // (R * heads * hi)))
    elif kind == "append":
        R = _log_int(rng, 1, max(1, min(128, (1 << 26) // (H * hi * D))))
        over["new"] = rng.choice([1, 1, 3, hi, hi])
        over["dtype"] = rng.choice(["bf16", "fp16", "fp32"])
    else:
        R = _log_int(rng, 1, max(1, min(1024, (1 << 20) // hi)))
        over["new"] = rng.choice([1, 4, hi])
    case = _case("", kind, R, lo, hi, **over)
    del case["name"]
    return case


def _lengths(case):
    """Each request's length, its new tokens among them, and how many those are."""
    rng = random.Random(case["shape"])
    lengths = [rng.randint(case["lo"], case["hi"]) for _ in range(case["R"])]
    lengths[0] = case["hi"]
    if case["kind"] == "prompt":
        return lengths, lengths
    # of many new tokens every third request has just one: it decodes beside the others' prompts
    return lengths, [min(n, case["new"]) if case["new"] < 8 or i % 3 != 2 or case["kind"] == "append" else 1
                     for i, n in enumerate(lengths)]


def _starts(counts):
    return list(itertools.accumulate(counts, initial=0))


def _generator(seed, device="cuda"):
    return torch.Generator(device=device).manual_seed(seed)


def _key_factor(case, seed):
    """[H, D]: 10 for a sixteenth of each KV head's channels, 1 for the others."""
    host = _generator(seed + 1, "cpu")
    order = torch.rand(case["H"], case["D"], generator=host).argsort(-1)
    return torch.where(order < case["D"] // 16, 10.0, 1.0).cuda()


def _qkv(case, seed, tokens):
    """Queries [tokens, H * G, D] and keys and values [tokens, H, D] of the case's type."""
    gen, H, D = _generator(seed), case["H"], case["D"]
    q = torch.randn(tokens, H * case["G"], D, generator=gen, device="cuda")
    k = torch.randn(tokens, H, D, generator=gen, device="cuda") * _key_factor(case, seed)
    v = torch.randn(tokens, H, D, generator=gen, device="cuda")
    return [t.to(DTYPES[case["dtype"]]) for t in (q, k, v)]


def _block_scale(amax):
    """The least power of two s with amax <= 448 s, as fp32 (the least of all for a block of zeros)."""
    mantissa, exponent = torch.frexp(amax)  # amax = mantissa * 2^exponent, mantissa in [1/2, 1); 448 = 7/8 * 2^9
    exponent = exponent - 9 + (mantissa > 0.875).to(exponent.dtype)
    exponent = torch.where(amax > 0, exponent, MIN_EXPONENT).clamp(MIN_EXPONENT, MAX_EXPONENT)
    return torch.ldexp(torch.ones_like(amax), exponent)


def _random_blocks(case, seed, blocks, factor):
    """Codes [blocks, H, bs, D] and scales [blocks, H] of random rows."""
    x = torch.randn(blocks, case["H"], case["bs"], case["D"], generator=_generator(seed), device="cuda")
    if factor is not None:
        x *= factor[None, :, None, :]
    scale = _block_scale(x.abs().amax((-1, -2)))
    return (x / scale[..., None, None]).to(E4M3), scale


def _tables(case, seed, held):
    """A block table with ``held`` tokens of each request, the lengths, the free stack and its state
    [free blocks, status, 0, 0]: blocks in random order, as after a while of serving."""
    lengths, _ = _lengths(case)
    bs = case["bs"]
    most = max(-(-n // bs) for n in lengths)
    total = sum(-(-n // bs) for n in lengths) + 3
    order = torch.randperm(total, generator=_generator(seed + 2, "cpu"), dtype=torch.int32)
    table = torch.full((case["R"], most), -1, dtype=torch.int32)
    used = torch.arange(most) < torch.tensor([-(-n // bs) for n in held])[:, None]
    at = int(used.sum())
    table[used] = order[:at]
    free = torch.full((total,), -1, dtype=torch.int32)
    free[:total - at] = order[at:]
    state = torch.tensor([total - at, 0, 0, 0], dtype=torch.int32)
    return table.cuda(), torch.tensor(held, dtype=torch.int32).cuda(), free.cuda(), state.cuda(), total


def prepare(case, seed):
    lengths, new = _lengths(case)
    kind, H, D = case["kind"], case["H"], case["D"]
    if kind == "prompt":
        q, k, v = _qkv(case, seed, sum(lengths))
        if case["batch"]:  # [B, H, T, D] views of the projections' [B, T, H, D]
            q, k, v = (t.view(case["R"], case["hi"], -1, D).transpose(1, 2) for t in (q, k, v))
            return {"kind": "batch", "q": q, "k": k, "v": v}
        starts = torch.tensor(_starts(lengths), dtype=torch.int32).cuda()
        return {"kind": kind, "q": q, "k": k, "v": v, "starts": starts, "most": max(lengths)}
    if kind == "tables":
        table, held, free, state, _ = _tables(case, seed, lengths)
        return {"kind": kind, "table": table, "lengths": held, "free": free, "state": state, "bs": case["bs"],
                "new": torch.tensor(new, dtype=torch.int32).cuda(), "total": sum(new)}
    table, held, _, _, blocks = _tables(case, seed, lengths)
    starts = torch.tensor(_starts(new), dtype=torch.int32).cuda()
    kcode, kscale = _random_blocks(case, seed + 3, blocks, _key_factor(case, seed))
    vcode, vscale = _random_blocks(case, seed + 4, blocks, None)
    out = {"kind": kind, "keys": kcode, "values": vcode, "kscale": kscale, "vscale": vscale}
    if kind == "attend":
        q = _qkv({**case, "H": H * case["G"], "G": 1}, seed, sum(new))[0]
        return {**out, "q": q, "table": table, "lengths": held, "starts": starts, "most": max(new)}
    # append: the slots of the new tokens, the last ones of each request
    _, k, v = _qkv({**case, "G": 1}, seed, sum(new))
    slots = _slots(table, held - (starts[1:] - starts[:-1]), starts, sum(new), case["bs"])
    return {**out, "k": k, "v": v, "slots": slots}


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    import dartkv_amd as dart

    kind = state["kind"]
    if kind == "batch":
        return dart.prompt_attention(state["q"], state["k"], state["v"])
    if kind == "prompt":
        return dart.prompt_attention(state["q"], state["k"], state["v"], state["starts"])
    if kind == "attend":
        return dart.block_attention(state["q"], state["keys"], state["values"], state["kscale"], state["vscale"],
                                    state["table"], state["lengths"], state["starts"], max_tokens=state["most"])
    if kind == "append":
        dart.append_blocks(state["k"], state["v"], state["slots"], state["keys"], state["values"], state["kscale"],
                           state["vscale"])
        return [state["keys"], state["values"], state["kscale"], state["vscale"]]
    tables = (state["table"], state["lengths"], state["free"], state["state"])
    dart.release_blocks(*tables, state["new"], block_size=state["bs"])
    slots, starts = dart.reserve_blocks(*tables, state["new"], state["total"], block_size=state["bs"])
    return [slots, starts, *tables]


# ---- the same in elementary torch operations ----

def _softmax_(s):
    """Softmax over the last axis, in place; rows without a finite logit are 0."""
    top = s.amax(-1, keepdim=True)
    s.sub_(top.clamp_min(torch.finfo(s.dtype).min)).exp_()
    total = s.sum(-1, keepdim=True)
    return s.div_(total.clamp_min(torch.finfo(s.dtype).tiny))


def _attention(q, k, v, seen):
    """q [R, H, n, D] over k, v [R, H, T, D]; query row i of request r sees the first seen[r, i] keys."""
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(1.0 / math.sqrt(q.shape[-1]))
    hidden = torch.arange(k.shape[2], device=q.device) >= seen[:, None, :, None]
    s.masked_fill_(hidden, -math.inf)
    return torch.matmul(_softmax_(s), v)


def _rows(starts, most):
    """Indexes [R, most] of each request's rows in the packed tensor, clamped, and which are real."""
    at = torch.arange(most, device=starts.device)
    return torch.minimum(starts[:-1, None] + at, starts[1:, None] - 1).clamp_min(0).long(), \
        at < (starts[1:] - starts[:-1])[:, None]


def _slots(table, before, starts, total, bs):
    """The slot of each of the packed new tokens; -1 behind the last."""
    t = torch.arange(total, device=table.device)
    row = torch.searchsorted(starts[1:].contiguous(), t, right=True).clamp_max(table.shape[0] - 1)
    at = before[row] + t - starts[row]
    block = table[row, (at // bs).clamp(0, table.shape[1] - 1)].long()
    return torch.where(t < starts[-1], block * bs + at % bs, -1)


def _run_plain(state):
    kind = state["kind"]
    if kind == "batch":
        q, k, v = (state[n].float() for n in "qkv")
        B, Hq, T, D = q.shape
        H = k.shape[1]
        seen = torch.arange(1, T + 1, device=q.device).repeat(Hq // H).expand(B, -1)
        return _attention(q.reshape(B, H, -1, D), k, v, seen).view(B, Hq, T, D).to(state["q"].dtype)
    if kind == "prompt":
        return _prompt_plain(state)
    if kind == "attend":
        return _attend_plain(state)
    if kind == "append":
        return _append_plain(state)
    return _tables_plain(state)


def _prompt_plain(state):
    starts, most = state["starts"], state["most"]
    rows, real = _rows(starts, most)
    R, H, D = rows.shape[0], state["k"].shape[1], state["k"].shape[2]
    q = state["q"].float()[rows].view(R, most, H, -1, D).permute(0, 2, 3, 1, 4).reshape(R, H, -1, D)
    k, v = (state[n].float()[rows].transpose(1, 2).contiguous() for n in "kv")
    groups = q.shape[2] // most
    seen = torch.arange(1, most + 1, device=q.device).repeat(groups).expand(R, -1)
    o = _attention(q, k, v, seen).view(R, H, groups, most, D).permute(0, 3, 1, 2, 4).reshape(R, most, -1, D)
    return o[real].to(state["q"].dtype)


def _attend_plain(state):
    starts, table, lengths, most = state["starts"], state["table"], state["lengths"], state["most"]
    rows, real = _rows(starts, most)
    N, H, bs, D = state["keys"].shape
    R = table.shape[0]
    blocks = table.clamp_min(0).long()

    def dense(codes, scale):
        x = codes.view(torch.uint8)[blocks].view(E4M3).float() * scale[blocks][..., None, None]
        return x.permute(0, 2, 1, 3, 4).reshape(R, H, -1, D)

    k, v = dense(state["keys"], state["kscale"]), dense(state["values"], state["vscale"])
    tail = torch.arange(k.shape[2], device=k.device) >= lengths[:, None]
    v.masked_fill_(tail[:, None, :, None], 0.0)
    q = state["q"].float()[rows].view(R, most, H, -1, D).permute(0, 2, 3, 1, 4).reshape(R, H, -1, D)
    groups = q.shape[2] // most
    first = lengths - (starts[1:] - starts[:-1]) + 1
    seen = (first[:, None] + torch.arange(most, device=q.device)).repeat(1, groups)
    o = _attention(q, k, v, seen).view(R, H, groups, most, D).permute(0, 3, 1, 2, 4).reshape(R, most, -1, D)
    return o[real].to(state["q"].dtype)


def _append_plain(state):
    slots = state["slots"]
    bs = state["keys"].shape[2]
    blocks, inverse = torch.unique(slots // bs, return_inverse=True)
    at = slots % bs
    # the block's first new row: rows before it hold tokens already
    first = torch.full((blocks.numel(),), bs, device=at.device).scatter_reduce_(0, inverse, at, "amin")
    _append_rows(state["keys"], state["kscale"], state["k"].float(), slots, blocks, inverse, first)
    _append_rows(state["values"], state["vscale"], state["v"].float(), slots, blocks, inverse, first)
    return [state["keys"], state["values"], state["kscale"], state["vscale"]]


def _append_rows(codes, scales, x, slots, blocks, inverse, first):
    bs = codes.shape[2]
    amax = torch.zeros(blocks.numel(), x.shape[1], device=x.device)
    amax.index_reduce_(0, inverse, x.abs().amax(-1), "amax")
    before = scales[blocks]
    scale = _block_scale(amax)
    scale = torch.where((first > 0)[:, None], torch.maximum(before, scale), scale)
    raw = codes.view(torch.uint8)
    held = raw[blocks]
    moved = (held.view(E4M3).float() * (before / scale)[..., None, None]).to(E4M3).view(torch.uint8)
    keep = (torch.arange(bs, device=x.device) < first[:, None])[:, None, :, None]
    raw[blocks] = torch.where(keep, moved, held)
    raw[slots // bs, :, slots % bs] = (x / scale[inverse][..., None]).to(E4M3).view(torch.uint8)
    scales[blocks] = scale


def _tables_plain(state):
    table, lengths, free, st, bs = (state[n] for n in ("table", "lengths", "free", "state", "bs"))
    column = torch.arange(table.shape[1], device=table.device)
    place = torch.arange(free.shape[0], device=table.device)

    def blocks_of(n):
        return (n + bs - 1) // bs

    # release: the last blocks of each row go onto the stack, the first row's on top
    drop = state["new"].clamp_min(0).minimum(lengths)
    keep = blocks_of(lengths - drop)
    gone = blocks_of(lengths) - keep
    before = gone.cumsum(0) - gone
    count = st[0] + gone.sum()
    given = (column >= keep[:, None]) & (column < (keep + gone)[:, None])
    at = torch.where(given, count - 1 - (before[:, None] + column - keep[:, None]), free.shape[0])
    stack = torch.cat((free, free.new_zeros(1))).scatter_(0, at.flatten(), table.flatten())
    free.copy_(stack[:-1])
    table.masked_fill_(given, -1)
    lengths.sub_(drop)
    # reserve: blocks from the top of the stack, in the rows' order
    new = state["new"]
    starts = torch.cat((new.new_zeros(1), new.cumsum(0).to(torch.int32)))
    old = blocks_of(lengths)
    need = blocks_of(lengths + new) - old
    before = need.cumsum(0) - need
    fits = (need.sum() <= count) & (starts[-1] <= state["total"]) & (new.min() >= 0) \
        & (blocks_of(lengths + new).max() <= table.shape[1])
    taken = (column >= old[:, None]) & (column < (old + need)[:, None]) & fits
    at = (count - 1 - (before[:, None] + column - old[:, None])).clamp(0, free.shape[0] - 1)
    table.copy_(torch.where(taken, free[at], table))
    used = torch.where(fits, need.sum(), 0)
    free.masked_fill_((place >= count - used) & (place < count), -1)
    slots = torch.where(fits, _slots(table, lengths, starts, state["total"], bs), -1)
    lengths.add_(torch.where(fits, new, 0))
    st[0] = count - used
    return [slots, starts, table, lengths, free, st]


# ---- from the definition, in 64 bits ----

def exact(case, seed):
    def attention(q, k, v, first):
        """q [n, D] of one head over k, v [T, D]: query i sees the keys up to ``first + i``, in pieces of rows."""
        out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
        for a in range(0, q.shape[0], 2048):
            b = min(q.shape[0], a + 2048)
            top = first + b
            logits = (q[a:b] @ k[:top].t().contiguous()) / math.sqrt(D)
            limit = torch.arange(a, b, device=q.device)[:, None] + first
            logits = torch.where(torch.arange(top, device=q.device)[None] <= limit, logits, -math.inf)
            out[a:b] = torch.softmax(logits, -1) @ v[:top]
        return out

    def decoded(codes, scale):
        return codes.view(E4M3).double() * scale.double()[..., None, None]

    lengths, new = _lengths(case)
    H, G, D, kind = case["H"], case["G"], case["D"], case["kind"]
    if kind == "tables":  # whole numbers
        return None
    state = prepare(case, seed)
    if kind == "prompt":
        q, k, v = (state[n].transpose(1, 2).reshape(-1, state[n].shape[1], D) if case["batch"] else state[n]
                   for n in "qkv")
        out = torch.empty(q.shape, dtype=torch.float64, device="cuda")
        at = _starts(lengths)
        for r in range(case["R"]):
            part = slice(at[r], at[r + 1])
            for h in range(H * G):
                out[part, h] = attention(q[part, h].double(), k[part, h // G].double(), v[part, h // G].double(), 0)
        if case["batch"]:
            out = out.view(case["R"], case["hi"], H * G, D).transpose(1, 2)
        return out
    bs = case["bs"]
    if kind == "attend":
        out = torch.empty(state["q"].shape, dtype=torch.float64, device="cuda")
        at = _starts(new)
        for r, n in enumerate(lengths):
            ids = state["table"][r, :-(-n // bs)].long()
            part = slice(at[r], at[r + 1])
            for h in range(H):
                k, v = (decoded(state[c].view(torch.uint8)[ids, h], state[s][ids, h]).view(-1, D)[:n]
                        for c, s in (("keys", "kscale"), ("values", "vscale")))
                for g in range(h * G, h * G + G):
                    out[part, g] = attention(state["q"][part, g].double(), k, v, n - new[r])
        return out
    # append: every request's new tokens lie in consecutive blocks of its own
    at, R = _starts(new), case["R"]
    if sum(-(-n // bs) for n in new) > 20000:
        return None
    first_slots = state["slots"].tolist()
    got = []
    for codes, scales, rows in ((state["keys"], state["kscale"], state["k"]),
                                (state["values"], state["vscale"], state["v"])):
        values, scales = codes.double(), scales.double()
        for r in range(R):
            first = lengths[r] - new[r]
            for j in range(first // bs, -(-lengths[r] // bs)):
                a, b = max(first, j * bs), min(lengths[r], (j + 1) * bs)
                x = rows[at[r] + a - first:at[r] + b - first].double().transpose(0, 1)  # [H, b - a, D]
                block = first_slots[at[r] + a - first] // bs
                top = x.abs().amax((1, 2))
                scale = torch.exp2(torch.ceil(torch.log2(top / E4M3_MAX)).clamp_min(MIN_EXPONENT))
                held = a - j * bs
                if held:
                    old = scales[block].clone()
                    scale = torch.maximum(old, scale)
                    moved = values[block, :, :held] * (old / scale)[:, None, None]
                    values[block, :, :held] = moved.to(E4M3).double()
                values[block, :, held:held + b - a] = (x / scale[:, None, None]).to(E4M3).double()
                scales[block] = scale
        got += [values, scales]
    return [got[0], got[2], got[1], got[3]]


# ---- what a pass cannot do without ----

def work(case):
    lengths, new = _lengths(case)
    H, G, D, kind, bs = case["H"], case["G"], case["D"], case["kind"], case["bs"]
    esize = DTYPES[case["dtype"]].itemsize
    heads = H * G
    pairs = sum(n * (2 * length - n + 1) // 2 for length, n in zip(lengths, new))
    tokens, blocks = sum(new), sum(-(-n // bs) for n in lengths)
    if kind == "prompt":
        return {"bytes": 2 * tokens * (heads + H) * D * esize, "flops": 4 * D * heads * pairs}
    if kind == "attend":
        cache = sum(lengths) * H * D * 2 + blocks * (8 * H + 4) + 8 * case["R"]
        return {"bytes": cache + 2 * tokens * heads * D * esize, "flops": 4 * D * heads * pairs}
    if kind == "append":
        touched = sum(-(-n // bs) - (n - m) // bs for n, m in zip(lengths, new))
        return {"bytes": tokens * (2 * H * D * (esize + 1) + 8) + touched * 16 * H, "flops": 4 * tokens * H * D}
    touched = sum(-(-n // bs) - -(-(n - m) // bs) for n, m in zip(lengths, new))
    return {"bytes": 8 * tokens + 24 * case["R"] + 16 * touched, "flops": 0}
