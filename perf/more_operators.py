"""The operators around a block cache's attention: what each computes, in plain torch, and the calls that a
program makes of the framework's own.

Four kinds of work:

* ``rotate``: RMS norm of each query and key head and the rotation by its position, in one pass; with
  ``grad`` the gradients of the inputs and of the norms' weights too;
* ``store``: the same for new tokens whose keys and values go into e4m3 blocks: the queries come back
  rotated, the keys and values as codes and scales;
* ``fork`` / ``compact``: rows of the block table that become copies of others (their blocks are shared until
  one of them writes), and blocks moved together, with the copies of their contents;
* ``logprob``: log probabilities of given tokens, the entropy and the most likely alternatives of rows of
  logits; with ``grad`` the gradient of the logits.
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
EPS = 1e-6


def _heads(name, kind, T, **over):
    """T tokens of H KV heads and H * G query heads of D channels, the first ``rotated`` of them turned."""
    case = dict(name=name, kind=kind, T=T, H=8, G=4, D=128, rotated=128, pairs="half", dtype="bf16", wtype="bf16",
                far=40960, batch=0, grad=False, shape=1)
    case.update(over)
    return case


def _store(name, R, lo, hi, new, **over):
    """R requests of lo to hi tokens, of which at most ``new`` are new."""
    case = dict(name=name, kind="store", R=R, lo=lo, hi=hi, new=new, H=8, G=4, D=128, rotated=128, pairs="half",
                dtype="bf16", bs=64, shape=1)
    case.update(over)
    return case


def _tables(name, kind, R, lo, hi, **over):
    """R rows of lo to hi tokens over blocks of bs tokens; ``group``: rows that descend from one."""
    case = dict(name=name, kind=kind, R=R, lo=lo, hi=hi, group=4, layers=2, H=8, D=128, bs=64, spare=0.1, shape=1)
    case.update(over)
    return case


def _logits(name, T, V, **over):
    case = dict(name=name, kind="logprob", T=T, V=V, dtype="bf16", top=0, grad=False, masked=False, shape=1)
    case.update(over)
    return case


def listed():
    return [
        # one new token of one interactive request: latency
        _heads("rotate_token", "rotate", 1),
        # a scheduler's packed prompts, far positions among them
        _heads("rotate_prompts", "rotate", 32768),
        # a training step's batch [B, H, T, D], gradients of the inputs and of fp32 norm weights
        _heads("rotate_train", "rotate", 8192, batch=4, wtype="fp32", grad=True),
        # a small model in fp16: few heads of 80, a part of them turned in neighbouring pairs, an odd number of tokens
        _heads("rotate_partial", "rotate", 3001, H=2, G=7, D=80, rotated=32, pairs="next", dtype="fp16", wtype="fp16",
               grad=True),
        # a decode step of a full batch, one token for each request
        _store("store_step", 64, 100, 8000, 1),
        # prompts written at once
        _store("store_prompts", 16, 1000, 4096, 4096),
        # a step of beam search: four beams of each of 16 requests, their last block differs
        _tables("fork_beams", "fork", 64, 500, 4000),
        # many samples of a few long prompts, small blocks: the prompts' blocks are shared
        _tables("fork_samples", "fork", 256, 9000, 16384, group=32, H=2, bs=16),
        # requests that ended leave holes all over the pool: blocks move together, twice
        _tables("compact_pool", "compact", 96, 64, 2500, group=1, layers=1, spare=0.4),
        # a decode step of a full batch: the sampled tokens and 20 alternatives of each
        _logits("logprob_step", 64, 151936, top=20),
        # prompts that are scored token by token, five alternatives
        _logits("logprob_prompts", 4096, 151936, top=5),
        # a policy's update: log probabilities and entropy with their gradient, rows of an odd size
        _logits("logprob_train", 4096, 32003, grad=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed ranges, sizes spread over their logarithm."""
    kind = rng.choice(["rotate", "rotate", "rotate", "store", "store", "fork", "fork", "compact", "logprob", "logprob",
                       "logprob"])
    shape = rng.randint(1, 1 << 20)
    H, G = rng.choice([1, 2, 4, 8]), rng.randint(1, 8)
    if kind == "rotate":
        D = rng.choice([64, 128, 128, 80, 96, 256, 72])
        grad = rng.random() < 0.5
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        most = (1 << (25 if grad else 27)) // (H * (G + 1) * D) // (2 if dtype == "fp32" else 1)
        T = _log_int(rng, 1, min(32768, most))
        batch = rng.choice([0, 0, 1, 2, 5])
        case = _heads("", kind, max(T, batch) // max(1, batch) * max(1, batch), H=H, G=G, D=D, batch=batch, grad=grad,
                      rotated=rng.choice([D, D, D // 2, D // 4 // 2 * 2]), pairs=rng.choice(["half", "half", "next"]),
                      dtype=dtype, wtype=rng.choice(["none", "fp32", dtype]), far=_log_int(rng, 64, 131072), shape=shape)
    elif kind == "store":
        D = rng.choice([64, 128, 128, 80, 256])
        hi = _log_int(rng, 16, 8192)
        R = _log_int(rng, 1, max(1, min(128, (1 << 25) // (H * (G + 2) * hi * D // 4))))
        case = _store("", R, max(1, int(hi * rng.choice([0.02, 0.3, 1.0]))), hi, rng.choice([1, 1, 3, hi, hi]), H=H, G=G,
                      D=D, rotated=rng.choice([D, D, D // 16 // 2 * 16]), pairs=rng.choice(["half", "half", "next"]),
                      dtype=rng.choice(["bf16", "bf16", "fp16"]), bs=rng.choice([16, 32, 64, 64, 128]), shape=shape)
    elif kind in ("fork", "compact"):
        D, layers, bs = rng.choice([64, 128, 256]), rng.randint(1, 4), rng.choice([16, 32, 64, 64, 128])
        hi = _log_int(rng, 16, 16384)
        most = (1 << (23 if kind == "fork" else 24)) // (layers * H * (hi + bs) * D // 16)
        R = _log_int(rng, 2, max(2, min(256, most)))
        case = _tables("", kind, R, max(1, int(hi * rng.choice([0.02, 0.3, 1.0]))), hi,
                       group=rng.choice([2, 3, 4, 16]) if kind == "fork" else 1, layers=layers, H=H, D=D, bs=bs,
                       spare=rng.choice([0.05, 0.4]), shape=shape)
    else:
        V = _log_int(rng, 500, 160000)
        grad = rng.random() < 0.4
        T = _log_int(rng, 1, min(8192, (1 << (27 if grad else 28)) // V))
        case = _logits("", T, V, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), grad=grad,
                       top=rng.choice([0, 1, 5, 20, 64]), masked=rng.random() < 0.3, shape=shape)
    del case["name"]
    return case


def _generator(seed, device="cuda"):
    return torch.Generator(device=device).manual_seed(seed)


def _starts(counts):
    return list(itertools.accumulate(counts, initial=0))


def _lengths(case):
    """Each request's length, its new tokens among them, and how many those are."""
    rng = random.Random(case["shape"])
    lengths = [rng.randint(case["lo"], case["hi"]) for _ in range(case["R"])]
    lengths[0] = case["hi"]
    return lengths, [min(n, case.get("new", 1)) for n in lengths]


def _rotations(rows, half):
    """cos and sin [rows, half] of each position's angles, in fp32 from angles in 64 bits."""
    speed = 1e6 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / max(1, half))
    angle = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * speed
    return angle.cos().float(), angle.sin().float()


def _weights(case, seed):
    """The norms' weights of queries and keys: around 1, as a model learns them."""
    if case.get("wtype") == "none":
        return None, None
    gen = _generator(seed + 5)
    kind = DTYPES[case.get("wtype", case["dtype"])]
    return [(1 + 0.3 * torch.randn(case["D"], generator=gen, device="cuda")).to(kind) for _ in range(2)]


def _projections(case, seed, tokens, kinds):
    """Queries, keys (and values) [tokens, heads, D] as views of one projection's output; heads of different sizes."""
    H, G, D = case["H"], case["G"], case["D"]
    heads = [H * G, H, H][:kinds]
    gen = _generator(seed)
    x = torch.randn(tokens, sum(heads), D, generator=gen, device="cuda")
    x *= torch.rand(1, sum(heads), 1, generator=gen, device="cuda") * 4 + 0.2
    return list(x.to(DTYPES[case["dtype"]]).split(heads, 1))


def prepare(case, seed):
    return {"rotate": _prepare_rotate, "store": _prepare_store, "fork": _prepare_fork, "compact": _prepare_compact,
            "logprob": _prepare_logprob}[case["kind"]](case, seed)


def _prepare_rotate(case, seed):
    T, B = case["T"], case["batch"]
    q, k = _projections(case, seed, T, 2)
    cos, sin = _rotations(case["far"], case["rotated"] // 2)
    positions = torch.randint(0, case["far"], (T,), generator=_generator(seed + 1), device="cuda", dtype=torch.int32)
    if B:  # [B, H, T, D] views of the projection's [B, T, H, D]
        q, k = (t.unflatten(0, (B, T // B)).transpose(1, 2) for t in (q, k))
        positions = positions.view(B, T // B)
    wq, wk = _weights(case, seed)
    state = {"kind": "rotate", "q": q, "k": k, "cos": cos, "sin": sin, "positions": positions, "wq": wq, "wk": wk,
             "next": case["pairs"] == "next", "grad": case["grad"]}
    if case["grad"]:
        state["leaves"] = [t.detach().requires_grad_() for t in (q, k, wq, wk) if t is not None]
        state["q"], state["k"] = state["leaves"][:2]
        if wq is not None:
            state["wq"], state["wk"] = state["leaves"][2:]
        gen = _generator(seed + 2)
        state["given"] = [torch.randn(t.shape, generator=gen, device="cuda").to(t.dtype) for t in (q, k)]
    return state


def _block_scale(amax):
    """The least power of two s with amax <= 448 s, as fp32 (the least of all for a block of zeros)."""
    mantissa, exponent = torch.frexp(amax)  # amax = mantissa * 2^exponent, mantissa in [1/2, 1); 448 = 7/8 * 2^9
    exponent = exponent - 9 + (mantissa > 0.875).to(exponent.dtype)
    exponent = torch.where(amax > 0, exponent, MIN_EXPONENT).clamp(MIN_EXPONENT, MAX_EXPONENT)
    return torch.ldexp(torch.ones(amax.shape, device=amax.device), exponent)


def _random_blocks(seed, layers, blocks, H, bs, D):
    """Codes [layers, blocks, H, bs, D] and scales [layers, blocks, H] of random rows."""
    x = torch.randn(layers, blocks, H, bs, D, generator=_generator(seed), device="cuda")
    scale = _block_scale(x.abs().amax((-1, -2)))
    return x.div_(scale[..., None, None]).to(E4M3), scale


def _pools(case, seed, layers, blocks):
    pools = [_random_blocks(seed + 3 + i, layers, blocks, case["H"], case["bs"], case["D"]) for i in range(2)]
    return {"kcode": pools[0][0], "vcode": pools[1][0], "kscale": pools[0][1], "vscale": pools[1][1]}


def _block_table(case, seed, lengths, total, columns=None):
    """A block table of requests of their own blocks in random order, the free stack and its state [free, 0, 0, 0]."""
    bs = case["bs"]
    held = torch.tensor([-(-n // bs) for n in lengths])
    order = torch.randperm(total, generator=_generator(seed + 2, "cpu"), dtype=torch.int32)
    most = max(int(held.max()), columns or 1)
    used = torch.arange(most) < held[:, None]
    at = int(used.sum())
    table = torch.full((len(lengths), most), -1, dtype=torch.int32)
    table[used] = order[:at]
    free = torch.full((total,), -1, dtype=torch.int32)
    free[:total - at] = order[at:]
    return {"table": table.cuda(), "lengths": torch.tensor(lengths, dtype=torch.int32).cuda(), "free": free.cuda(),
            "state": torch.tensor([total - at, 0, 0, 0], dtype=torch.int32).cuda(), "bs": bs}


def _prepare_store(case, seed):
    lengths, new = _lengths(case)
    bs, total = case["bs"], sum(new)
    blocks = sum(-(-n // bs) for n in lengths) + 3
    state = _block_table(case, seed, lengths, blocks)
    q, k, v = _projections(case, seed, total, 3)
    cos, sin = _rotations(case["hi"], case["rotated"] // 2)
    starts = torch.tensor(_starts(new), dtype=torch.int32).cuda()
    wq, wk = _weights(case, seed)
    pools = {n: t[0] for n, t in _pools(case, seed, 1, blocks).items()}
    slots, positions = _slots(state["table"], state["lengths"] - (starts[1:] - starts[:-1]), starts, total, bs)
    return {**state, **pools, "kind": "store", "q": q, "k": k, "v": v, "cos": cos, "sin": sin, "wq": wq, "wk": wk,
            "next": case["pairs"] == "next", "positions": positions.to(torch.int32), "slots": slots}


def _forks(case):
    """The first row of each row's group, the rows' lengths, their sources and how many tokens each gives back before."""
    R, group, rng = case["R"], case["group"], random.Random(case["shape"])
    roots = [r // group * group for r in range(R)]
    lengths = {r: rng.randint(case["lo"], case["hi"]) for r in range(0, R, group)}
    lengths = [lengths[r] for r in roots]
    if group <= 4:  # beams: each goes on from one of its group
        return roots, lengths, [root + rng.randrange(min(group, R - root)) for root in roots], [1] * R
    # samples: the roots stay, the others begin anew from them
    return roots, lengths, [-1 if r == root else root for r, root in enumerate(roots)], \
        [1 if r == root else n for r, (n, root) in enumerate(zip(lengths, roots))]


def _prepare_fork(case, seed):
    """Groups of rows that descend from their first: they share its full blocks, and each has a last one of its own."""
    R, bs = case["R"], case["bs"]
    roots, lengths, sources, drop = _forks(case)
    own_blocks = [-(-n // bs) if r == root else (1 if n % bs else 0) for r, (n, root) in enumerate(zip(lengths, roots))]
    blocks = int(sum(own_blocks) * (1 + case["spare"])) + R + 3
    full = torch.tensor([n // bs for n in lengths], dtype=torch.int64)
    width = max(-(-(n + 1) // bs) for n in lengths)
    order = torch.randperm(blocks, generator=_generator(seed + 2, "cpu"), dtype=torch.int32)
    first = torch.tensor(_starts(own_blocks), dtype=torch.int64)
    column = torch.arange(width)
    root = torch.tensor(roots)
    shared = order[(first[root][:, None] + column).clamp_max(blocks - 1)]
    last = order[(first[1:] - 1)]
    table = torch.where(column < full[:, None], shared, torch.tensor(-1, dtype=torch.int32))
    partial = torch.tensor([n % bs > 0 for n in lengths])
    table[partial, full[partial]] = last[partial]
    at = int(first[-1])
    free = torch.full((blocks,), -1, dtype=torch.int32)
    free[:blocks - at] = order[at:].sort(descending=True).values
    shares = torch.zeros(blocks, dtype=torch.int32)
    shares.index_add_(0, table[table >= 0].long(), torch.ones(int((table >= 0).sum()), dtype=torch.int32))
    shares -= (shares > 0).int()
    i32 = dict(dtype=torch.int32)
    return {"kind": "fork", **_pools(case, seed, case["layers"], blocks), "table": table.cuda(), "bs": bs,
            "lengths": torch.tensor(lengths, **i32).cuda(), "free": free.cuda(), "shares": shares.cuda(),
            "state": torch.tensor([blocks - at, 0, 0, 0], **i32).cuda(), "sources": torch.tensor(sources, **i32).cuda(),
            "drop": torch.tensor(drop, **i32).cuda(), "one": torch.ones(R, **i32).cuda()}


def _prepare_compact(case, seed):
    lengths, _ = _lengths(case)
    bs, R = case["bs"], case["R"]
    blocks = int(sum(-(-n // bs) for n in lengths) * (1 + case["spare"])) + 3
    state = _block_table(case, seed, lengths, blocks)
    half = torch.arange(R) % 2
    n = state["lengths"].cpu()
    parts = [torch.where(half == i, n, 0).to(torch.int32) for i in range(2)]
    return {**state, **_pools(case, seed, case["layers"], blocks), "kind": "compact",
            "parts": [t.cuda() for t in parts], "totals": [int(t.sum()) for t in parts],
            "shares": torch.zeros(blocks, dtype=torch.int32, device="cuda")}


def _prepare_logprob(case, seed):
    T, V = case["T"], case["V"]
    gen = _generator(seed)
    logits = torch.randn(T, V, generator=gen, device="cuda") * (torch.rand(T, 1, generator=gen, device="cuda") * 3 + 0.5)
    tokens = torch.randint(0, V, (T,), generator=gen, device="cuda")
    # half of the tokens are likely ones, as sampled
    likely = logits[:, :min(V, 2048)].argmax(-1)
    tokens = torch.where(torch.rand(T, generator=gen, device="cuda") < 0.5, likely, tokens)
    if case["masked"]:  # what a grammar allows: a tenth of the vocabulary, the given token among it
        allowed = torch.rand(V, generator=gen, device="cuda") < 0.1
        allowed[:min(V, 100)] = True
        keep = logits.gather(1, tokens[:, None])
        logits = logits.masked_fill_(~allowed, -math.inf).scatter_(1, tokens[:, None], keep)
    logits = logits.to(DTYPES[case["dtype"]])
    state = {"kind": "logprob", "logits": logits, "tokens": tokens, "top": case["top"], "grad": case["grad"]}
    if case["grad"]:
        state["logits"] = logits.requires_grad_()
        state["given"] = [torch.randn(T, generator=gen, device="cuda"), 0.01 * torch.randn(T, generator=gen, device="cuda")]
        if case["top"]:
            state["given"].append(0.1 * torch.randn(T, min(case["top"], V), generator=gen, device="cuda"))
    return state


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    import dartkv_amd as dart

    kind = state["kind"]
    if kind == "rotate":
        out = dart.rotate_heads(state["q"], state["k"], state["cos"], state["sin"], state["positions"],
                                q_weight=state["wq"], k_weight=state["wk"], eps=EPS, interleaved=state["next"])
        grads = torch.autograd.grad(out, state["leaves"], state["given"]) if state["grad"] else ()
        return [*(t.detach() for t in out), *grads]
    if kind == "store":
        q = dart.append_rotated_blocks(state["q"], state["k"], state["v"], state["cos"], state["sin"],
                                       state["positions"], state["slots"], *_pool_of(state), q_weight=state["wq"],
                                       k_weight=state["wk"], eps=EPS, interleaved=state["next"])
        return [q, *_pool_of(state)]
    if kind == "fork":
        tables, bs, shares, one = _tables_of(state), state["bs"], state["shares"], state["one"]
        dart.release_blocks(*tables, state["drop"], block_size=bs, shares=shares)
        dart.fork_blocks(*tables, shares, state["sources"], block_size=bs)
        slots, starts, copies = dart.reserve_blocks(*tables, one, one.numel(), block_size=bs, shares=shares)
        dart.copy_blocks(copies, *_pool_of(state))
        return [slots, starts, copies, *tables, shares, *_pool_of(state)]
    if kind == "compact":
        return [x for i in range(2) for x in _compact_own(state, i)] + [*_tables_of(state), *_pool_of(state)]
    out = dart.token_logprobs(state["logits"], state["tokens"], top=state["top"])
    if not state["grad"]:
        return [*out]
    into = (out.logprobs, out.entropy, out.top_logprobs)[:len(state["given"])]
    return [t.detach() for t in out] + [*torch.autograd.grad(into, state["logits"], state["given"])]


def _compact_own(state, i):
    """Half of the requests end, the others' blocks move together, and as many tokens come again."""
    import dartkv_amd as dart

    tables, bs, shares = _tables_of(state), state["bs"], state["shares"]
    dart.release_blocks(*tables, state["parts"][i], block_size=bs, shares=shares)
    copies = dart.compact_blocks(*tables, shares, block_size=bs)
    dart.copy_blocks(copies, *_pool_of(state))
    slots, _, _ = dart.reserve_blocks(*tables, state["parts"][i], state["totals"][i], block_size=bs, shares=shares)
    return copies, slots


def _pool_of(state):
    return [state[n] for n in ("kcode", "vcode", "kscale", "vscale")]


def _tables_of(state):
    return [state[n] for n in ("table", "lengths", "free", "state")]


# ---- the same in elementary torch operations ----

def _run_plain(state):
    return {"rotate": _rotate_plain, "store": _store_plain, "fork": _fork_plain, "compact": _compact_plain,
            "logprob": _logprob_plain}[state["kind"]](state)


def _turned(x, weight, cos, sin, neighbours, kind=torch.float32):
    """x [.., T, H, D] normed over D and turned by cos, sin [.., T, half], in ``kind``."""
    x, half = x.to(kind), cos.shape[-1]
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.to(kind)
    cos, sin = cos.to(kind)[..., None, :], sin.to(kind)[..., None, :]
    if neighbours:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, x[..., 2 * half:]), -1)


def _rotate_plain(state):
    at = state["positions"].long()
    cos, sin = state["cos"][at], state["sin"][at]

    def turn(x, weight):
        if x.dim() == 4:
            return _turned(x.transpose(1, 2), weight, cos, sin, state["next"]).transpose(1, 2).to(x.dtype)
        return _turned(x, weight, cos, sin, state["next"]).to(x.dtype)

    out = [turn(state["q"], state["wq"]), turn(state["k"], state["wk"])]
    grads = torch.autograd.grad(out, state["leaves"], state["given"]) if state["grad"] else ()
    return [*(t.detach() for t in out), *grads]


def _slots(table, before, starts, total, bs):
    """The slot of each of the packed new tokens (-1 behind the last), and its position."""
    t = torch.arange(total, device=table.device)
    row = torch.searchsorted(starts[1:].contiguous(), t, right=True).clamp_max(table.shape[0] - 1)
    at = before[row] + t - starts[row]
    block = table[row, (at // bs).clamp(0, table.shape[1] - 1)].long()
    return torch.where(t < starts[-1], block * bs + at % bs, -1), at


def _store_plain(state):
    slots, at = state["slots"], state["positions"].long()
    cos, sin = state["cos"][at], state["sin"][at]
    q = _turned(state["q"], state["wq"], cos, sin, state["next"]).to(state["q"].dtype)
    # (in 64 bits: a key next to the border of two codes, or of two scales, goes to its own side)
    k = _turned(state["k"], state["wk"], cos, sin, state["next"], torch.float64).to(state["k"].dtype)
    bs = state["bs"]
    blocks, inverse = torch.unique(slots // bs, return_inverse=True)
    # the block's first new row: rows before it hold tokens already
    first = torch.full((blocks.numel(),), bs, device=at.device).scatter_reduce_(0, inverse, slots % bs, "amin")
    _store_rows(state["kcode"], state["kscale"], k.float(), slots, blocks, inverse, first)
    _store_rows(state["vcode"], state["vscale"], state["v"].float(), slots, blocks, inverse, first)
    return [q, *_pool_of(state)]


def _store_rows(codes, scales, x, slots, blocks, inverse, first):
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


def _blocks_of(n, bs):
    return (n + bs - 1) // bs


def _columns(table):
    return torch.arange(table.shape[1], device=table.device)


def _holders(table):
    """How many rows hold each block, as a function of a block's number: counts with a place behind for -1."""
    return lambda blocks: torch.zeros(blocks + 1, dtype=torch.int64, device=table.device).index_add_(
        0, torch.where(table >= 0, table, blocks).flatten().long(),
        torch.ones(table.numel(), dtype=torch.int64, device=table.device))[:blocks]


def _settle_(state, before):
    """Shares from the rows, and blocks that no row holds any more onto the stack: the lowest one on top."""
    blocks = state["free"].shape[0]
    now = _holders(state["table"])(blocks)
    state["shares"].copy_((now - 1).clamp_min(0))
    gone = ((before > 0) & (now == 0)).nonzero().flatten().flip(0)
    # (entries behind the stack's top are -1, and gone are so many of them as there are blocks)
    place = torch.arange(blocks, device=now.device)
    count = state["state"][0]
    given = torch.cat((gone.to(torch.int32), gone.new_zeros(1, dtype=torch.int32)))
    at = (place - count).clamp(0, gone.numel())
    state["free"].copy_(torch.where((place >= count) & (place < count + gone.numel()), given[at], state["free"]))
    state["state"][0] += gone.numel()


def _release_plain(state, drop):
    table, lengths, bs = state["table"], state["lengths"], state["bs"]
    before = _holders(table)(state["free"].shape[0])
    lengths.sub_(torch.minimum(drop, lengths))
    table.masked_fill_(_columns(table) >= _blocks_of(lengths, bs)[:, None], -1)
    _settle_(state, before)


def _reserve_plain(state, new, total):
    """Slots, starts and the copies of blocks that are written while other rows hold them."""
    table, lengths, free, bs = state["table"], state["lengths"], state["free"], state["bs"]
    R, count = table.shape[0], state["state"][0].clone()
    rows = torch.arange(R, device=table.device)
    starts = torch.cat((new.new_zeros(1), new.cumsum(0).to(torch.int32)))
    # a writer copies its last block if other rows go on holding it, or writers behind it in the order do
    last = (lengths // bs).clamp_max(table.shape[1] - 1).long()
    block = table[rows, last]
    writes = (new > 0) & (lengths % bs > 0)
    same = writes[:, None] & writes[None] & (block[:, None] == block[None]) & (rows[None] < rows[:, None])
    copied = writes & (same.sum(1) < state["shares"][block.clamp_min(0).long()])
    old = _blocks_of(lengths, bs)
    need = _blocks_of(lengths + new, bs) - old + copied
    before = need.cumsum(0) - need
    # the copy first, then the new blocks, from the top of the stack in the rows' order
    column = _columns(table)
    start = torch.where(copied, last, old.long())
    taken = (column >= start[:, None]) & (column < (start + need)[:, None])
    at = (count - 1 - (before[:, None] + column - start[:, None])).clamp(0, free.shape[0] - 1)
    table.copy_(torch.where(taken, free[at], table))
    place = torch.arange(free.shape[0], device=table.device)
    used = need.sum()
    free.masked_fill_((place >= count - used) & (place < count), -1)
    state["shares"].index_add_(0, block.clamp_min(0).long(), -copied.to(torch.int32))
    order = copied.cumsum(0) - 1
    copies = torch.full((R + 1, 3), -1, dtype=torch.int32, device=table.device)
    copies[torch.where(copied, order, R)] = torch.stack((block, table[rows, last], lengths % bs), 1)
    slots, _ = _slots(table, lengths, starts, total, bs)
    lengths.add_(new)
    state["state"][0] = count - used
    return slots, starts, copies[:R]


def _copy_plain(state, copies):
    copies = copies[copies[:, 0] >= 0].long()
    source, target, tokens = copies.unbind(1)
    for codes, scales in ((state["kcode"], state["kscale"]), (state["vcode"], state["vscale"])):
        raw = codes.view(torch.uint8)
        keep = (torch.arange(raw.shape[-2], device=raw.device) < tokens[:, None])[:, None, :, None]
        raw[:, target] = torch.where(keep, raw[:, source], raw[:, target])
        scales[:, target] = scales[:, source]


def _fork_plain(state):
    _release_plain(state, state["drop"])
    table, lengths = state["table"], state["lengths"]
    before = _holders(table)(state["free"].shape[0])
    rows = torch.arange(table.shape[0], device=table.device)
    source = torch.where(state["sources"] >= 0, state["sources"], rows).long()
    table.copy_(table[source])
    lengths.copy_(lengths[source])
    _settle_(state, before)
    slots, starts, copies = _reserve_plain(state, state["one"], table.shape[0])
    _copy_plain(state, copies)
    return [slots, starts, copies, *_tables_of(state), state["shares"], *_pool_of(state)]


def _compact_plain(state):
    out = [*_compact_half(state, 0), *_compact_half(state, 1)]
    return [*out, *_tables_of(state), *_pool_of(state)]


def _compact_half(state, i):
    _release_plain(state, state["parts"][i])
    table, free, shares = state["table"], state["free"], state["shares"]
    blocks, count = free.shape[0], state["state"][0]
    place = torch.arange(blocks, device=table.device)
    used = torch.ones(blocks + 1, dtype=torch.bool, device=table.device)
    used[torch.where(place < count, free, blocks).long()] = False
    used = used[:blocks]
    movers = (used & (place >= blocks - count)).nonzero().flatten()
    holes = (~used & (place < blocks - count)).nonzero().flatten()
    to = torch.arange(blocks + 1, device=table.device)
    to[movers] = holes
    table.copy_(torch.where(table >= 0, to[table.clamp_min(0).long()].to(torch.int32), -1))
    shares[holes] = shares[movers]
    shares[movers] = 0
    free.copy_(torch.where(place < count, blocks - 1 - place, -1))
    copies = torch.full((blocks // 2, 3), -1, dtype=torch.int32, device=table.device)
    copies[:movers.numel()] = torch.stack((movers, holes, torch.full_like(movers, state["bs"])), 1).to(torch.int32)
    _copy_plain(state, copies)
    slots, _, _ = _reserve_plain(state, state["parts"][i], state["totals"][i])
    return copies, slots


def _top(x, k):
    """The k largest of each row in their order, the lower index first among equals: keys that are never equal."""
    bits = x.view(torch.int32).long()
    order = torch.where(bits < 0, bits ^ 0x7fffffff, bits)
    key = (order << 32) | (x.shape[-1] - 1 - torch.arange(x.shape[-1], device=x.device))
    return x.shape[-1] - 1 - (torch.topk(key, k).values & 0xffffffff)


def _logprob_plain(state):
    x = state["logits"].float()
    x = x + 0.0  # (-0 and 0 are equal)
    top = x.detach().amax(-1, keepdim=True)
    lse = (x - top).exp().sum(-1, keepdim=True).log() + top
    logp = x - lse
    got = logp.gather(1, state["tokens"][:, None]).squeeze(1)
    entropy = -(logp.exp() * logp.clamp_min(torch.finfo(torch.float32).min)).sum(-1)
    ids = _top(x.detach(), min(state["top"], x.shape[1]))
    out = [got, entropy, logp.gather(1, ids), ids]
    if not state["grad"]:
        return out
    return [t.detach() for t in out] + [*torch.autograd.grad(out[:len(state["given"])], state["logits"], state["given"])]


# ---- from the definition, in 64 bits ----

def exact(case, seed):
    if case["kind"] in ("fork", "compact"):  # whole numbers, and codes that are only moved
        return None
    if case["kind"] == "logprob":
        return _exact_logprob(case, seed)
    state = prepare(case, seed)
    half, D = case["rotated"] // 2, case["D"]

    # each channel's partner and the sign of its sine
    channel = torch.arange(D, device="cuda")
    if case["pairs"] == "next":
        partner, sign, angle = channel ^ 1, (channel & 1) * 2 - 1, channel // 2
    else:
        partner, sign, angle = (channel + half) % max(1, 2 * half), torch.where(channel < half, -1, 1), channel % max(1, half)
    still = channel >= 2 * half
    partner, angle = torch.where(still, channel, partner), torch.where(still, 0, angle)

    def forward(x, weight, at):
        """x [n, H, D] -> outputs; also the norm's factor, cos and sin of each channel, for the gradients."""
        x = x.double()
        factor = torch.ones_like(x[..., :1])
        if weight is not None:
            factor = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS)
        cos, sin = torch.ones(at.numel(), D, dtype=torch.float64, device="cuda"), torch.zeros(at.numel(), D,
                                                                                             dtype=torch.float64, device="cuda")
        if half:
            cos = torch.where(still, cos, state["cos"].double()[at][:, angle])
            sin = torch.where(still, sin, state["sin"].double()[at][:, angle] * sign)
        n = x * factor
        scaled = n if weight is None else n * weight.double()
        return scaled * cos[:, None] + scaled[..., partner] * sin[:, None], n, factor, cos, sin

    def backward(g, weight, n, factor, cos, sin):
        g = g.double()
        # the transposed rotation: a channel gets its partner's sine
        gs = g * cos[:, None] + (g * sin[:, None])[..., partner]
        gs = torch.where(still, g, gs)
        if weight is None:
            return gs, None
        gn = gs * weight.double()
        return factor * (gn - n * (gn * n).mean(-1, keepdim=True)), (gs * n).sum((0, 1))

    if case["kind"] == "store":
        lengths, new = _lengths(case)
        at = torch.tensor([p for n, m in zip(lengths, new) for p in range(n - m, n)], device="cuda")
        return [forward(state["q"].detach(), state["wq"], at)[0], None, None, None, None]
    B, T = case["batch"], case["T"]
    at = state["positions"].long().flatten()
    flat = lambda x: x.transpose(1, 2).flatten(0, 1) if B else x  # noqa: E731
    whole = lambda x: x.unflatten(0, (B, T // B)).transpose(1, 2) if B else x  # noqa: E731
    out, gx, gw = [], [], []
    for i, (x, w) in enumerate(((state["q"], state["wq"]), (state["k"], state["wk"]))):
        x, w = x.detach(), w if w is None else w.detach()
        y, *saved = forward(flat(x), w, at)
        out.append(whole(y))
        if case["grad"]:
            g, weight = backward(flat(state["given"][i]), w, *saved)
            gx.append(whole(g))
            gw += [] if weight is None else [weight]
    return [*out, *gx, *gw]


def _exact_logprob(case, seed):
    state = prepare(case, seed)
    logits, tokens, k = state["logits"].detach(), state["tokens"], min(case["top"], case["V"])
    pieces = []
    for rows in torch.arange(case["T"], device="cuda").split(max(1, (1 << 27) // case["V"])):
        x = logits[rows].double()
        p = torch.softmax(x, -1)
        norm = torch.logsumexp(x, -1, keepdim=True)
        entropy = torch.special.entr(p).sum(-1)
        best = torch.topk(x, k)
        got = x.gather(1, tokens[rows, None]) - norm
        piece = [got[:, 0], entropy, best.values - norm]
        if case["grad"]:
            given = [g.double()[rows] for g in state["given"]]
            # d logp(t)/dx = 1[t] - p; dH/dx = -p (log p + H)
            g = p * -given[0][:, None] - given[1][:, None] * (torch.xlogy(p, p) + p * entropy[:, None])
            g.scatter_add_(1, tokens[rows, None], given[0][:, None])
            if k:
                ids = _run_ids(state, rows, k)
                g -= p * given[2].sum(-1, keepdim=True)
                g.scatter_add_(1, ids, given[2])
            piece.append(g)
        pieces.append(piece)
    out = [torch.cat(t) for t in zip(*pieces)]
    return [*out[:3], None, *out[3:]]


def _run_ids(state, rows, k):
    """The first k of each row's stable order."""
    return torch.sort(state["logits"].detach()[rows].double(), dim=-1, descending=True, stable=True).indices[:, :k]


# ---- what a pass cannot do without ----

def work(case):
    kind = case["kind"]
    if kind == "logprob":
        n, size = case["T"] * case["V"], DTYPES[case["dtype"]].itemsize
        k = min(case["top"], case["V"])
        return {"bytes": n * size * (2 if case["grad"] else 1) + case["T"] * (16 + 12 * k),
                "flops": n * (9 if case["grad"] else 5)}
    H, D, bs = case["H"], case["D"], case.get("bs")
    if kind == "rotate":
        n, size = case["T"] * H * (case["G"] + 1) * D, DTYPES[case["dtype"]].itemsize
        angles = 4 * case["rotated"] * min(case["T"], case["far"])
        return {"bytes": n * size * (4 if case["grad"] else 2) + angles + 4 * case["T"], "flops": n * (20 if case["grad"] else 8)}
    if kind == "store":
        lengths, new = _lengths(case)
        tokens = sum(new)
        touched = sum(-(-n // bs) - (n - m) // bs for n, m in zip(lengths, new))
        size = DTYPES[case["dtype"]].itemsize
        row = D * H * (2 * case["G"] * size + 2 * size + 2)
        return {"bytes": tokens * (row + 4 * case["rotated"] + 12) + touched * 16 * H, "flops": tokens * D * H * 8 * (case["G"] + 2)}
    layers = case["layers"]
    if kind == "fork":
        _, lengths, sources, _ = _forks(case)
        sources = [r if s < 0 else s for r, s in enumerate(sources)]
        # all rows that go on from a source but one copy the tokens of its last block
        copied = sum((sources.count(s) - 1) * ((lengths[s] - 1) % bs) for s in set(sources))
        held = sum(-(-n // bs) for n in lengths)
        return {"bytes": copied * layers * H * D * 4 + 8 * held + 40 * case["R"], "flops": 0}
    lengths, _ = _lengths(case)
    held = sum(-(-n // bs) for n in lengths)
    return {"bytes": held // 2 * layers * H * bs * D * 4 + 24 * held + 8 * sum(lengths), "flops": 0}
