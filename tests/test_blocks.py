"""The block cache's operators: tables, appends, attention, and a serving loop of them together.

Tables and appends are compared exactly: with a plain model of the stack and the lengths, and with scales and codes
computed in 64 bits.  Attention is compared with attention in 64 bits over the decoded values.

Attention's tolerance.  Codes and their scales (powers of two) are exact.  Products are summed in fp32.  Few rows: the
weights keep 16 bits (two bf16 parts, 2^-17 relative), so only the result's rounding u |o| shows (u half a step of
the type): |error| <= u |o| + 2^-16 W, W = sum(p |v|) / sum(p), the second term also covering the fp32 sums.  Chunks:
bf16 weights are rounded once more, u W; fp16 chunks keep 16 bits too.
"""

from __future__ import annotations

import math
import random

import pytest
import torch

DEV = "cuda"
E4M3 = torch.float8_e4m3fn


# ---- tables ----

class TableModel:
    """The stack and the lengths in plain Python."""

    def __init__(self, requests, blocks, max_blocks, bs):
        self.table = [[-1] * max_blocks for _ in range(requests)]
        self.lengths, self.bs = [0] * requests, bs
        self.free = list(range(blocks - 1, -1, -1))
        self.blocks = blocks

    def _blocks(self, n):
        return -(-n // self.bs)

    def reserve(self, counts, total):
        slots, starts = [-1] * total, [0]
        at = 0
        for r, n in enumerate(counts):
            old, new = self._blocks(self.lengths[r]), self._blocks(self.lengths[r] + n)
            for j in range(old, new):
                self.table[r][j] = self.free.pop()
            for i in range(n):
                p = self.lengths[r] + i
                slots[at] = self.table[r][p // self.bs] * self.bs + p % self.bs
                at += 1
            self.lengths[r] += n
            starts.append(at)
        return slots, starts

    def release(self, counts):
        back = []
        for r, n in enumerate(counts):
            n = min(n, self.lengths[r])
            keep, old = self._blocks(self.lengths[r] - n), self._blocks(self.lengths[r])
            back += self.table[r][keep:old]
            self.table[r][keep:old] = [-1] * (old - keep)
            self.lengths[r] -= n
        self.free += back[::-1]


def _state(requests, blocks, max_blocks):
    i32 = dict(dtype=torch.int32, device=DEV)
    return (torch.full((requests, max_blocks), -1, **i32), torch.zeros(requests, **i32),
            torch.arange(blocks - 1, -1, -1, **i32), torch.tensor([blocks, 0, 0, 0], **i32))


def _same_state(state, model):
    table, lengths, free, st = (t.cpu().tolist() for t in state)
    assert table == model.table and lengths == model.lengths
    assert st == [len(model.free), 0, 0, 0]
    assert free == model.free + [-1] * (model.blocks - len(model.free))


@pytest.mark.gpu
@pytest.mark.parametrize("requests,bs,most", [(1, 16, 100), (5, 64, 300), (64, 16, 40), (65, 128, 1000), (257, 32, 90),
                                              (1000, 16, 30), (3, 256, 5000)])
def test_tables_against_a_plain_model(requests, bs, most):
    import dartkv_amd as dart
    rng = random.Random(requests)
    max_blocks = -(-6 * most // bs)
    blocks = requests * max_blocks
    state, model = _state(requests, blocks, max_blocks), TableModel(requests, blocks, max_blocks, bs)
    for step in range(6):
        counts = [rng.choice([0, 1, rng.randint(0, most)]) for _ in range(requests)]
        total = sum(counts) + rng.choice([0, 0, 37])
        tokens = torch.tensor(counts, dtype=rng.choice([torch.int32, torch.int64]), device=DEV)
        slots, starts = dart.reserve_blocks(*state, tokens, total, block_size=bs)
        want_slots, want_starts = model.reserve(counts, total)
        assert slots.cpu().tolist() == want_slots and starts.cpu().tolist() == want_starts
        _same_state(state, model)
        drop = [rng.choice([0, 0, 1, rng.randint(0, most), 10 ** 6]) for _ in range(requests)]
        dart.release_blocks(*state, torch.tensor(drop, device=DEV), block_size=bs)
        model.release(drop)
        _same_state(state, model)
    dart.release_blocks(*state, block_size=bs)
    model.release(model.lengths[:])
    _same_state(state, model)
    assert sorted(model.free) == list(range(blocks))


@pytest.mark.gpu
def test_release_undoes_a_reserve():
    import dartkv_amd as dart
    state = _state(7, 60, 20)
    dart.reserve_blocks(*state, torch.tensor([3, 0, 40, 16, 1, 17, 33], device=DEV), 110, block_size=16)
    before = [t.clone() for t in state]
    tokens = torch.tensor([14, 2, 0, 1, 15, 100, 0], device=DEV)
    dart.reserve_blocks(*state, tokens, 132, block_size=16)
    dart.release_blocks(*state, tokens, block_size=16)
    assert all(torch.equal(a, b) for a, b in zip(state, before))


@pytest.mark.gpu
@pytest.mark.parametrize("counts,total,bit", [
    ([100, 60, 1], 200, 1),  # 7 + 4 + 1 blocks, ten are free
    ([129, 1, 1], 200, 2),  # more than eight blocks
    ([1, -1, 1], 200, 4), ([10, 10, 10], 29, 8), ([2 ** 31 - 1] * 3, 200, 8)])
def test_reserve_that_cannot_be_met_changes_nothing(counts, total, bit):
    import dartkv_amd as dart
    state = _state(3, 10, 8)
    before = [t.clone() for t in state]
    slots, starts = dart.reserve_blocks(*state, torch.tensor(counts, dtype=torch.int64, device=DEV), total, block_size=16)
    assert bool((slots == -1).all()) and bool((starts == 0).all())
    assert all(torch.equal(a, b) for a, b in zip(state[:3], before[:3]))
    got = state[3].cpu().tolist()
    assert got[0] == 10 and got[1] & bit and got[2] == 0
    slots, starts = dart.reserve_blocks(*state, torch.tensor([100, 48, 0], device=DEV), 148, block_size=16)
    assert starts.cpu().tolist() == [0, 100, 148, 148] and int(state[3][0]) == 0  # all ten blocks


# ---- appends ----

def _scale64(amax):
    e = torch.ceil(torch.log2(amax.double() / 448)).clamp(-120, 121)
    return torch.where(amax > 0, torch.exp2(e), torch.tensor(2.0 ** -120, dtype=torch.float64))


def _append64(x, slots, codes, scales, bs):
    """codes [N, H, bs, D] (values of codes, 64 bits) and scales [N, H] after x [T, H, D] went to ``slots``."""
    t = 0
    while t < len(slots):
        if slots[t] < 0:
            t += 1
            continue
        block, stop = slots[t] // bs, t
        while stop < len(slots) and slots[stop] >= 0 and slots[stop] // bs == block:
            stop += 1
        held = slots[t] % bs
        new = x[t:stop].double().transpose(0, 1)
        finite = torch.where(torch.isfinite(new), new, 0.0)
        scale = _scale64(finite.abs().amax((1, 2)))
        if held:
            old = scales[block].clone()
            scale = torch.maximum(old, scale)
            codes[block, :, :held] = (codes[block, :, :held] * (old / scale)[:, None, None]).float().to(E4M3).double()
        codes[block, :, held:held + stop - t] = (new / scale[:, None, None]).float().to(E4M3).double()
        scales[block] = scale
        t = stop


def _pool(N, H, bs, D):
    return [torch.zeros(N, H, bs, D, dtype=torch.uint8, device=DEV).view(E4M3) for _ in range(2)] + \
        [torch.ones(N, H, device=DEV) for _ in range(2)]


def _same_values(got, want):
    got, want = got.float().double().cpu(), want
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("H,D,bs,sizes", [
    (1, 16, 16, [1, 1, 14, 1, 33]), (8, 128, 64, [5, 59, 1, 200, 1, 1]), (2, 80, 32, [100, 1, 27, 1]),
    (3, 256, 128, [129, 1, 1]), (5, 48, 256, [300, 1])])
def test_appends_against_64_bits(dtype, H, D, bs, sizes):
    """Requests that grow by the given sizes, values whose range grows from append to append."""
    import dartkv_amd as dart
    gen = torch.Generator().manual_seed(D)
    R, most = 3, -(-sum(sizes) // bs)
    state = _state(R, R * most + 1, most)
    pool = _pool(R * most + 1, H, bs, D)
    want = [t.float().double().cpu() for t in pool]
    for i, n in enumerate(sizes):
        counts = [n, max(0, n - 1), n if i % 2 else 0]
        T = sum(counts) + 2
        slots, _ = dart.reserve_blocks(*state, torch.tensor(counts, device=DEV), T, block_size=bs)
        spread = 10.0 ** torch.empty(T, H, 1).uniform_(-3, 0.3 * i, generator=gen)
        k, v = ((torch.randn(T, H, D, generator=gen) * spread).to(dtype) for _ in range(2))
        k[:1] = 0
        dart.append_blocks(k.to(DEV), v.to(DEV), slots, *pool)
        for x, c, s in ((k, want[0], want[2]), (v, want[1], want[3])):
            _append64(x, slots.cpu().tolist(), c, s, bs)
        for got, w in zip(pool, want):
            _same_values(got, w)


@pytest.mark.gpu
@pytest.mark.parametrize("value", [448.0, 449.0, 2.0 ** -130, 3.0e38, 65504.0, 0.0, 7 / 8 * 2.0 ** -100])
def test_scales_at_their_borders(value):
    import dartkv_amd as dart
    pool = _pool(2, 1, 16, 16)
    x = torch.full((1, 1, 16), value, device=DEV)
    dart.append_blocks(x, -x, torch.tensor([16], device=DEV), *pool)
    scale = float(pool[2][1, 0])
    assert scale == float(_scale64(torch.tensor(float(x.flatten()[0]))))
    assert torch.equal(pool[0][1, 0, 0].float().cpu().double(), (x.flatten().cpu().double() / scale).float().to(E4M3).double())
    assert torch.equal(pool[1][1, 0, 0].float(), -pool[0][1, 0, 0].float())
    assert float(pool[2][0, 0]) == 1.0 and bool((pool[0][0].float() == 0).all())


@pytest.mark.gpu
def test_values_are_within_half_a_step():
    """A value of a block is off by half a step of e4m3 at its size, or by half the block's smallest step."""
    import dartkv_amd as dart
    pool = _pool(1, 4, 128, 64)
    x = torch.randn(128, 4, 64, generator=torch.Generator().manual_seed(1)).to(DEV)
    dart.append_blocks(x, x * 100, torch.arange(128, device=DEV), *pool)
    for y, codes, scale in ((x, pool[0], pool[2]), (x * 100, pool[1], pool[3])):
        got = codes[0].float() * scale[0][:, None, None]
        err = (got - y.transpose(0, 1)).abs()
        half = torch.maximum(y.transpose(0, 1).abs() * 2 ** -4, scale[0][:, None, None] * 2 ** -10)
        assert bool((err <= half).all())


@pytest.mark.gpu
def test_nonfinite_values_become_nan_and_are_reported():
    import dartkv_amd as dart
    pool = _pool(1, 2, 16, 32)
    x = torch.randn(3, 2, 32, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(DEV)
    flag = torch.zeros(1, dtype=torch.int32, device=DEV)
    dart.append_blocks(x, x, torch.arange(3, device=DEV), *pool, nonfinite=flag)
    assert int(flag) == 0
    clean = pool[0].float().clone()
    x[1, 0, 5], x[1, 0, 6], x[2, 0, 7] = float("inf"), float("-inf"), float("nan")
    dart.append_blocks(x, x, torch.arange(3, device=DEV), *pool, nonfinite=flag)
    assert int(flag) == 1
    bad = torch.isnan(pool[0].float())
    assert int(bad.sum()) == 3 and bool(bad[0, 0, 1, 5] & bad[0, 0, 1, 6] & bad[0, 0, 2, 7])
    assert torch.equal(pool[0].float()[0, 1], clean[0, 1])


@pytest.mark.gpu
def test_append_strides_and_slots_outside():
    import dartkv_amd as dart
    pool, want = _pool(2, 2, 16, 32), _pool(2, 2, 16, 32)
    x = torch.randn(6, 7, 40, generator=torch.Generator().manual_seed(1)).to(torch.float16).to(DEV)
    slots = torch.tensor([3, 4, 5, -1, 32, 1 << 40], device=DEV)
    for k, v in ((x[:, :2, :32], x[:, 2:4, 8:]), (x[:, 4:6, 3:35], x[:, 5:7, 1:33])):
        dart.append_blocks(k, v, slots, *pool)
        dart.append_blocks(k[:3].contiguous(), v[:3].contiguous(), slots[:3], *want)
        assert all(torch.equal(a.float(), b.float()) for a, b in zip(pool, want))
    assert bool((pool[0][1].float() == 0).all()) and float(pool[2][1, 0]) == 1.0
    assert bool((pool[0][0, :, 3:6].float() != 0).any()) and bool((pool[0][0, :, 6:].float() == 0).all())


# ---- attention ----

def _cache(lengths, H, D, bs, seed, spare=3):
    """Random codes and scales, a table of blocks in random order; bytes behind the lengths are NaN."""
    gen = torch.Generator().manual_seed(seed)
    most = max(1, max(-(-n // bs) for n in lengths))
    N = sum(-(-n // bs) for n in lengths) + spare
    order = torch.randperm(N, generator=gen)
    table = torch.full((len(lengths), most + 1), -1, dtype=torch.int32)
    codes = [torch.full((N, H, bs, D), 0x7f, dtype=torch.uint8) for _ in range(2)]
    scales = [torch.exp2(torch.randint(-8, 3, (N, H), generator=gen).float()) for _ in range(2)]
    at = 0
    for r, n in enumerate(lengths):
        for j in range(-(-n // bs)):
            b = int(order[at])
            table[r, j] = b
            at += 1
            rows = min(bs, n - j * bs)
            for i in range(2):
                x = torch.randn(H, rows, D, generator=gen) * (1.0 / scales[i][b])[:, None, None]
                codes[i][b, :, :rows] = x.clamp(-448, 448).to(E4M3).view(torch.uint8)
    lens = torch.tensor(lengths, dtype=torch.int32)
    return [t.to(DEV) for t in (codes[0].view(E4M3), codes[1].view(E4M3), *scales, table, lens)]


def _dense(cache, r):
    """Request r's keys and values [n, H, D] in 64 bits."""
    kc, vc, ks, vs, table, lens = (t.cpu() for t in cache)
    n, bs = int(lens[r]), kc.shape[2]
    ids = table[r, :-(-n // bs)].long()
    return [(c.view(torch.uint8)[ids].view(E4M3).float().double() * s[ids].double()[..., None, None])
            .transpose(1, 2).reshape(-1, c.shape[1], c.shape[3])[:n] for c, s in ((kc, ks), (vc, vs))]


def _check_attention(got, q, cache, new, dtype, chunk=False, scale=None):
    u = torch.finfo(dtype).eps / 2
    at = 0
    for r, n in enumerate(new):
        if n == 0:
            continue
        k, v = _dense(cache, r)
        H, D = k.shape[1], k.shape[2]
        x = q[at:at + n].double().cpu().view(n, H, -1, D).permute(1, 2, 0, 3)
        s = x @ k.permute(1, 2, 0)[:, None] * (scale or 1 / math.sqrt(D))
        seen = k.shape[0] - n + 1 + torch.arange(n)
        hidden = torch.arange(k.shape[0]) >= seen[:, None]
        p = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
        o, w = (torch.matmul(p, t.permute(1, 0, 2)[:, None]).permute(2, 0, 1, 3).reshape(n, -1, D) for t in (v, v.abs()))
        err = (got[at:at + n].double().cpu() - o).abs()
        bound = 1.01 * u * o.abs() + (1.01 * u if chunk and dtype == torch.bfloat16 else 2 ** -16) * w
        # (a value of 0 alone has an error and a bound of 0)
        assert bool((err <= bound).all()), f"request {r}: error is {float((err / bound).max()):.3f} of its bound"
        at += n


def _query(tokens, heads, D, dtype, seed):
    return torch.randn(tokens, heads, D, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def _starts(new):
    at = [0]
    for n in new:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device=DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [16, 64, 80, 128, 144, 256])
@pytest.mark.parametrize("bs", [16, 64, 256])
def test_single_tokens(dtype, D, bs):
    import dartkv_amd as dart
    lengths = [1, 2, 15, 16, 17, 31, 33, 100, 257, 700]
    cache = _cache(lengths, 2, D, bs, D + bs)
    q = _query(len(lengths), 6, D, dtype, 1)
    _check_attention(dart.block_attention(q, *cache), q, cache, [1] * len(lengths), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("G", [1, 2, 5, 8, 16, 17, 40])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_head_groups(G, D):
    import dartkv_amd as dart
    lengths = [70, 1, 300]
    cache = _cache(lengths, 3, D, 32, G)
    q = _query(3, 3 * G, D, torch.float16, G)
    _check_attention(dart.block_attention(q, *cache, scale=0.3), q, cache, [1] * 3, torch.float16, scale=0.3)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,lengths", [(1, [9000]), (8, [5000, 3, 2500]), (2, [33] * 70 + [4000] + [1] * 9), (3, [640] * 5)])
def test_requests_that_several_waves_share(dtype, H, lengths):
    import dartkv_amd as dart
    cache = _cache(lengths, H, 128, 64, H)
    q = _query(len(lengths), 4 * H, 128, dtype, 2)
    got = dart.block_attention(q, *cache)
    _check_attention(got, q, cache, [1] * len(lengths), dtype)
    assert torch.equal(got, dart.block_attention(q, *cache))  # the same bits every time


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,G,new,limit", [
    (64, 4, [4, 1, 0, 16, 3], 16), (64, 8, [8, 5], 8), (128, 4, [8, 1, 0, 7], 8), (128, 2, [1, 2, 3, 4, 5], 5),
    (256, 4, [4, 2, 0, 3], 4), (256, 1, [16, 9], 16), (256, 7, [5, 9, 1, 2, 9], 9), (128, 8, [8, 7, 1], 8),
    (80, 21, [3, 1, 2], 3)])
def test_a_few_tokens(dtype, D, G, new, limit):
    """Drafted tokens: each sees its own key and those before it."""
    import dartkv_amd as dart
    lengths = [max(1, n) + extra for n, extra in zip(new, (0, 1000, 5, 40, 211))]
    cache = _cache(lengths, 2, D, 16, D)
    q = _query(sum(new), 2 * G, D, dtype, 3)
    got = dart.block_attention(q, *cache, _starts(new), max_tokens=limit)
    _check_attention(got, q, cache, new, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,G,new", [(64, 4, 4), (128, 4, 8), (128, 1, 3), (256, 4, 4), (64, 4, 150), (128, 8, 60)])
def test_nan_codes_reach_only_the_rows_that_see_them(dtype, D, G, new):
    import dartkv_amd as dart
    lengths, H = [new, 100 + new, 37 + new], 2
    cache = _cache(lengths, H, D, 32, D)
    q = _query(3 * new, H * G, D, dtype, 9)
    starts = _starts([new] * 3)
    want = dart.block_attention(q, *cache, starts, max_tokens=new)
    raw = [c.view(torch.uint8) for c in cache[:2]]
    bad = [new // 2, new - 1, 0]  # of each request's new tokens, the one with a NaN value (channel 3 + r of head 1)
    for r, i in enumerate(bad):
        t = lengths[r] - new + i
        raw[1][int(cache[4][r, t // 32]), 1, t % 32, 3 + r] = 0xff
    t = lengths[1] - 2
    raw[0][int(cache[4][1, t // 32]), 0, t % 32, 5] = 0x7f  # and a NaN key of head 0
    got = dart.block_attention(q, *cache, starts, max_tokens=new).view(3, new, H, G, D)
    want = want.view(3, new, H, G, D)
    hit = torch.zeros(got.shape, dtype=torch.bool)
    for r, i in enumerate(bad):
        hit[r, i:, 1, :, 3 + r] = True
    hit[1, new - 2:, 0] = True
    assert torch.equal(torch.isnan(got).cpu(), hit)
    assert torch.equal(got[~hit.to(DEV)], want[~hit.to(DEV)])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 80, 128, 256])
@pytest.mark.parametrize("bs", [16, 64])
def test_chunks_beside_single_tokens(dtype, D, bs):
    import dartkv_amd as dart
    new = [100, 1, 0, 33, 1, 64, 200]
    lengths = [100, 77, 50, 533, 1, 64, 1001]
    cache = _cache(lengths, 2, D, bs, D)
    q = _query(sum(new), 6, D, dtype, 4)
    got = dart.block_attention(q, *cache, _starts(new))
    _check_attention(got, q, cache, new, dtype, chunk=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("H,G,new,lengths", [(1, 8, [20], [6000]), (2, 40, [1, 1], [3000, 9]),
                                             (1, 3, [50, 1, 12], [2500, 4000, 333])])
def test_few_rows_over_long_contexts(dtype, D, H, G, new, lengths):
    """Chunks too few to fill the GPU: their keys come in parts that are joined."""
    import dartkv_amd as dart
    cache = _cache(lengths, H, D, 64, D)
    q = _query(sum(new), H * G, D, dtype, 8)
    starts = None if max(new) == 1 else _starts(new)
    _check_attention(dart.block_attention(q, *cache, starts), q, cache, new, dtype, chunk=True)


@pytest.mark.gpu
def test_lengths_that_leave_rows_empty():
    """More new tokens than the length: the first see nothing and are 0; a request without keys is 0."""
    import dartkv_amd as dart
    cache = _cache([3, 40, 0, 5], 1, 64, 16, 1)
    for new in ([5, 1, 2, 0], [50, 2, 1, 30]):
        q = _query(sum(new), 2, 64, torch.bfloat16, 5)
        got = dart.block_attention(q, *cache, _starts(new)).float().cpu()
        assert bool(torch.isfinite(got).all())
        assert bool((got[:new[0] - 3] == 0).all()) and bool((got[new[0] - 3:new[0]].abs().sum((1, 2)) > 0).all())
        at = new[0] + new[1]
        assert bool((got[at:at + new[2]] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("many", [False, True])
def test_bad_table_entries_are_nan_for_who_sees_them(many):
    import dartkv_amd as dart
    cache = _cache([100, 100, 60], 2, 64, 16, 6)
    new = [40, 40, 40] if many else [1, 1, 1]
    q = _query(sum(new), 4, 64, torch.bfloat16, 6)
    want = dart.block_attention(q, *cache, _starts(new))
    cache[4][1, 3], cache[4][2, 3] = 10 ** 9, -5
    got = dart.block_attention(q, *cache, _starts(new)).float()
    a, b = new[0], new[0] + new[1]
    assert torch.equal(got[:a], want[:a].float()) and bool(torch.isnan(got[a:b]).all())
    first = 48 - (60 - new[2])  # the first row of request 2 that sees key 48
    assert bool(torch.isnan(got[b + max(0, first):]).all())
    if first > 0:
        assert torch.equal(got[b:b + first], want[b:b + first].float())


@pytest.mark.gpu
def test_out_strides_and_padding_rows():
    import dartkv_amd as dart
    new, lengths = [2, 1, 3], [40, 300, 3]
    cache = _cache(lengths, 2, 64, 32, 7)
    q = _query(9, 4, 64, torch.bfloat16, 7)
    got = dart.block_attention(q, *cache, _starts(new), max_tokens=3)
    assert bool((got[6:] == 0).all())
    _check_attention(got[:6], q[:6], cache, new, torch.bfloat16)
    out = torch.full((9, 4, 72), 5.0, dtype=torch.bfloat16, device=DEV)
    wide = torch.zeros(9, 6, 80, dtype=torch.bfloat16, device=DEV)
    wide[:, 1:5, 8:72] = q
    for many in (3, None):
        out.fill_(5.0)
        dart.block_attention(wide[:, 1:5, 8:72], *cache, _starts(new), max_tokens=many, out=out[..., :64])
        _check_attention(out[:6, :, :64], q[:6], cache, new, torch.bfloat16)
        assert bool((out[6:] == 5).all()) and bool((out[..., 64:] == 5).all())


# ---- together ----

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_serving_loop(dtype):
    """Prompts, decode steps, drafts that are rejected, a request that ends and another that takes its row, and a
    captured step replayed while the requests grow: attention over the cache against 64 bits over what was appended."""
    import dartkv_amd as dart
    H, G, D, bs, R, L = 2, 4, 64, 16, 4, 2
    cache = dart.BlockKVCache(R, 64, H, D, layers=L, block_size=bs, max_blocks=40)
    gen = torch.Generator().manual_seed(1)

    def step(counts, total=None, release=None):
        if release is not None:
            cache.release(torch.tensor(release, device=DEV))
        total = sum(counts) if total is None else total
        plan = cache.reserve(torch.tensor(counts, device=DEV), total)
        for layer in range(L):
            k, v = (torch.randn(total, H, D, generator=gen).to(dtype).to(DEV) for _ in range(2))
            q = torch.randn(total, H * G, D, generator=gen).to(dtype).to(DEV)
            cache.append(layer, k, v, plan)
            got = cache.attention(layer, q, plan)
            view = [cache.key_codes[layer], cache.value_codes[layer], cache.key_scale[layer], cache.value_scale[layer],
                    cache.table, cache.lengths]
            _check_attention(got[:sum(counts)], q[:sum(counts)], view, counts, dtype, chunk=True)
            assert bool((got[sum(counts):] == 0).all())
        cache.check()

    step([50, 1, 0, 33])
    step([1, 1, 0, 1])
    step([4, 4, 0, 4])
    step([1, 1, 0, 1], release=[3, 4, 0, 1])
    step([1, 0, 90, 1], total=100, release=[0, 10 ** 6, 0, 0])
    step([1, 20, 1, 1])

    # a decode step as a graph: the same tensors, growing requests
    ones = torch.ones(R, dtype=torch.int32, device=DEV)
    k, v = (torch.randn(R, H, D, generator=gen).to(dtype).to(DEV) for _ in range(2))
    q = torch.randn(R, H * G, D, generator=gen).to(dtype).to(DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan = cache.reserve(ones, R, max_tokens=1)
        cache.append(0, k, v, plan)
        cache.append(1, v, k, plan)
        got = cache.attention(0, q, plan), cache.attention(1, q, plan)
    for i in range(20):
        k.copy_(torch.randn(R, H, D, generator=gen))
        before = cache.lengths.clone()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(cache.lengths, before + 1)
        for layer in range(L):
            view = [cache.key_codes[layer], cache.value_codes[layer], cache.key_scale[layer], cache.value_scale[layer],
                    cache.table, cache.lengths]
            _check_attention(got[layer], q, view, [1] * R, dtype)
            eager = dart.block_attention(q, *view)
            assert torch.equal(eager, got[layer])
    cache.check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_prompts_then_tokens(dtype):
    """Packed prompts attended in 16 bits while they go into the blocks, then tokens over the blocks: the prompts'
    results against 64 bits over what was given, the tokens' over the codes, which are within half a step of it."""
    import dartkv_amd as dart
    from tests.test_prompt_attention import _packed_check
    H, G, D, lengths = 2, 3, 128, [70, 1, 333]
    total = sum(lengths)
    cache = dart.BlockKVCache(3, 16, H, D, block_size=64)
    k, v = (torch.randn(total, H, D, generator=torch.Generator().manual_seed(i)).to(dtype).to(DEV) for i in (1, 2))
    q = _query(total, H * G, D, dtype, 3)
    plan = cache.reserve(torch.tensor(lengths, device=DEV), total)
    cache.append(0, k, v, plan)
    _packed_check(dart.prompt_attention(q, k, v, plan.starts), q, k, v, lengths, lengths, True, D ** -0.5, dtype)
    view = [cache.key_codes[0], cache.value_codes[0], cache.key_scale[0], cache.value_scale[0], cache.table, cache.lengths]
    at = 0
    for r, n in enumerate(lengths):
        for x, got in zip((k, v), _dense(view, r)):
            x = x[at:at + n].double().cpu()
            assert bool(((got - x).abs() <= torch.maximum(x.abs() * 2 ** -4, torch.tensor(2.0 ** -16))).all())
        at += n
    _check_attention(cache.attention(0, q, plan), q, view, lengths, dtype, chunk=True)
    for step in range(3):
        plan = cache.reserve(torch.ones(3, dtype=torch.int32, device=DEV), 3, max_tokens=1)
        k, v = (torch.randn(3, H, D, generator=torch.Generator().manual_seed(9 + step + i)).to(dtype).to(DEV) for i in (0, 50))
        q = _query(3, H * G, D, dtype, step)
        cache.append(0, k, v, plan)
        _check_attention(cache.attention(0, q, plan), q, view, [1] * 3, dtype)
    cache.check()


@pytest.mark.gpu
def test_check_reports_and_clears():
    import dartkv_amd as dart
    cache = dart.BlockKVCache(2, 4, 1, 64, block_size=16)
    plan = cache.reserve(torch.tensor([100, 1], device=DEV), 101)
    x = torch.ones(101, 1, 64, dtype=torch.bfloat16, device=DEV)
    cache.append(0, x, x, plan)
    assert bool((cache.attention(0, x, plan) == 0).all())
    with pytest.raises(RuntimeError, match="too few free blocks"):
        cache.check()
    cache.check()
    plan = cache.reserve(torch.tensor([1, 0], device=DEV), 1)
    cache.append(0, x[:1] * float("inf"), x[:1], plan)
    with pytest.raises(ValueError, match="finite"):
        cache.check()
    cache.check()


@pytest.mark.gpu
def test_plans_of_earlier_steps_are_refused():
    import dartkv_amd as dart
    cache = dart.BlockKVCache(2, 8, 1, 64, block_size=16)
    x = torch.ones(2, 1, 64, dtype=torch.bfloat16, device=DEV)
    one = torch.ones(2, dtype=torch.int32, device=DEV)
    plan = cache.reserve(one, 2)
    cache.append(0, x, x, plan)
    cache.append(0, x, x, plan)  # (again: the same tokens)
    assert torch.equal(cache.attention(0, x, plan), x)
    cache.release(one)
    for call in (lambda: cache.append(0, x, x, plan), lambda: cache.attention(0, x, plan)):
        with pytest.raises(ValueError, match="earlier"):
            call()
    new = cache.reserve(one, 2)
    with pytest.raises(ValueError, match="earlier"):
        cache.append(0, x, x, plan)
    cache.append(0, x, x, new)


@pytest.mark.gpu
def test_two_graphs_and_two_streams_at_once():
    """Two captured calls that need workspaces, replayed on two streams at once, and eager calls beside them."""
    import dartkv_amd as dart
    calls = []
    for seed in (1, 2):
        cache = _cache([4000, 3000], 2, 128, 64, seed)
        q = _query(2, 8, 128, torch.bfloat16, seed)
        calls.append((q, cache, dart.block_attention(q, *cache)))
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    for q, cache, _ in calls:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(dart.block_attention(q, *cache))
        graphs.append(graph)
    for _ in range(10):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        eager = [dart.block_attention(q, *cache) for q, cache, _ in calls]
        torch.cuda.synchronize()
        for got, again, (_, _, want) in zip(outs, eager, calls):
            assert torch.equal(got, want) and torch.equal(again, want)


# ---- refusals ----

@pytest.mark.gpu
def test_python_refusals():
    import dartkv_amd as dart
    state = _state(2, 8, 4)
    tokens = torch.ones(2, dtype=torch.int32, device=DEV)
    bad = [
        (ValueError, lambda: dart.reserve_blocks(*state, tokens, 2, block_size=48)),
        (ValueError, lambda: dart.reserve_blocks(*state, tokens, -1, block_size=16)),
        (ValueError, lambda: dart.reserve_blocks(*state, tokens[:1], 2, block_size=16)),
        (TypeError, lambda: dart.reserve_blocks(*state, tokens.float(), 2, block_size=16)),
        (ValueError, lambda: dart.reserve_blocks(*state, tokens.cpu(), 2, block_size=16)),
        (TypeError, lambda: dart.reserve_blocks(state[0].long(), *state[1:], tokens, 2, block_size=16)),
        (ValueError, lambda: dart.release_blocks(state[0][:1], *state[1:], tokens, block_size=16)),
    ]
    pool = _pool(4, 2, 16, 32)
    x = torch.zeros(3, 2, 32, dtype=torch.bfloat16, device=DEV)
    slots = torch.arange(3, device=DEV)
    bad += [
        (TypeError, lambda: dart.append_blocks(x.double(), x.double(), slots, *pool)),
        (TypeError, lambda: dart.append_blocks(x, x.half(), slots, *pool)),
        (ValueError, lambda: dart.append_blocks(x[:, :1], x[:, :1], slots, *pool)),
        (TypeError, lambda: dart.append_blocks(x, x, slots.int(), *pool)),
        (TypeError, lambda: dart.append_blocks(x, x, slots[:2], *pool)),
        (TypeError, lambda: dart.append_blocks(x, x, slots, pool[0].view(torch.uint8), *pool[1:])),
        (TypeError, lambda: dart.append_blocks(x, x, slots, pool[0].transpose(0, 1).contiguous().transpose(0, 1), *pool[1:])),
        (ValueError, lambda: dart.append_blocks(x, x, slots, *pool[:2], pool[2][:2], pool[3])),
        (TypeError, lambda: dart.append_blocks(x, x, slots, *pool, nonfinite=torch.zeros(1, device=DEV))),
    ]
    table, lens = torch.zeros(3, 2, dtype=torch.int32, device=DEV), torch.ones(3, dtype=torch.int32, device=DEV)
    grad = torch.zeros(3, 2, 32, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    bad += [
        (TypeError, lambda: dart.block_attention(x.float(), *pool, table, lens)),
        (ValueError, lambda: dart.block_attention(x[..., :16], *pool, table, lens)),
        (ValueError, lambda: dart.block_attention(x[:, :1], *pool, table, lens)),
        (ValueError, lambda: dart.block_attention(x[:2], *pool, table, lens)),
        (TypeError, lambda: dart.block_attention(x, *pool, table.long(), lens)),
        (TypeError, lambda: dart.block_attention(x, *pool, table, lens[:2])),
        (ValueError, lambda: dart.block_attention(x, *pool, table, lens, torch.zeros(3, dtype=torch.int32, device=DEV))),
        (ValueError, lambda: dart.block_attention(x, *pool, table, lens, max_tokens=0)),
        (ValueError, lambda: dart.block_attention(x, *pool, table, lens, scale=-1.0)),
        (RuntimeError, lambda: dart.block_attention(grad, *pool, table, lens)),
        (ValueError, lambda: dart.block_attention(x, *pool, table, lens, out=x[:2])),
        (ValueError, lambda: dart.BlockKVCache(2, 4, 1, 60)),
        (ValueError, lambda: dart.BlockKVCache(2, 4, 1, 64, block_size=8)),
        (ValueError, lambda: dart.BlockKVCache(0, 4, 1, 64)),
    ]
    for i, (error, call) in enumerate(bad):
        with pytest.raises(error):
            call()
            print("accepted:", i)


def test_cpu_tensors_are_refused():
    import dartkv_amd as dart
    x = torch.zeros(1, 1, 64, dtype=torch.bfloat16)
    i = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        dart.reserve_blocks(i.view(1, 4), i[:1], i, i, i[:1], 1, block_size=16)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        dart.block_attention(x, x, x, x, x, i.view(1, 4), i[:1])
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        dart.append_blocks(x, x, i, x, x, x, x)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        dart.BlockKVCache(1, 1, 1, 64, device="cpu")


@pytest.mark.parametrize("entry,field,value,code,text", [
    ("reserve", "requests", 0, 1, "requests"), ("reserve", "requests", 8191, 1, "requests"),
    ("reserve", "block_size", 24, 1, "block_size"), ("reserve", "max_blocks", 0, 1, "counts"),
    ("reserve", "blocks", 0, 1, "counts"), ("reserve", "tokens", None, 1, "NULL"), ("reserve", "slots", None, 1, "NULL"),
    ("reserve", "total", -1, 1, "total"), ("reserve", "state", None, 1, "NULL"), ("release", "table", None, 1, "NULL"),
    ("release", "block_size", 512, 1, "block_size"),
    ("append", "dtype", 3, 3, "bf16"), ("append", "D", 24, 1, "16"), ("append", "D", 528, 1, "512"),
    ("append", "block_size", 0, 1, "block_size"), ("append", "keys", 8, 1, "aligned"), ("append", "k_st", 4, 1, "aligned"),
    ("append", "slots", None, 1, "NULL"), ("append", "blocks", 0, 1, "counts"),
    ("attention", "dtype", 0, 3, "bf16 or fp16"), ("attention", "Hq", 3, 1, "divisible"), ("attention", "D", 272, 1, "256"),
    ("attention", "requests", 0, 1, "counts"), ("attention", "starts", None, 1, "one token"),
    ("attention", "scale", -1.0, 1, "scale"), ("attention", "table", None, 1, "NULL"),
    ("attention", "query", 8, 1, "aligned"), ("attention", "o_st", 2, 1, "aligned"),
    ("attention", "workspace_bytes", 100, 1, "workspace"), ("attention", "max_tokens", 0, 1, "counts"),
])
def test_c_entries_refuse_on_the_host(entry, field, value, code, text):
    """Bad arguments return an error before anything is launched (no GPU)."""
    from dartkv_amd import _lib
    lib = _lib.load()
    if entry in ("reserve", "release"):
        a = _lib.BlockTablesArgs(table=256, lengths=256, free=256, state=256, tokens=256, slots=256, starts=256, total=4,
                                 requests=2, max_blocks=4, blocks=8, block_size=16)
        call = lib.dkv_reserve_blocks if entry == "reserve" else lib.dkv_release_blocks
    elif entry == "append":
        a = _lib.AppendBlocksArgs(keys=256, values=256, dtype=2, k_st=64, k_sh=32, v_st=64, v_sh=32, slots=256, tokens=4,
                                  H=2, D=32, blocks=2, block_size=16, key_codes=256, value_codes=256, key_scale=256,
                                  value_scale=256)
        call = lib.dkv_append_blocks
    else:
        a = _lib.BlockAttentionArgs(query=256, out=256, dtype=2, q_st=128, q_sh=32, o_st=128, o_sh=32, tokens=4, starts=256,
                                    table=256, lengths=256, requests=2, max_blocks=4, blocks=8, block_size=16, key_codes=256,
                                    value_codes=256, key_scale=256, value_scale=256, Hq=4, Hkv=2, D=32, scale=1.0,
                                    max_tokens=4, workspace=256, workspace_bytes=1 << 40)
        call = lib.dkv_block_attention
    setattr(a, field, value)
    assert call(a, None) == code
    assert text in lib.dkv_last_error().decode()
    assert call(None, None) == 1


def test_ctypes_structs_match_the_header(tmp_path):
    """Field offsets and sizes of the ctypes mirrors equal the C compiler's."""
    import ctypes
    import os
    import subprocess
    from dartkv_amd import _lib
    structs = {"dkv_prompt_attention_args": _lib.PromptAttentionArgs, "dkv_block_tables_args": _lib.BlockTablesArgs,
               "dkv_append_blocks_args": _lib.AppendBlocksArgs, "dkv_block_attention_args": _lib.BlockAttentionArgs}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "dartkv.h"', "int main(void) {"]
    for cname, cls in structs.items():
        lines.append(f'  printf("{cname} size %zu\\n", sizeof({cname}));')
        lines += [f'  printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));' for f, _ in cls._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["  return 0;", "}"]) + "\n")
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    subprocess.run(["gcc", "-I", include, str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout
    got = {tuple(line.split()[:2]): int(line.split()[2]) for line in out.splitlines()}
    for cname, cls in structs.items():
        assert got[(cname, "size")] == ctypes.sizeof(cls), cname
        for field, _ in cls._fields_:
            assert got[(cname, field)] == getattr(cls, field).offset, (cname, field)
