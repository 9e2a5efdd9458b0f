"""Forked, released, reserved and compacted requests of a block cache, and the copies of their blocks.

Everything is compared exactly with a plain model of the tables in which the holders of a block are counted anew from the
rows, and the blocks' contents with what each request should hold: tokens are written as tags, so a block that is written
for one request while another holds it, or a copy that is missed, shows in the other's tokens.
"""

from __future__ import annotations

import random

import pytest
import torch

DEV = "cuda"


@pytest.fixture(autouse=True)
def _seed():
    torch.manual_seed(0)


E4M3 = torch.float8_e4m3fn


class Model:
    """Rows of blocks, the stack, and each request's tokens."""

    def __init__(self, requests, blocks, max_blocks, bs):
        self.rows, self.lengths, self.tokens = [[] for _ in range(requests)], [0] * requests, [[] for _ in range(requests)]
        self.free, self.blocks, self.max_blocks, self.bs = list(range(blocks - 1, -1, -1)), blocks, max_blocks, bs

    def holders(self):
        count = [0] * self.blocks
        for row in self.rows:
            for b in row:
                count[b] += 1
        return count

    def _settle(self, before):
        now = self.holders()
        gone = [b for b in range(self.blocks) if before[b] and not now[b]]
        self.free += gone[::-1]

    def release(self, counts):
        before = self.holders()
        for r, n in enumerate(counts):
            self.lengths[r] -= min(max(n, 0), self.lengths[r])
            del self.rows[r][-(-self.lengths[r] // self.bs):]
            del self.tokens[r][self.lengths[r]:]
        self._settle(before)

    def fork(self, sources, counts=None):
        before = self.holders()
        old = [(list(row), n, list(t)) for row, n, t in zip(self.rows, self.lengths, self.tokens)]
        for r, s in enumerate(sources):
            if s == -1 or not 0 <= s < len(old) or (counts is not None and counts[r] < 0):
                continue
            row, n, tokens = old[s]
            n = n if counts is None else min(n, counts[r])
            self.rows[r], self.lengths[r], self.tokens[r] = row[:-(-n // self.bs)], n, tokens[:n]
        self._settle(before)

    def needs(self, counts):
        return sum(-(-(n + c) // self.bs) - -(-n // self.bs) for n, c in zip(self.lengths, counts)) + len(self.copied(counts))

    def copied(self, counts):
        shares = [max(0, n - 1) for n in self.holders()]
        out, seen = [], {}
        for r, c in enumerate(counts):
            n = self.lengths[r]
            if c > 0 and n % self.bs:
                b = self.rows[r][-1]
                if seen.get(b, 0) < shares[b]:
                    out.append(r)
                seen[b] = seen.get(b, 0) + 1
        return out

    def reserve(self, counts, total, tags):
        copied = self.copied(counts)
        slots, starts, positions, copies = [], [0], [], []
        for r, c in enumerate(counts):
            n = self.lengths[r]
            if r in copied:
                copies.append([self.rows[r][-1], self.free[-1], n % self.bs])
                self.rows[r][-1] = self.free.pop()
            for _ in range(-(-(n + c) // self.bs) - len(self.rows[r])):
                self.rows[r].append(self.free.pop())
            for i in range(n, n + c):
                slots.append(self.rows[r][i // self.bs] * self.bs + i % self.bs)
                positions.append(i)
            self.lengths[r] += c
            self.tokens[r] += tags[starts[-1]:starts[-1] + c]
            starts.append(len(slots))
        pad = [-1] * (total - len(slots))
        return slots + pad, starts, positions + pad, copies + [[-1] * 3] * (len(counts) - len(copies))

    def compact(self):
        used = self.blocks - len(self.free)
        holes = sorted(b for b in self.free if b < used)
        movers = sorted(set(range(used, self.blocks)) - set(self.free))
        to = dict(zip(movers, holes))
        self.rows = [[to.get(b, b) for b in row] for row in self.rows]
        self.free = list(range(self.blocks - 1, used - 1, -1))
        copies = [[m, h, self.bs] for m, h in zip(movers, holes)]
        return copies + [[-1] * 3] * (self.blocks // 2 - len(copies))


class Device:
    """The same on the GPU: the tables' state and two layers of tagged blocks."""

    def __init__(self, requests, blocks, max_blocks, bs, H=2, D=16, layers=2):
        i32 = dict(dtype=torch.int32, device=DEV)
        self.tables = (torch.full((requests, max_blocks), -1, **i32), torch.zeros(requests, **i32),
                       torch.arange(blocks - 1, -1, -1, **i32), torch.tensor([blocks, 0, 0, 0], **i32))
        self.shares, self.bs = torch.zeros(blocks, **i32), bs
        self.pools = [torch.zeros(layers, blocks, H, bs, D, dtype=torch.uint8, device=DEV).view(E4M3) for _ in range(2)] + \
            [torch.zeros(layers, blocks, H, device=DEV) for _ in range(2)]

    def write(self, slots, tags):
        """A token's tag into its rows, another in each layer, head and pool; scales count the writes of a block."""
        at = torch.tensor([s for s in slots if s >= 0], device=DEV)
        tag = torch.tensor(tags, dtype=torch.uint8, device=DEV)
        for i, pool in enumerate(self.pools[:2]):
            raw = pool.view(torch.uint8)
            for layer in range(raw.shape[0]):
                for h in range(raw.shape[2]):
                    raw[layer, at // self.bs, h, at % self.bs] = ((tag + 17 * i + 5 * layer + h) % 120)[:, None].expand(-1, raw.shape[-1])

    def tokens(self, row, length):
        at = torch.arange(length, device=DEV)
        block = self.tables[0][row, at // self.bs].long()
        out = None
        for i, pool in enumerate(self.pools[:2]):
            raw = pool.view(torch.uint8)
            for layer in range(raw.shape[0]):
                for h in range(raw.shape[2]):
                    x = raw[layer, block, h, at % self.bs].int()
                    assert bool((x == x[:, :1]).all())
                    x = (x[:, 0] - 17 * i - 5 * layer - h) % 120
                    assert out is None or torch.equal(x, out)
                    out = x
        return out.tolist()


def same(dev, model, contents=True):
    table, lengths, free, state = (t.cpu().tolist() for t in dev.tables)
    assert lengths == model.lengths
    assert table == [row + [-1] * (len(table[0]) - len(row)) for row in model.rows]
    assert free == model.free + [-1] * (model.blocks - len(model.free)) and state[0] == len(model.free) and state[2] == 0
    assert dev.shares.cpu().tolist() == [max(0, n - 1) for n in model.holders()]
    if contents:
        for r, n in enumerate(lengths):
            assert dev.tokens(r, n) == model.tokens[r], r


@pytest.mark.gpu
@pytest.mark.parametrize("requests,bs,most,steps,contents", [(1, 16, 60, 8, True), (6, 16, 50, 25, True), (16, 32, 90, 14, True),
                                                             (65, 16, 40, 8, True), (300, 16, 30, 8, False),
                                                             (1100, 64, 300, 5, False), (5, 256, 2000, 8, False)])
def test_lifecycles_against_a_plain_model(requests, bs, most, steps, contents):
    import dartkv_amd as dart
    rng = random.Random(requests + bs)
    max_blocks = -(-4 * most // bs)
    blocks = max(8, requests * max_blocks // 2)
    dev, model = Device(requests, blocks, max_blocks, bs, layers=2 if contents else 1), Model(requests, blocks, max_blocks, bs)
    kinds = ["reserve", "fork", "step", "prefix", "release", "step", "fork", "compact", "step"]
    for step in range(steps):
        kind = kinds[step % len(kinds)]
        if kind in ("reserve", "step"):
            counts = [rng.choice([0, 1, 1]) if kind == "step" else rng.randint(0, most) for _ in range(requests)]
            counts = [min(c, max_blocks * bs - n) for c, n in zip(counts, model.lengths)]
            if model.needs(counts) > len(model.free):
                counts = [0] * (requests - 1) + [1 if model.lengths[-1] < max_blocks * bs and model.free else 0]
            total = sum(counts) + rng.choice([0, 5])
            tags = [rng.randrange(120) for _ in range(sum(counts))]
            positions = torch.empty(total, dtype=torch.int32, device=DEV)
            slots, starts, copies = dart.reserve_blocks(*dev.tables, torch.tensor(counts, device=DEV), total, block_size=bs,
                                                        shares=dev.shares, positions=positions)
            dart.copy_blocks(copies, *dev.pools)
            want = model.reserve(counts, total, tags)
            assert [slots.tolist(), starts.tolist(), positions.tolist(), copies.tolist()] == list(want)
            if contents:
                dev.write(want[0], tags)
        elif kind in ("fork", "prefix"):
            sources = [rng.choice([-1, r, rng.randrange(requests), rng.randrange(max(1, requests // 4))]) for r in range(requests)]
            counts = None if kind == "fork" else [rng.choice([0, 10 ** 6, rng.randint(0, 2 * most)]) for _ in range(requests)]
            dart.fork_blocks(*dev.tables, dev.shares, torch.tensor(sources, device=DEV, dtype=rng.choice([torch.int32, torch.int64])),
                             None if counts is None else torch.tensor(counts, device=DEV), block_size=bs)
            model.fork(sources, counts)
        elif kind == "release":
            counts = [rng.choice([0, 1, rng.randint(0, most), 10 ** 6]) for _ in range(requests)]
            dart.release_blocks(*dev.tables, torch.tensor(counts, device=DEV), block_size=bs, shares=dev.shares)
            model.release(counts)
        else:
            copies = dart.compact_blocks(*dev.tables, dev.shares, block_size=bs)
            dart.copy_blocks(copies, *dev.pools)
            assert copies.tolist() == model.compact()
        same(dev, model, contents)
    dart.release_blocks(*dev.tables, block_size=bs, shares=dev.shares)
    model.release(model.lengths[:])
    same(dev, model)
    assert sorted(model.free) == list(range(blocks)) and not dev.shares.any()


@pytest.mark.gpu
def test_a_pool_of_several_segments():
    """More blocks than one workgroup looks through for what became free."""
    import dartkv_amd as dart
    requests, bs, blocks, max_blocks = 9, 16, 70000, 9000
    dev, model = Device(requests, blocks, max_blocks, bs, H=1, layers=1), Model(requests, blocks, max_blocks, bs)
    counts = [8000 * 16 - 3, 5, 100000, 7, 0, 1000, 16 * 8999, 33, 64]
    dart.reserve_blocks(*dev.tables, torch.tensor(counts, device=DEV), sum(counts), block_size=bs, shares=dev.shares)
    model.reserve(counts, sum(counts), [0] * sum(counts))
    sources = [-1, 0, -1, 0, 6, 2, 6, 7, 6]
    dart.fork_blocks(*dev.tables, dev.shares, torch.tensor(sources, device=DEV), block_size=bs)
    model.fork(sources)
    same(dev, model, False)
    drop = [10 ** 6, 3, 50000, 10 ** 6, 77, 0, 10 ** 6, 1, 16 * 8000]
    dart.release_blocks(*dev.tables, torch.tensor(drop, device=DEV), block_size=bs, shares=dev.shares)
    model.release(drop)
    same(dev, model, False)
    copies = dart.compact_blocks(*dev.tables, dev.shares, block_size=bs)
    assert copies.tolist() == model.compact()
    same(dev, model, False)


@pytest.mark.gpu
def test_many_requests_write_into_blocks_of_others():
    """8,190 requests of 40 prompts, all in the middle of a block: all but one of each prompt's copy it."""
    import dartkv_amd as dart
    requests, bs, blocks = 8190, 16, 8400
    dev, model = Device(requests, blocks, 3, bs, H=1, layers=1), Model(requests, blocks, 3, bs)
    counts = [20 if r < 40 else 0 for r in range(requests)]
    dart.reserve_blocks(*dev.tables, torch.tensor(counts, device=DEV), 800, block_size=bs, shares=dev.shares)
    tags = [r % 120 for r in range(40) for _ in range(20)]
    dev.write(model.reserve(counts, 800, tags)[0], tags)
    sources = [-1 if r < 40 else r * 7 % 40 for r in range(requests)]
    dart.fork_blocks(*dev.tables, dev.shares, torch.tensor(sources, device=DEV), block_size=bs)
    model.fork(sources)
    same(dev, model, False)
    ones = [1] * requests
    tags = [r * 11 % 120 for r in range(requests)]
    slots, _, copies = dart.reserve_blocks(*dev.tables, torch.tensor(ones, device=DEV), requests, block_size=bs, shares=dev.shares)
    dart.copy_blocks(copies, *dev.pools)
    want = model.reserve(ones, requests, tags)
    assert slots.tolist() == want[0] and copies.tolist() == want[3]
    dev.write(want[0], tags)
    same(dev, model, False)
    for r in (0, 39, 40, 4000, 8189):
        assert dev.tokens(r, 21) == model.tokens[r]


@pytest.mark.gpu
def test_a_reserve_that_cannot_be_met_copies_nothing():
    import dartkv_amd as dart
    dev = Device(3, 4, 4, 16)
    dart.reserve_blocks(*dev.tables, torch.tensor([40, 0, 0], device=DEV), 40, block_size=16, shares=dev.shares)
    dart.fork_blocks(*dev.tables, dev.shares, torch.tensor([-1, 0, 0], device=DEV), block_size=16)
    before = [t.clone() for t in (*dev.tables, dev.shares)]
    assert before[4].tolist().count(2) == 3
    ones = torch.ones(3, dtype=torch.int32, device=DEV)
    # (two copies, and one block is free)
    slots, starts, copies = dart.reserve_blocks(*dev.tables, ones, 3, block_size=16, shares=dev.shares)
    assert slots.tolist() == [-1] * 3 and not starts.any() and bool((copies == -1).all())
    assert int(dev.tables[3][1]) == 1
    dev.tables[3][1] = 0
    assert all(torch.equal(a, b) for a, b in zip((*dev.tables, dev.shares), before))
    for _ in range(2):  # one writer: it copies; then it writes into its own
        tokens = torch.tensor([0, 1, 0], device=DEV)
        copies = dart.reserve_blocks(*dev.tables, tokens, 1, block_size=16, shares=dev.shares)[2]
        assert copies.tolist() == ([[int(before[0][0, 2]), int(dev.tables[0][1, 2]), 8]] if _ == 0 else [[-1] * 3]) + [[-1] * 3] * 2
    assert int(dev.tables[3][0]) == 0 and dev.shares.tolist().count(1) == 1


@pytest.mark.gpu
def test_forks_that_are_no_forks():
    """Sources outside the requests and negative counts leave their row, the others are served; check() says so."""
    import dartkv_amd as dart
    cache = dart.BlockKVCache(4, 16, 1, 16, block_size=16, sharing=True)
    cache.reserve(torch.tensor([30, 5, 17, 0], device=DEV), 52)
    before = [t.clone() for t in (cache.table, cache.lengths)]
    cache.fork(torch.tensor([4, -2, 0, -1], device=DEV))
    assert cache.lengths.tolist() == [30, 5, 30, 0] and torch.equal(cache.table[2, :2], before[0][0, :2])
    assert torch.equal(cache.table[:2], before[0][:2])
    with pytest.raises(RuntimeError, match="source that is not a request"):
        cache.check()
    cache.check()
    cache.fork(torch.tensor([-1, 0, 0, 0], device=DEV), torch.tensor([9, -1, 0, 16], device=DEV))
    assert cache.lengths.tolist() == [30, 5, 0, 16]
    with pytest.raises(RuntimeError, match="negative token count"):
        cache.check()
    cache.fork(torch.tensor([3, -2 ** 40, 2 ** 40, 0], device=DEV))
    assert cache.lengths.tolist() == [16, 5, 0, 30]
    with pytest.raises(RuntimeError, match="source that is not a request"):
        cache.check()


@pytest.mark.gpu
def test_a_stack_that_is_none_is_left_alone():
    import dartkv_amd as dart
    for state, at, value in ((-3, None, None), (99, None, None), (None, 0, 40), (None, 1, -7), (None, 0, 8)):
        dev = Device(2, 12, 6, 16)
        dart.reserve_blocks(*dev.tables, torch.tensor([40, 50], device=DEV), 90, block_size=16, shares=dev.shares)
        dart.release_blocks(*dev.tables, torch.tensor([40, 0], device=DEV), block_size=16, shares=dev.shares)
        if state is not None:
            dev.tables[3][0] = state
        if at is not None:  # (8 is then twice on the stack)
            dev.tables[2][at] = value
        before = [t.clone() for t in (*dev.tables, dev.shares)]
        copies = dart.compact_blocks(*dev.tables, dev.shares, block_size=16)
        assert bool((copies == -1).all()) and int(dev.tables[3][1]) == 1
        dev.tables[3][1] = 0
        assert all(torch.equal(a, b) for a, b in zip((*dev.tables, dev.shares), before))


@pytest.mark.gpu
@pytest.mark.parametrize("H,D,bs,layers", [(1, 16, 16, 1), (8, 128, 64, 3), (3, 80, 32, 2), (2, 256, 256, 1), (5, 48, 128, 4)])
def test_copies(H, D, bs, layers):
    """Whole and partial blocks, entries to be skipped, many entries, pools with a stride between layers."""
    import dartkv_amd as dart
    gen = torch.Generator(DEV).manual_seed(H)
    N = 400
    wide = [torch.randint(0, 120, (layers, N + 1, H, bs, D), generator=gen, device=DEV, dtype=torch.uint8) for _ in range(2)]
    scales = [torch.rand(layers, N + 2, H, generator=gen, device=DEV) for _ in range(2)]
    order = torch.randperm(N, generator=torch.Generator().manual_seed(D)).tolist()
    entries = [[order[2 * i % 100 * 2], order[2 * i + 1], random.Random(i).choice([0, 1, bs // 2, bs, bs + 5, -3])] for i in range(150)]
    entries[3][0], entries[40][1], entries[70][0], entries[149][1] = -1, N, N + 7, -9
    entries.insert(60, [5, 5, bs])
    copies = torch.tensor(entries, dtype=torch.int32, device=DEV)
    want = [t.clone() for t in (*wide, *scales)]
    for a, b, n in entries:
        if 0 <= a < N and 0 <= b < N:
            n = min(max(n, 0), bs)
            for t in want[:2]:
                t[:, b, :, :n] = t[:, a, :, :n]
            for t in want[2:]:
                t[:, b] = t[:, a]
    pools = [t[:, :N].view(E4M3) for t in wide] + [t[:, :N] for t in scales]
    dart.copy_blocks(copies, *pools)
    assert all(torch.equal(a, b) for a, b in zip((*wide, *scales), want))
    dart.copy_blocks(copies, *(t[0] for t in pools))  # one layer without its dimension: the same again
    assert all(torch.equal(a, b) for a, b in zip((*wide, *scales), want))
    dart.copy_blocks(copies[:0], *pools)


@pytest.mark.gpu
def test_many_copies_of_many_heads():
    """More entries than a launch has workgroups for, so that a lane looks at each of 64."""
    import dartkv_amd as dart
    layers, N, H = 40, 900, 30
    codes = [torch.randint(0, 120, (layers, N, H, 16, 16), device=DEV, dtype=torch.uint8) for _ in range(2)]
    scales = [torch.rand(layers, N, H, device=DEV) for _ in range(2)]
    source = torch.arange(0, N, 2, device=DEV, dtype=torch.int32)
    copies = torch.stack((source, source + 1, torch.full_like(source, 16)), 1)
    copies[::3] = -1
    copies = copies.contiguous()
    want = [t.clone() for t in (*codes, *scales)]
    at = copies[copies[:, 0] >= 0].long()
    for t in want:
        t[:, at[:, 1]] = t[:, at[:, 0]]
    dart.copy_blocks(copies, *(t.view(E4M3) for t in codes), *scales)
    assert all(torch.equal(a, b) for a, b in zip((*codes, *scales), want))


@pytest.mark.gpu
def test_copies_of_very_many_heads():
    """More heads of all layers than a launch's second dimension counts."""
    import dartkv_amd as dart
    layers, H = 260, 140
    codes = [torch.randint(0, 120, (layers, 3, H, 16, 16), device=DEV, dtype=torch.uint8) for _ in range(2)]
    scales = [torch.rand(layers, 3, H, device=DEV) for _ in range(2)]
    want = [t.clone() for t in (*codes, *scales)]
    for t in want:
        t[:, 1] = t[:, 2]
    dart.copy_blocks(torch.tensor([[2, 1, 16]], dtype=torch.int32, device=DEV), *(t.view(E4M3) for t in codes), *scales)
    assert all(torch.equal(a, b) for a, b in zip((*codes, *scales), want))


@pytest.mark.gpu
def test_a_captured_step_of_beams():
    """fork, reserve and copy, replayed while the beams grow: the same state as eager calls leave."""
    import dartkv_amd as dart
    R, bs = 6, 16

    def cache():
        c = dart.BlockKVCache(R, 60, 2, 16, layers=2, block_size=bs, max_blocks=8, sharing=True)
        c.key_codes.view(torch.uint8).random_(0, 120, generator=torch.Generator(DEV).manual_seed(1))
        c.reserve(torch.tensor([14, 0, 0, 30, 0, 0], device=DEV), 44)
        return c

    sources = torch.tensor([0, 0, 0, 3, 3, 3], device=DEV)
    one = torch.ones(R, dtype=torch.int32, device=DEV)
    eager, replayed = cache(), cache()

    def step(c):
        c.fork(sources)
        plan = c.reserve(one, R, max_tokens=1, positions=True)
        return plan.slots, plan.starts, plan.positions

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(cache())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(replayed)
    rng = random.Random(3)
    for i in range(20):
        sources.copy_(torch.tensor([rng.randrange(3) for _ in range(3)] + [3 + rng.randrange(3) for _ in range(3)]) if i
                      else torch.tensor([0, 0, 0, 3, 3, 3]))
        want = step(eager)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        for name in ("table", "lengths", "free", "state", "shares", "key_codes", "value_codes", "key_scale"):
            a, b = getattr(eager, name), getattr(replayed, name)
            assert torch.equal(a.view(torch.uint8) if a.dtype == E4M3 else a, b.view(torch.uint8) if b.dtype == E4M3 else b), name
        assert want[2].tolist() == [14 + i] * 3 + [30 + i] * 3
    eager.check()


@pytest.mark.gpu
def test_a_prefix_that_ends_within_a_block():
    """A request that begins with another's first tokens does not write into the other's block."""
    import dartkv_amd as dart
    dev, model = Device(2, 10, 4, 16), Model(2, 10, 4, 16)
    for sources, prefix, counts in ((None, None, [50, 0]), ([-1, 0], [0, 20], [0, 7]), ([-1, 0], [0, 16], [1, 20]), ([1, -1], None, [3, 3])):
        if sources:
            dart.fork_blocks(*dev.tables, dev.shares, torch.tensor(sources, device=DEV),
                             prefix and torch.tensor(prefix, device=DEV), block_size=16)
            model.fork(sources, prefix)
            same(dev, model)
        tags = [len(model.tokens[0]) + i for i in range(sum(counts))]
        copies = dart.reserve_blocks(*dev.tables, torch.tensor(counts, device=DEV), len(tags), block_size=16, shares=dev.shares)[2]
        dart.copy_blocks(copies, *dev.pools)
        dev.write(model.reserve(counts, len(tags), tags)[0], tags)
        same(dev, model)


@pytest.mark.gpu
def test_refusals():
    import dartkv_amd as dart
    dev = Device(3, 8, 4, 16)
    s = torch.zeros(3, dtype=torch.int32, device=DEV)
    fork, tables, shares = dart.fork_blocks, dev.tables, dev.shares
    for error, call in (
            (TypeError, lambda: fork(*tables, shares, [0, 0, 0], block_size=16)),
            (TypeError, lambda: fork(*tables, shares, s.float(), block_size=16)),
            (ValueError, lambda: fork(*tables, shares, s[:2], block_size=16)),
            (ValueError, lambda: fork(*tables, shares, s, s[:2], block_size=16)),
            (TypeError, lambda: fork(*tables, None, s, block_size=16)),
            (TypeError, lambda: fork(*tables, shares.long(), s, block_size=16)),
            (ValueError, lambda: fork(*tables, shares[:7], s, block_size=16)),
            (ValueError, lambda: fork(*tables, shares, s, block_size=17)),
            (ValueError, lambda: fork(*tables, shares, s.cpu(), block_size=16)),
            (ValueError, lambda: dart.release_blocks(*tables, s, block_size=16, shares=shares[:4])),
            (TypeError, lambda: dart.reserve_blocks(*tables, s, 0, block_size=16, shares=shares.float())),
            (ValueError, lambda: dart.reserve_blocks(*tables, s, 4, block_size=16, positions=s)),
            (ValueError, lambda: dart.reserve_blocks(*tables, s, 3, block_size=16, positions=s.long())),
            (TypeError, lambda: dart.compact_blocks(*tables, shares.float(), block_size=16)),
            (TypeError, lambda: dart.copy_blocks(s, *dev.pools)),
            (TypeError, lambda: dart.copy_blocks(torch.zeros(2, 3, device=DEV), *dev.pools)),
            (ValueError, lambda: dart.copy_blocks(s[None], *dev.pools[:2], *(t[0] for t in dev.pools[2:]))),
            (ValueError, lambda: dart.copy_blocks(s[None], dev.pools[0][:1], *dev.pools[1:])),
            (TypeError, lambda: dart.copy_blocks(s[None], dev.pools[0].view(torch.uint8), *dev.pools[1:])),
            (ValueError, lambda: dart.copy_blocks(s[None], *dev.pools[:2], dev.pools[2][:, :3], dev.pools[3])),
            (RuntimeError, lambda: dart.copy_blocks(s[None].cpu(), *dev.pools)),
            (ValueError, lambda: dart.BlockKVCache(2, 4, 1, 16).fork(s[:2]))):
        for _ in range(2):
            with pytest.raises(error):
                call()
            fork(*tables, shares, s, block_size=16)
    cache = dart.BlockKVCache(3, 8, 1, 16, sharing=True)
    plan = cache.reserve(s + 1, 3)
    cache.fork(s)
    x = torch.zeros(3, 1, 16, device=DEV)
    with pytest.raises(ValueError, match="earlier reserve"):
        cache.append(0, x, x, plan)
    plan = cache.reserve(s + 1, 3)
    cache.compact()
    with pytest.raises(ValueError, match="earlier reserve"):
        cache.append(0, x, x, plan)


def test_refusals_of_the_c_entries():
    from dartkv_amd import _lib
    lib = _lib.load()
    good = dict(table=256, lengths=256, free=256, state=256, shares=256, sources=256, copies=256, slots=256, starts=256, tokens=256,
                requests=4, max_blocks=4, blocks=64, block_size=16, total=4, workspace=256, workspace_bytes=1 << 20)
    entries = {n: getattr(lib, "dkv_" + n) for n in ("fork_blocks", "compact_blocks", "release_blocks", "reserve_blocks")}
    for change, text in ((dict(requests=0), "requests"), (dict(requests=8191), "requests"), (dict(block_size=48), "block_size"),
                         (dict(max_blocks=0), "block counts"), (dict(blocks=0), "block counts"), (dict(table=0), "NULL")):
        for name, entry in entries.items():
            assert entry(_lib.BlockTablesArgs(**{**good, **change}), None) != 0 and text in lib.dkv_last_error().decode(), name
    for change, names in ((dict(workspace_bytes=100), ("fork_blocks", "compact_blocks", "release_blocks")),
                          (dict(workspace=264), ("fork_blocks", "compact_blocks", "release_blocks")),
                          (dict(shares=264), ("fork_blocks", "compact_blocks", "release_blocks")),
                          (dict(shares=0), ("fork_blocks",)), (dict(sources=0), ("fork_blocks",)),
                          (dict(copies=0), ("compact_blocks", "reserve_blocks")), (dict(positions=260), ("reserve_blocks",)),
                          (dict(blocks=(1 << 20) + 1, workspace_bytes=1 << 40), ("compact_blocks",))):
        for name in names:
            assert entries[name](_lib.BlockTablesArgs(**{**good, **change}), None) != 0, (change, name)
    assert all(entry(None, None) == 1 for entry in entries.values())
    assert lib.dkv_share_workspace_bytes(_lib.BlockTablesArgs(**good)) == 64 * 4 + 4
    assert lib.dkv_share_workspace_bytes(_lib.BlockTablesArgs(**{**good, "requests": 100})) == 100 * 4 * 4 + 4
    copy = dict(copies=256, count=3, layers=2, blocks=8, H=2, block_size=16, D=16, key_codes=256, value_codes=256, key_scale=256,
                value_scale=256, key_stride=4096, value_stride=4096, key_scale_stride=16, value_scale_stride=16)
    for change in (dict(block_size=20), dict(D=24), dict(D=528), dict(count=-1), dict(layers=0), dict(H=0), dict(blocks=0),
                   dict(layers=1 << 20), dict(layers=1 << 19, H=1 << 19), dict(copies=0), dict(key_codes=0), dict(value_scale=0), dict(key_codes=264),
                   dict(value_stride=4100)):
        assert lib.dkv_copy_blocks(_lib.CopyBlocksArgs(**{**copy, **change}), None) != 0, change
    assert lib.dkv_copy_blocks(_lib.CopyBlocksArgs(**{**copy, "count": 0}), None) == 0 and lib.dkv_copy_blocks(None, None) == 1


def test_ctypes_structs_match_the_header(tmp_path):
    import ctypes
    import os
    import subprocess
    from dartkv_amd import _lib
    header = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    structs = {"dkv_block_tables_args": _lib.BlockTablesArgs, "dkv_copy_blocks_args": _lib.CopyBlocksArgs,
               "dkv_rotate_heads_args": _lib.RotateHeadsArgs, "dkv_token_logprobs_args": _lib.TokenLogprobsArgs,
               "dkv_token_logprobs_grads": _lib.TokenLogprobsGrads, "dkv_append_blocks_args": _lib.AppendBlocksArgs}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "dartkv.h"', "int main(void) {"]
    for name, cls in structs.items():
        lines.append(f'  printf("%zu\\n", sizeof({name}));')
        lines += [f'  printf("%zu\\n", offsetof({name}, {field}));' for field, _ in cls._fields_]
    (tmp_path / "layout.c").write_text("\n".join(lines + ["  return 0;", "}"]))
    subprocess.run(["gcc", "-I", header, str(tmp_path / "layout.c"), "-o", str(tmp_path / "layout")], check=True)
    got = [int(n) for n in subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [n for cls in structs.values() for n in (ctypes.sizeof(cls), *(getattr(cls, f).offset for f, _ in cls._fields_))]
