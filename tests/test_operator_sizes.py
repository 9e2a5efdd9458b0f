"""The operators at the sizes where their launches change form: more workgroups than CUs, more than 64 sequences, appends
of many tokens, more than 64 query heads a KV head.  Rows are sampled; bounds are those of test_prompt_attention and
test_blocks (u half a step of the type, W the weighted mean of |v|)."""

from __future__ import annotations

import math
import random

import pytest
import torch

from tests.test_blocks import E4M3, _append64, _cache, _check_attention, _pool, _query, _same_values, _starts, _state
from tests.test_prompt_attention import _check, _packed_check, _rand

DEV = "cuda"


def _some(n, rng, count=24):
    """Rows of n: the first and last, those around tile borders, and some others."""
    rows = {i for i in (0, 1, 31, 32, 63, 64, 127, 128, n - 2, n - 1) if 0 <= i < n}
    return sorted(rows | {rng.randrange(n) for _ in range(count)}) if n else []


def _rows64(q, k, v, rows, seen, scale):
    """(o, W) [rows, Hq, D] in 64 bits: row i of q [n, Hq, D] over the first seen[i] keys of k, v [T, Hkv, D]."""
    o, w = [], []
    H, D = k.shape[1], k.shape[2]
    k, v = k.double().permute(1, 2, 0).contiguous(), v.double().transpose(0, 1).contiguous()
    for i, n in zip(rows, seen):
        p = torch.softmax(torch.matmul(q[i].double().view(H, -1, D), k[..., :n].contiguous()) * scale, -1)
        o.append(torch.matmul(p, v[:, :n].contiguous()).reshape(-1, D))
        w.append(torch.matmul(p, v[:, :n].abs().contiguous()).reshape(-1, D))
    return torch.stack(o).cpu(), torch.stack(w).cpu()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 80, 128, 256])
@pytest.mark.parametrize("lengths", [[700, 3, 1501, 0, 64, 901], [2050, 1100]])
def test_packed_prompts_of_more_workgroups_than_cus(dtype, D, lengths):
    import dartkv_amd as dart
    rng = random.Random(D)
    q, k, v = (_rand((sum(lengths), h, D), dtype, h) for h in (32, 8, 8))
    got = dart.prompt_attention(q, k, v, _starts(lengths))
    at = 0
    for n in lengths:
        part, rows = slice(at, at + n), _some(n, rng)
        if rows:
            o, w = _rows64(q[part], k[part], v[part], rows, [i + 1 for i in rows], 1 / math.sqrt(D))
            _check(got[part][rows], o, w, dtype)
        at += n


@pytest.mark.gpu
@pytest.mark.parametrize("D,causal", [(64, True), (128, True), (128, False), (256, True)])
def test_more_than_64_sequences(D, causal):
    """Their tiles are found a wave's width of sequences at a time, in the sequences' order."""
    import dartkv_amd as dart
    rng = random.Random(3)
    lengths = [rng.choice([0, 1, rng.randint(1, 40)]) for _ in range(150)] + [300, 0, 5]
    total = sum(lengths)
    q, k, v = (_rand((total + 9, h, D), torch.bfloat16, h) for h in (4, 2, 2))
    got = dart.prompt_attention(q, k, v, _starts(lengths), causal=causal)
    _packed_check(got, q, k, v, lengths, lengths, causal, 1 / math.sqrt(D), torch.bfloat16)
    assert bool((got[total:] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("new", [[1500, 1, 700], [1100, 0, 1, 40]])
def test_chunks_of_more_workgroups_than_cus(dtype, D, new):
    """With 256 tiles of 256 rows and more (the first) bf16 has eight waves a workgroup, under that four."""
    import dartkv_amd as dart
    rng = random.Random(D)
    lengths = [n + more for n, more in zip(new, (333, 77, 1, 2000))]
    cache = _cache(lengths, 8, D, 64, D)
    q = _query(sum(new), 32, D, dtype, 4)
    got = dart.block_attention(q, *cache, _starts(new))
    u = torch.finfo(dtype).eps / 2
    at = 0
    for r, n in enumerate(new):
        ids = cache[4][r, :-(-lengths[r] // 64)].long()
        k, v = ((c.view(torch.uint8)[ids].view(E4M3).double() * s[ids].double()[..., None, None])
                .transpose(1, 2).reshape(-1, 8, D)[:lengths[r]] for c, s in ((cache[0], cache[2]), (cache[1], cache[3])))
        rows = _some(n, rng)
        if rows:
            o, w = _rows64(q[at:at + n], k, v, rows, [lengths[r] - n + 1 + i for i in rows], 1 / math.sqrt(D))
            err = (got[at:at + n][rows].double().cpu() - o).abs()
            bound = 1.01 * u * o.abs() + (1.01 * u if dtype == torch.bfloat16 else 2 ** -16) * w
            assert bool((err <= bound).all()), f"request {r}: error is {float((err / bound).max()):.3f} of its bound"
        at += n


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_more_than_64_heads_a_kv_head(dtype, D):
    """Single tokens without starts whose rows the kernel for few rows does not take."""
    import dartkv_amd as dart
    cache = _cache([3000, 9, 64, 1], 2, D, 64, D)
    q = _query(4, 144, D, dtype, 8)
    _check_attention(dart.block_attention(q, *cache), q, cache, [1] * 4, dtype, chunk=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("H,D,bs,R,sizes", [(8, 64, 64, 5, [37, 700, 11]), (32, 32, 16, 3, [5, 300]), (4, 144, 32, 4, [1, 1500]),
                                            (8, 16, 16, 2100, [1, 1, 1])])
def test_appends_of_many_tokens(dtype, H, D, bs, R, sizes):
    """Over 16,384 rows of KV heads a wave looks through 64 tokens for the runs that begin there: ragged requests, blocks
    that held tokens before, slots of -1 between requests' tokens and behind them, and decode steps of many requests."""
    import dartkv_amd as dart
    gen, rng = torch.Generator().manual_seed(D), random.Random(D)
    most = -(-sum(sizes) // bs)
    state = _state(R, R * most + 1, most)
    pool = _pool(R * most + 1, H, bs, D)
    want = [t.float().double().cpu() for t in pool]
    for i, n in enumerate(sizes):
        counts = [n if r % 3 else max(0, n - rng.randint(0, n // 2)) for r in range(R)]
        T = sum(counts) + 70
        slots, starts = dart.reserve_blocks(*state, torch.tensor(counts, device=DEV), T, block_size=bs)
        slots[int(starts[-2]):int(starts[-1])] = -1  # (the last request's tokens are not written)
        spread = 10.0 ** torch.empty(T, H, 1).uniform_(-3, 0.3 * i, generator=gen)
        k, v = ((torch.randn(T, H, D, generator=gen) * spread).to(dtype) for _ in range(2))
        dart.append_blocks(k.to(DEV), v.to(DEV), slots, *pool)
        for x, c, s in ((k, want[0], want[2]), (v, want[1], want[3])):
            _append64(x, slots.cpu().tolist(), c, s, bs)
    assert max(sizes) * R * H > 16384
    for got, w in zip(pool, want):
        _same_values(got, w)


@pytest.mark.gpu
def test_tables_of_the_most_requests():
    """8,190 requests, whose prefix sums take 96 KiB of LDS; one more is refused."""
    import dartkv_amd as dart
    from tests.test_blocks import TableModel, _same_state
    R, bs, most = 8190, 16, 3
    rng = random.Random(1)
    state, model = _state(R, R * most, most), TableModel(R, R * most, most, bs)
    for _ in range(2):
        counts = [rng.choice([0, 1, rng.randint(0, 20)]) for _ in range(R)]
        total = sum(counts) + 5
        slots, starts = dart.reserve_blocks(*state, torch.tensor(counts, dtype=torch.int32, device=DEV), total, block_size=bs)
        want_slots, want_starts = model.reserve(counts, total)
        assert slots.cpu().tolist() == want_slots and starts.cpu().tolist() == want_starts
        _same_state(state, model)
        drop = [rng.randint(0, 9) for _ in range(R)]
        dart.release_blocks(*state, torch.tensor(drop, dtype=torch.int32, device=DEV), block_size=bs)
        model.release(drop)
        _same_state(state, model)
    with pytest.raises(ValueError, match="8190"):
        dart.release_blocks(*_state(R + 1, R, 1), block_size=bs)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_single_tokens_of_many_requests(dtype):
    import dartkv_amd as dart
    rng = random.Random(5)
    lengths = [rng.choice([1, 16, rng.randint(1, 60)]) for _ in range(2000)] + [3000, 1]
    cache = _cache(lengths, 2, 64, 16, 9)
    q = _query(len(lengths), 8, 64, dtype, 2)
    _check_attention(dart.block_attention(q, *cache), q, cache, [1] * len(lengths), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
def test_chunks_among_more_than_64_requests(dtype, D):
    """The kernel for few rows takes the requests of up to 16 rows, the chunk kernel finds the others among all."""
    import dartkv_amd as dart
    rng = random.Random(6)
    new = [rng.choice([0, 1, 1, 1, 4, 5, 40]) for _ in range(150)] + [100, 0, 1]
    lengths = [max(1, n) + rng.randint(0, 70) for n in new]
    cache = _cache(lengths, 2, D, 16, D)
    q = _query(sum(new) + 3, 8, D, dtype, 3)
    got = dart.block_attention(q, *cache, _starts(new))
    _check_attention(got, q, cache, new, dtype, chunk=True)
    assert bool((got[sum(new):] == 0).all())
