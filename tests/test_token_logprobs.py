"""token_logprobs: log probabilities, entropy, alternatives and the gradient, against the definition in 64 bits.

Tolerances (all fp32).  A thread adds up to V / 256 + 32 terms of its own, then 6 lanes, 4 waves and up to 38 parts come
together: n = V / 256 + 128 additions on any way, each 2^-24 of the sum, whose terms all have one sign.  A term 2^z is
off by 2^-22 (|z| + 2) relative; |z| 2^z is at most 0.54, and sum 2^z |z| / s = t / s.  So ln s is off by at most
n 2^-24 + 2^-21 (1 + t / s) and its own rounding, t / s by as much of itself:
  log p:   2^-23 |x - m| + e,   e = (n 2^-24 + 2^-20) (1 + t / s) + 2^-23 ln s
  entropy: 2 e
  gradient: the type's half step of it, and p times: (2^-21 (|z| + 4) + 4 e) (|G| + |h| (|log p| + H)) + |h| 2 e.
"""

from __future__ import annotations

import math

import pytest
import torch

DEV = "cuda"


@pytest.fixture(autouse=True)
def _seed():
    torch.manual_seed(0)


HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -124, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -124}  # (2^z is 0 below 2^-126)


def expected(x, tokens):
    """x [T, V] in 64 bits: log probabilities of tokens and of all, entropy, and the error e of each row."""
    m = x.amax(-1, keepdim=True)
    z = x - m
    s = z.exp().sum(-1, keepdim=True)
    logp = z - s.log()
    p = logp.exp()
    entropy = torch.special.entr(p).sum(-1)
    spread = -(p * z.clamp_min(-1e300)).sum(-1)
    n = x.shape[-1] / 256 + 128
    e = (n * 2.0 ** -24 + 2.0 ** -20) * (1 + spread) + 2.0 ** -23 * s.log().squeeze(-1)
    return logp.gather(1, tokens[:, None]).squeeze(1), logp, entropy, z, e


def check(out, logits, tokens, top):
    x = logits.detach().double().cpu()
    got, logp, entropy, z, e = expected(x, tokens.cpu().long())
    picked = z.gather(1, tokens.cpu().long()[:, None]).squeeze(1)
    fine = torch.isfinite(picked)
    error = (out.logprobs.detach().double().cpu() - got).abs()
    assert bool((error[fine] <= (2.0 ** -23 * picked.abs() + e)[fine]).all()), float(error[fine].max())
    assert bool((out.logprobs.detach().cpu()[~fine] == -math.inf).all())
    error = (out.entropy.detach().double().cpu() - entropy).abs()
    assert bool((error <= 2 * e).all()), float((error / e).max())
    ids = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(out.top_tokens.cpu(), ids)
    want, away = logp.gather(1, ids), z.gather(1, ids)
    real = torch.isfinite(want)
    error = (out.top_logprobs.detach().double().cpu() - want).abs()
    limit = 2.0 ** -23 * away.abs() + e[:, None]
    assert bool((error[real] <= limit[real]).all()) and bool((out.top_logprobs.detach().cpu()[~real] == -math.inf).all())
    assert out.top_logprobs.dtype == torch.float32 and out.top_tokens.dtype == torch.int64


def rows(T, V, dtype, seed, spread=3.0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(T, V, generator=gen) * torch.empty(T, 1).uniform_(0.2, spread, generator=gen)
    return x.to(dtype), torch.randint(0, V, (T,), generator=gen)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,V,top", [(1, 1, 1), (3, 2, 2), (2, 63, 63), (5, 64, 64), (1, 1000, 5), (7, 4097, 20),
                                     (2, 8191, 64), (1, 32768, 1), (64, 32001, 20), (3, 151936, 64), (300, 1537, 3),
                                     (2100, 333, 7), (1, 151936, 0), (9, 2055, 0), (2049, 9001, 33), (2300, 4500, 0)])
def test_against_64_bits(T, V, top, dtype):
    import dartkv_amd as dart
    x, tokens = rows(T, V, dtype, V + T)
    out = dart.token_logprobs(x.to(DEV), tokens.to(DEV), top=top)
    check(out, x, tokens, top)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind", ["rising", "falling", "equal", "two", "coarse", "peak", "zeros"])
def test_orders_that_a_selection_finds_hard(kind, dtype):
    """Rows whose every value displaces the last, ties all over, and one value far above."""
    import dartkv_amd as dart
    V = 20011
    ramp = torch.linspace(-8, 8, V)
    x = {"rising": ramp, "falling": ramp.flip(0), "equal": torch.full((V,), 1.5), "two": (torch.arange(V) % 2).float(),
         "coarse": (torch.arange(V) * 7919 % 13).float(), "peak": torch.zeros(V).index_fill_(0, torch.tensor([V - 1]), 80.0),
         "zeros": torch.where(torch.arange(V) % 3 == 0, -0.0, 0.0)}[kind]
    x = torch.stack((x, x.roll(5003))).to(dtype)
    for T in (2, 600):  # rows in parts, and whole
        logits = x.repeat(T // 2, 1)
        tokens = torch.arange(T) * 31 % V
        check(dart.token_logprobs(logits.to(DEV), tokens.to(DEV), top=33), logits, tokens, 33)
    # a wave for each of very many rows
    T = 2200
    logits, tokens = x.repeat(T // 2, 1).to(DEV), torch.tensor([31, 62]).repeat(T // 2).to(DEV)
    out = dart.token_logprobs(logits, tokens, top=33)
    check(dart.TokenLogprobs(*(t[:8] for t in out)), x.repeat(4, 1), tokens[:8], 33)
    # (rows of an odd size begin at eight offsets, each with an order of its sums)
    assert all(torch.equal(t, t[:8].repeat(T // 8, *[1] * (t.dim() - 1))) for t in out)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_masked_rows(dtype):
    import dartkv_amd as dart
    x, tokens = rows(6, 5000, dtype, 3)
    low = torch.finfo(dtype).min
    x[0, torch.arange(5000) != 4321] = -math.inf  # one token is allowed
    x[1, 100:] = -math.inf
    x[2] = -math.inf  # none
    x[3] = low  # a row of equals
    x[4, :4990] = low
    x[5, :2500] = torch.finfo(dtype).max / 4
    tokens[0], tokens[1], tokens[4] = 4321, 200, 4995
    out = dart.token_logprobs(x.to(DEV), tokens.to(DEV), top=12)
    keep = [0, 1, 3, 4, 5]
    check(dart.TokenLogprobs(*(t[keep] for t in out)), x[keep], tokens[keep], 12)
    assert out.logprobs[0] == 0 and out.entropy[0] == 0 and out.logprobs[2] == -math.inf and out.entropy[2] == 0
    assert out.top_tokens[2].tolist() == list(range(12)) and bool((out.top_logprobs[2] == -math.inf).all())
    leaf = x.to(DEV).requires_grad_()
    out = dart.token_logprobs(leaf, tokens.to(DEV))
    grad = torch.autograd.grad(out.logprobs[keep].clamp_min(-100).sum() + out.entropy.sum(), leaf)[0]
    assert not grad[2].any() and bool(grad[keep].isfinite().all()) and not grad[1, 100:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("T", [24, 2112])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_maxima_that_come_late(T, dtype):
    """Rows that rise by far more than 2^z can hold between what a thread reads first and last, and rows that begin with
    masked logits."""
    import dartkv_amd as dart
    x, tokens = rows(3, 30011, dtype, 20)
    x[0] += torch.linspace(0, 200, 30011).to(dtype)
    x[1, :20000] = -math.inf
    x[2, 29000:] += 95
    tokens = torch.tensor([30000, 25000, 29500])
    out = dart.token_logprobs(x.repeat(T // 3, 1).to(DEV), tokens.repeat(T // 3).to(DEV), top=11)
    check(dart.TokenLogprobs(*(t[:24] for t in out)), x.repeat(8, 1), tokens.repeat(8), 11)
    assert all(torch.equal(t, t[:24].repeat(T // 24, *[1] * (t.dim() - 1))) for t in out)


@pytest.mark.gpu
def test_values_that_are_not_finite():
    import dartkv_amd as dart
    x, tokens = rows(5, 3001, torch.float32, 4)
    x[1, 77], x[2, 2999], x[3] = math.nan, math.inf, math.nan
    x[4, 5:] = math.nan
    out = dart.token_logprobs(x.to(DEV), tokens.to(DEV), top=8)
    assert bool(out.logprobs[1:].isnan().all()) and bool(out.entropy[1:].isnan().all())
    check(dart.TokenLogprobs(*(t[:1] for t in out)), x[:1], tokens[:1], 8)
    order = torch.sort(x.nan_to_num(-math.inf, math.inf), dim=-1, descending=True, stable=True).indices[:, :8]
    assert torch.equal(out.top_tokens[1:3].cpu(), order[1:3]) and out.top_tokens[3].tolist() == [-1] * 8
    assert out.top_tokens[4].tolist() == [*order[4, :5].tolist(), -1, -1, -1]
    assert bool(out.top_logprobs[1:].isnan().all())


@pytest.mark.gpu
def test_tokens_of_no_interest_and_behind_the_vocabulary():
    import dartkv_amd as dart
    x, _ = rows(5, 999, torch.bfloat16, 5)
    leaf = x.to(DEV).requires_grad_()
    for kind in (torch.int32, torch.int64):
        tokens = torch.tensor([-1, 998, 999, -100, 0], dtype=kind, device=DEV)
        out = dart.token_logprobs(leaf, tokens)
        assert out.logprobs[0] == 0 and out.logprobs[3] == 0 and bool(out.logprobs[2].isnan())
        assert bool((out.logprobs[[1, 4]] < 0).all())
        grad = torch.autograd.grad(out.logprobs, leaf, torch.ones(5, device=DEV))[0]
        assert not grad[[0, 2, 3]].any() and bool(grad[[1, 4]].any(-1).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,V,top", [(1, 5, 0), (1, 1, 1), (4, 2049, 3), (17, 32003, 20), (2, 151936, 64), (700, 511, 5)])
def test_gradients_against_the_formula(T, V, top, dtype):
    import dartkv_amd as dart
    x, tokens = rows(T, V, dtype, 6 + V)
    gen = torch.Generator().manual_seed(7)
    g, h, g_top = torch.randn(T, generator=gen), torch.randn(T, generator=gen), torch.randn(T, top, generator=gen)
    leaf = x.to(DEV).requires_grad_()
    out = dart.token_logprobs(leaf, tokens.to(DEV), top=top)
    got = torch.autograd.grad(out[:3], leaf, [t.to(DEV) for t in (g, h, g_top)])[0].double().cpu()
    _, logp, entropy, z, e = expected(x.double(), tokens)
    p, G = logp.exp(), (g + g_top.sum(-1)).double()[:, None]
    g, h, g_top, entropy, e = g.double()[:, None], h.double()[:, None], g_top.double(), entropy[:, None], e[:, None]
    want = -p * (G + h * (logp + entropy))
    want.scatter_add_(1, tokens[:, None], g)
    want.scatter_add_(1, out.top_tokens.cpu(), g_top)
    size = p * ((2.0 ** -21 * (z.abs() / math.log(2) + 4) + 4 * e) * (G.abs() + h.abs() * (logp.abs() + entropy)) + 2 * e * h.abs())
    # (fp32 sums of the gradients at one place: up to 65 of them)
    points = torch.zeros_like(want).scatter_add_(1, tokens[:, None], g.abs()).scatter_add_(1, out.top_tokens.cpu(), g_top.abs())
    limit = HALF_STEP[dtype] * want.abs() * (1 + 2.0 ** -8) + size + 2.0 ** -18 * (points + p * (g.abs() + g_top.abs().sum(-1, keepdim=True))) + TINY[dtype]
    error = (got - want).abs()
    assert bool((error <= limit).all()), float((error / limit).max())


def test_the_formula_against_differences():
    gen = torch.Generator().manual_seed(8)
    x, g, h = torch.randn(1, 40, dtype=torch.float64, generator=gen), 0.7, -1.3
    token = torch.tensor([11])

    def loss(x):
        got, _, entropy, _, _ = expected(x, token)
        return g * got[0] + h * entropy[0]

    _, logp, entropy, _, _ = expected(x, token)
    p = logp.exp()
    want = -p * (g + h * (logp + entropy))
    want[0, 11] += g
    for i in range(40):
        step = torch.zeros_like(x)
        step[0, i] = 1e-5  # (h^2 and 2^-52 / h are below 1e-9)
        assert abs((loss(x + step) - loss(x - step)) / 2e-5 - want[0, i]) < 1e-8


@pytest.mark.gpu
def test_gradients_against_differences_of_the_operator():
    """Along one direction: the quotient is off by the outputs' errors over h, and by what the quotient in 64 bits is off
    from the derivative."""
    import dartkv_amd as dart
    x, tokens = rows(3, 700, torch.float32, 9)
    gen = torch.Generator().manual_seed(10)
    v, g, h, d = torch.randn(3, 700, generator=gen), torch.randn(3, generator=gen), torch.randn(3, generator=gen), 2.0 ** -5

    def loss(x):
        out = dart.token_logprobs(x.to(DEV), tokens.to(DEV))
        return (out.logprobs.double().cpu() * g + out.entropy.double().cpu() * h).sum()

    def loss64(x):
        got, _, entropy, z, e = expected(x.double(), tokens)
        return (got * g + entropy * h).sum(), ((2.0 ** -23 * z.abs().amax(-1) + e) * g.abs() + 2 * e * h.abs()).sum()

    ends = [x + d * v, x - d * v]
    quotient = (loss(ends[0]) - loss(ends[1])) / (2 * d)
    quotient64, rounding = (loss64(ends[0])[0] - loss64(ends[1])[0]) / (2 * d), (loss64(ends[0])[1] + loss64(ends[1])[1]) / (2 * d)
    leaf = x.to(DEV).requires_grad_()
    out = dart.token_logprobs(leaf, tokens.to(DEV))
    derivative = (torch.autograd.grad(out[:2], leaf, (g.to(DEV), h.to(DEV)))[0].double().cpu() * v).sum()
    x64 = x.double().requires_grad_()
    derivative64 = (torch.autograd.grad(loss64(x64)[0], x64)[0] * v).sum()
    assert abs(quotient - derivative) <= rounding + abs(quotient64 - derivative64) + 2.0 ** -14 * v.abs().amax() * (g.abs() + h.abs() * 8).sum()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_layouts_give_one_result(dtype):
    """Rows that begin anywhere, strides, more dimensions, one row for all tokens, and the gradients' layouts."""
    import dartkv_amd as dart
    T, V = 6, 3333
    x, tokens = rows(T, V, dtype, 11)
    x, tokens = x.to(DEV), tokens.to(DEV)
    want = dart.token_logprobs(x, tokens, top=5)
    wide = torch.full((T, V + 13), 99.0, dtype=dtype, device=DEV)
    columns = torch.empty(V, T, dtype=dtype, device=DEV).t()
    g = torch.randn(T, device=DEV)
    leaf = x.clone().requires_grad_()
    grad = torch.autograd.grad(dart.token_logprobs(leaf, tokens, top=5)[:2], leaf, (g, g))[0]
    for layout in [wide[:, at:at + V] for at in range(0, 9)] + [columns]:
        layout.copy_(x)
        got = dart.token_logprobs(layout, tokens.int(), top=5)
        # (other parts of the row in other threads: sums in another order)
        assert torch.equal(got.top_tokens, want.top_tokens)
        check(got, x, tokens, 5)
        leaf = layout.detach().requires_grad_()
        again = torch.autograd.grad(dart.token_logprobs(leaf, tokens, top=5)[:2], leaf, (g, g))[0]
        assert bool(((again.double() - grad.double()).abs() <= 2 * HALF_STEP[dtype] * grad.double().abs() + 2.0 ** -18).all())
    got = dart.token_logprobs(x.view(2, 3, V), tokens.view(2, 3), top=5)
    assert all(torch.equal(a.reshape(b.shape), b) for a, b in zip(got, want)) and got.top_tokens.shape == (2, 3, 5)
    got = dart.token_logprobs(x[0], tokens[0], top=5)
    assert got.logprobs.shape == () and got.top_tokens.shape == (5,) and torch.equal(got.top_tokens, want.top_tokens[0])
    row = x[:1].expand(T, V)
    check(dart.token_logprobs(row, tokens, top=2), row, tokens, 2)
    leaf = x[:1].clone().requires_grad_()
    out = dart.token_logprobs(leaf.expand(T, V), tokens)
    shared = torch.autograd.grad(out.logprobs, leaf, g)[0]
    each = [torch.autograd.grad(dart.token_logprobs(leaf, t[None]).logprobs, leaf, g[i:i + 1])[0] for i, t in enumerate(tokens)]
    total = torch.stack(each).double().sum(0)
    size = torch.stack(each).double().abs().sum(0)
    assert bool(((shared.double() - total).abs() <= 8 * HALF_STEP[dtype] * size + 2.0 ** -18).all())


@pytest.mark.gpu
def test_the_same_result_every_time():
    import dartkv_amd as dart
    for T, V in ((1, 151936), (40, 40000)):
        x, tokens = (t.to(DEV) for t in rows(T, V, torch.bfloat16, 12))
        first = dart.token_logprobs(x, tokens, top=20)
        for _ in range(5):
            assert all(torch.equal(a, b) for a, b in zip(dart.token_logprobs(x, tokens, top=20), first))


@pytest.mark.gpu
@pytest.mark.parametrize("T,V", [(3, 50001), (2500, 401)])
def test_captured_with_its_gradient(T, V):
    import dartkv_amd as dart
    x, tokens = (t.to(DEV) for t in rows(T, V, torch.bfloat16, 13))
    g = torch.randn(T, device=DEV)

    def step(x):
        leaf = x.detach().requires_grad_()
        out = dart.token_logprobs(leaf, tokens, top=4)
        return [t.detach() for t in out] + [torch.autograd.grad(out[:2], leaf, (g, g))[0]]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):  # two graphs of their own workspaces
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step(x)
        graphs.append((graph, got))
    for i in range(3):
        x.normal_(generator=torch.Generator(DEV).manual_seed(i))
        tokens.copy_(torch.randint(-1, V, (T,)))
        want = step(x)
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, got in graphs:
            assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_two_streams_at_once():
    import dartkv_amd as dart
    data = [tuple(t.to(DEV) for t in rows(8, 100003, torch.bfloat16, 14 + i)) for i in range(2)]
    want = [dart.token_logprobs(*d, top=16) for d in data]
    streams = [torch.cuda.Stream() for _ in data]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(6):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(dart.token_logprobs(*data[i], top=16))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for i in range(2) for out in got[i] for a, b in zip(out, want[i]))


@pytest.mark.gpu
def test_nothing_to_do():
    import dartkv_amd as dart
    x = torch.zeros(0, 100, device=DEV, requires_grad=True)
    out = dart.token_logprobs(x, torch.zeros(0, dtype=torch.int64, device=DEV), top=3)
    assert out.logprobs.shape == (0,) and out.top_tokens.shape == (0, 3)
    assert torch.autograd.grad(out.logprobs.sum(), x)[0].shape == (0, 100)


@pytest.mark.gpu
def test_refusals():
    import torch.autograd.forward_ad as forward
    import dartkv_amd as dart
    x, t = torch.zeros(4, 70, device=DEV), torch.zeros(4, dtype=torch.int64, device=DEV)
    call = dart.token_logprobs
    for error, args, kwargs in (
            (TypeError, (x.double(), t), {}), (TypeError, (x, t.float()), {}), (TypeError, (x, [0] * 4), {}), (ValueError, (x, t[:3]), {}),
            (ValueError, (x, t[:, None]), {}), (ValueError, (x[:, :0], t), {}), (ValueError, (x, t), dict(top=65)),
            (ValueError, (x[:, :5], t), dict(top=6)), (ValueError, (x, t), dict(top=-1)), (RuntimeError, (x.cpu(), t), {}),
            (RuntimeError, (x, t.cpu()), {})):
        for _ in range(2):
            with pytest.raises(error):
                call(*args, **kwargs)
            call(x, t, top=3)
    leaf = x.clone().requires_grad_()
    once = torch.autograd.grad(call(leaf, t).logprobs.sum(), leaf, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        torch.autograd.grad(once.sum(), leaf)
    with forward.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        call(forward.make_dual(x, torch.ones_like(x)), t)


def test_refusals_of_the_c_entries():
    from dartkv_amd import _lib
    lib = _lib.load()
    good = dict(logits=256, tokens=256, logprobs=256, entropy=256, stats=256, top_logprobs=256, top_tokens=256, stride=100,
                rows=4, vocab=100, top=5, dtype=2)
    for change, text in ((dict(dtype=3), "bf16"), (dict(rows=-1), "counts"), (dict(vocab=0), "counts"),
                         (dict(vocab=1 << 31), "counts"), (dict(top=65), "top"), (dict(top=-1), "top"),
                         (dict(vocab=4), "top"), (dict(logits=257), "rows"), (dict(stride=-1), "rows"), (dict(logits=0), "NULL")):
        a = _lib.TokenLogprobsArgs(**{**good, **change})
        for call in (lambda a: lib.dkv_token_logprobs(a, None),
                     lambda a: lib.dkv_token_logprobs_backward(a, _lib.TokenLogprobsGrads(out=256, stride=100), None)):
            assert call(a) != 0 and text in lib.dkv_last_error().decode(), (change, lib.dkv_last_error())
    assert lib.dkv_token_logprobs(_lib.TokenLogprobsArgs(**{**good, "vocab": 100000, "stride": 100000}), None) == 1
    assert "workspace" in lib.dkv_last_error().decode()
    for change, grads in ((dict(stats=0), dict(out=256, stride=100)), ({}, dict(out=0, stride=100)), ({}, dict(out=256, stride=99)),
                          (dict(top_tokens=0), dict(out=256, stride=100, top_logprobs=256))):
        a, g = _lib.TokenLogprobsArgs(**{**good, **change}), _lib.TokenLogprobsGrads(**grads)
        assert lib.dkv_token_logprobs_backward(a, g, None) == 1
    empty = _lib.TokenLogprobsArgs(**{**good, "rows": 0})
    assert lib.dkv_token_logprobs(empty, None) == 0 and lib.dkv_token_logprobs(None, None) == 1
    assert lib.dkv_token_logprobs_backward(empty, _lib.TokenLogprobsGrads(), None) == 0
    assert lib.dkv_token_logprobs_backward(empty, None, None) == 1
    assert lib.dkv_token_logprobs_workspace_bytes(empty) == 0
    assert lib.dkv_token_logprobs_workspace_bytes(_lib.TokenLogprobsArgs(**good)) == 0  # a row is one part


def test_operators_want_the_gpu():
    import dartkv_amd as dart
    with pytest.raises(RuntimeError, match="ROCm"):
        dart.token_logprobs(torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64))
