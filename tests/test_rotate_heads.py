"""rotate_heads: norm and rotation of heads, and its gradients, against the formulas in 64 bits.

Tolerances.  u is half a step of the type (bf16 2^-8, fp16 2^-11, fp32 2^-24).  In fp32 the sum of up to 256 squares is
off by at most 2^-18 relative whatever the order, its root by half of that, and the products around by a few 2^-24, so a
result before its rounding is off by at most 2^-18 N, N the sum of its terms' magnitudes; then u |y| of the rounding (and
half of fp16's smallest step, 2^-25).  A gradient takes two such sums: 2^-17 of its terms' magnitudes.  A weight's gradient
adds rows: a thread up to 40 after each other here, then lanes, waves and workgroups, fewer than 256 additions on any
way: 256 * 2^-24 of the terms' magnitudes beside their own 2^-17.
"""

from __future__ import annotations

import pytest
import torch

DEV = "cuda"


@pytest.fixture(autouse=True)
def _seed():
    torch.manual_seed(0)


HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -149}


def reference(x, w, cos, sin, interleaved, eps=1e-6):
    """x [T, H, D] in 64 bits, cos and sin [T, half]; the outputs, and the magnitudes of their terms."""
    D, half = x.shape[-1], cos.shape[-1]
    xh = x if w is None else x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    n = xh if w is None else xh * w
    out, size = n.clone(), n.abs()
    i = torch.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    c, s = cos[:, None], sin[:, None]
    out[..., a], out[..., b] = n[..., a] * c - n[..., b] * s, n[..., b] * c + n[..., a] * s
    for one, other in ((a, b), (b, a)):
        size[..., one] = n[..., one].abs() * c.abs() + n[..., other].abs() * s.abs()
    return out, size


def gradients(x, w, cos, sin, interleaved, g, eps=1e-6):
    """From the formulas: dx and dw, and the magnitudes of their terms."""
    half = cos.shape[-1]
    i = torch.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    c, s = cos[:, None], sin[:, None]
    h, size = g.clone(), g.abs()
    h[..., a], h[..., b] = g[..., a] * c + g[..., b] * s, g[..., b] * c - g[..., a] * s
    for one, other in ((a, b), (b, a)):
        size[..., one] = g[..., one].abs() * c.abs() + g[..., other].abs() * s.abs()
    if w is None:
        return h, None, size, None
    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    y = x * r
    dx = r * (h * w - y * (h * w * y).mean(-1, keepdim=True))
    dx_size = r * (size * w.abs() + y.abs() * (size * w.abs() * y.abs()).mean(-1, keepdim=True))
    return dx, (h * y).sum((0, 1)), dx_size, (size * y.abs()).sum((0, 1))


def angles(rows, half, dtype, seed):
    t = torch.rand(rows, half, dtype=torch.float64, generator=torch.Generator().manual_seed(seed)) * 6.28
    return t.cos().to(dtype), t.sin().to(dtype)


def inputs(T, Hq, Hkv, D, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    size = torch.empty(1, Hq + Hkv, 1).uniform_(-2, 2, generator=gen).exp()
    x = (torch.randn(T, Hq + Hkv, D, generator=gen) * size).to(dtype)
    return x.split([Hq, Hkv], 1)


def close(got, want, size, factor):
    u = HALF_STEP[got.dtype]
    error = (got.double().cpu() - want).abs()
    limit = u * want.abs() + factor * size + TINY[got.dtype]
    assert bool((error <= limit).all()), float((error / limit).max())


CASES = [(1, 32, 8, 128, 128, False), (64, 4, 1, 64, 64, False), (37, 14, 2, 80, 80, False), (5, 3, 3, 256, 128, False),
         (130, 6, 2, 72, 18, True), (9, 1, 1, 8, 8, False), (33, 5, 5, 96, 48, True), (17, 7, 1, 200, 200, True),
         (3, 2, 1, 112, 2, False), (50, 2, 2, 256, 254, False), (20, 2, 2, 136, 6, True), (600, 40, 8, 128, 64, True)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,Hq,Hkv,D,turned,interleaved", CASES)
def test_forward_and_gradients_against_64_bits(T, Hq, Hkv, D, turned, interleaved, dtype):
    import dartkv_amd as dart
    q, k = inputs(T, Hq, Hkv, D, dtype, T)
    P = 50
    wide = T % 2 == 0
    angle_dtype = dtype if T % 3 == 0 else torch.float32
    cos, sin = angles(P, turned // 2, angle_dtype, T)
    gen = torch.Generator().manual_seed(T + 1)
    positions = torch.randint(0, P, (T,), generator=gen, dtype=torch.int64 if wide else torch.int32)
    wq, wk = ((1 + torch.randn(D, generator=gen) / 2).to(torch.float32 if T % 2 else dtype) for _ in range(2))
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, wq, wk)]
    out = dart.rotate_heads(*leaves[:2], cos.to(DEV), sin.to(DEV), positions.to(DEV), q_weight=leaves[2],
                            k_weight=leaves[3], interleaved=interleaved)
    given = [torch.randn(t.shape, generator=gen).to(dtype) for t in (q, k)]
    got = torch.autograd.grad(out, leaves, [g.to(DEV) for g in given])
    with torch.no_grad():
        again = dart.rotate_heads(*leaves[:2], cos.to(DEV), sin.to(DEV), positions.to(DEV), q_weight=leaves[2],
                                  k_weight=leaves[3], interleaved=interleaved)
    c, s = cos.double()[positions.long()], sin.double()[positions.long()]
    for i, (x, w) in enumerate(((q, wq), (k, wk))):
        want, size = reference(x.double(), w.double(), c, s, interleaved)
        assert out[i].shape == x.shape and torch.equal(out[i], again[i])
        close(out[i].detach(), want, size, 2.0 ** -18)
        dx, dw, dx_size, dw_size = gradients(x.double(), w.double(), c, s, interleaved, given[i].double())
        close(got[i], dx, dx_size, 2.0 ** -17)
        assert got[2 + i].dtype == w.dtype
        close(got[2 + i], dw, dw_size, 2.0 ** -16 + 2.0 ** -17)


def test_the_formulas_against_differences():
    x = torch.randn(3, 2, 16, dtype=torch.float64, generator=torch.Generator().manual_seed(1))
    w = torch.randn(16, dtype=torch.float64, generator=torch.Generator().manual_seed(2))
    g = torch.randn(3, 2, 16, dtype=torch.float64, generator=torch.Generator().manual_seed(3))
    for turned, interleaved in ((16, False), (12, True), (6, False)):
        cos, sin = angles(3, turned // 2, torch.float64, 4)
        dx, dw, _, _ = gradients(x, w, cos, sin, interleaved, g)
        h = 1e-5  # (the quotient is off by about h^2 and 2^-52 / h, both below 1e-9)

        def loss(x, w):
            return (reference(x, w, cos, sin, interleaved)[0] * g).sum()

        for i in range(16):
            step = torch.zeros_like(w)
            step[i] = h
            assert abs((loss(x, w + step) - loss(x, w - step)) / (2 * h) - dw[i]) < 1e-7
            step = torch.zeros_like(x)
            step[1, 1, i] = h
            assert abs((loss(x + step, w) - loss(x - step, w)) / (2 * h) - dx[1, 1, i]) < 1e-7


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,Hq,Hkv,D,turned,interleaved", [(3301, 33, 7, 128, 128, False), (8201, 3, 1, 72, 36, True),
                                                           (4801, 3, 1, 40, 18, False), (3301, 40, 1, 64, 32, False)])
def test_many_rows(T, Hq, Hkv, D, turned, interleaved, dtype):
    """Waves that make several rows a lane; tokens change between their rows, some of which are no token's."""
    import dartkv_amd as dart
    q, k = inputs(T, Hq, Hkv, D, dtype, T)
    cos, sin = angles(77, turned // 2, torch.float32, T)
    gen = torch.Generator().manual_seed(T)
    positions = torch.randint(0, 77, (T,), generator=gen)
    none = torch.rand(T, generator=gen) < 0.1
    w = 1 + torch.randn(D, generator=gen) / 2
    out = dart.rotate_heads(q.to(DEV), k.to(DEV), cos.to(DEV), sin.to(DEV), torch.where(none, -1, positions).to(DEV),
                            q_weight=w.to(DEV), k_weight=w.to(DEV), interleaved=interleaved)
    for got, x in zip(out, (q, k)):
        want, size = reference(x.double(), w.double(), cos.double()[positions], sin.double()[positions], interleaved)
        assert not got[none.to(DEV)].any()
        close(got[~none.to(DEV)], want[~none], size[~none], 2.0 ** -18)


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_gradients_against_differences_of_the_operator(interleaved):
    """Along one direction in fp32: the quotient is off by the sums' roundings over h, and by what the quotient in 64
    bits is off from the derivative."""
    import dartkv_amd as dart
    T, H, D, h = 6, 3, 64, 2.0 ** -6
    q, k = inputs(T, H, H, D, torch.float32, 5)
    cos, sin = angles(T, 16, torch.float32, 6)
    gen = torch.Generator().manual_seed(7)
    w, v, vw = torch.rand(D, generator=gen) + 0.5, torch.randn(T, H, D, generator=gen), torch.randn(D, generator=gen)
    g = torch.randn(T, H, D, generator=gen)

    def turn(x, w):
        return dart.rotate_heads(x.to(DEV), k.to(DEV), cos.to(DEV), sin.to(DEV), q_weight=w.to(DEV),
                                 interleaved=interleaved)[0].double().cpu()

    def turn64(x, w):
        return reference(x.double(), w.double(), cos.double(), sin.double(), interleaved)

    ends = [(q + t * v, w + t * vw) for t in (h, -h)]
    quotient = ((turn(*ends[0]) - turn(*ends[1])) * g.double()).sum() / (2 * h)
    quotient64 = ((turn64(*ends[0])[0] - turn64(*ends[1])[0]) * g.double()).sum() / (2 * h)
    x, wd = q.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    out = dart.rotate_heads(x, k.to(DEV), cos.to(DEV), sin.to(DEV), q_weight=wd, interleaved=interleaved)[0]
    dx, dw = torch.autograd.grad(out, (x, wd), g.to(DEV))
    derivative = (dx.double().cpu() * v).sum() + (dw.double().cpu() * vw).sum()
    d64 = gradients(q.double(), w.double(), cos.double(), sin.double(), interleaved, g.double())
    rounding = sum((turn64(*e)[1] * g.double().abs()).sum() for e in ends) * 2.0 ** -18 / (2 * h)
    away = abs(quotient64 - ((d64[0] * v).sum() + (d64[1] * vw).sum()))
    own = ((d64[2] * v.abs()).sum() + (d64[3] * vw.abs()).sum()) * 2.0 ** -16
    assert abs(quotient - derivative) <= rounding + away + own


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_layouts_give_one_result(dtype):
    """A batch, views of a projection, strides and offsets that are copied: each row's result is the same."""
    import dartkv_amd as dart
    B, T, Hq, Hkv, D = 3, 21, 6, 2, 64
    q, k = inputs(B * T, Hq, Hkv, D, dtype, 8)
    cos, sin = angles(B * T, 32, torch.float32, 9)
    w = torch.rand(D) + 0.5
    args = dict(q_weight=w.to(DEV), k_weight=w.to(DEV))
    q, k = torch.cat((q, k), 1).to(DEV).split([Hq, Hkv], 1)
    cos, sin = cos.to(DEV), sin.to(DEV)
    assert not q.is_contiguous()
    want = dart.rotate_heads(q, k, cos, sin, **args)
    pad = torch.empty(B * T, Hq, D + 3, dtype=dtype, device=DEV)
    pad[..., 3:] = q
    assert all(torch.equal(x, y) for x, y in zip(dart.rotate_heads(pad[..., 3:], k, cos, sin, **args), want))
    assert torch.equal(dart.rotate_heads(q.transpose(1, 2).contiguous().transpose(1, 2), k, cos, sin, **args)[0], want[0])
    batch = [t.unflatten(0, (B, T)).transpose(1, 2) for t in (q, k)]
    whole = [t.contiguous() for t in batch]
    turned = (cos.view(B, T, 32), sin.view(B, T, 32))
    for x in (batch, whole):
        got = dart.rotate_heads(*x, *turned, **args)
        assert all(torch.equal(y.transpose(1, 2).flatten(0, 1), z) for y, z in zip(got, want))
        assert got[0].shape == x[0].shape
    positions = torch.arange(B * T, device=DEV).view(B, T)
    got = dart.rotate_heads(*batch, cos, sin, positions, **args)
    assert all(torch.equal(y.transpose(1, 2).flatten(0, 1), z) for y, z in zip(got, want))
    # angles of [1, T, half] and of [T, half] serve the whole batch, also as the first half of rows of both halves
    one = dart.rotate_heads(*batch, cos[:T], sin[:T], **args)
    both = [torch.cat((t[None, :T], t[None, :T]), -1) for t in (cos, sin)]
    for angle in ((cos[None, :T], sin[None, :T]), (both[0][..., :32], both[1][..., :32]),
                  (cos[None, :T].expand(B, -1, -1), sin[None, :T].expand(B, -1, -1))):
        assert all(torch.equal(x, y) for x, y in zip(dart.rotate_heads(*batch, *angle, **args), one))
    # a gradient that is the same for all rows
    leaf = batch[0].detach().clone().requires_grad_()
    out = dart.rotate_heads(leaf, batch[1], *turned, **args)[0]
    g = torch.randn(D, device=DEV).to(dtype)
    a = torch.autograd.grad(out, leaf, g.expand(out.shape), retain_graph=True)[0]
    assert torch.equal(a, torch.autograd.grad(out, leaf, g.expand(out.shape).contiguous())[0])


@pytest.mark.gpu
def test_without_norm_and_one_of_two():
    import dartkv_amd as dart
    q, k = (t.to(DEV) for t in inputs(11, 4, 2, 48, torch.bfloat16, 10))
    cos, sin = (t.to(DEV) for t in angles(11, 24, torch.float32, 11))
    w = torch.rand(48, device=DEV)
    plain, normed = dart.rotate_heads(q, k, cos, sin), dart.rotate_heads(q, k, cos, sin, q_weight=w, k_weight=w)
    only_k = dart.rotate_heads(q, k, cos, sin, k_weight=w)
    assert torch.equal(only_k[0], plain[0]) and torch.equal(only_k[1], normed[1])
    want, size = reference(q.double().cpu(), None, cos.double().cpu(), sin.double().cpu(), False)
    close(plain[0], want, size, 2.0 ** -18)
    leaves = [t.clone().requires_grad_() for t in (q, k, w)]
    out = dart.rotate_heads(leaves[0], leaves[1], cos, sin, k_weight=leaves[2])
    g = torch.randn_like(q)
    dq, dw = torch.autograd.grad(out, (leaves[0], leaves[2]), (g, torch.zeros_like(k)))
    dx, _, dx_size, _ = gradients(q.double().cpu(), None, cos.double().cpu(), sin.double().cpu(), False, g.double().cpu())
    close(dq, dx, dx_size, 2.0 ** -17)
    assert not dw.any()
    same = dart.rotate_heads(q, k, cos[:, :0], sin[:, :0])
    assert torch.equal(same[0], q) and torch.equal(same[1], k)


@pytest.mark.gpu
def test_positions_of_no_token_and_behind_the_table():
    import dartkv_amd as dart
    q, k = (t.to(DEV) for t in inputs(6, 3, 1, 64, torch.bfloat16, 12))
    q = q.clone()
    q[4] = float("nan")  # what padding may hold
    cos, sin = (t.to(DEV) for t in angles(8, 16, torch.float32, 13))
    w = torch.rand(64, device=DEV)
    positions = torch.tensor([0, 8, 7, -1, -5, 2 ** 31 - 1], dtype=torch.int32, device=DEV)
    for p in (positions, positions.long() * 2 ** 31):
        leaves = [t.clone().requires_grad_() for t in (q, k, w)]
        out = dart.rotate_heads(leaves[0], leaves[1], cos, sin, p, q_weight=leaves[2])
        good = [0, 2] if p is positions else [0]
        assert not out[0][[3, 4]].any() and not out[1][[3, 4]].any()
        assert bool(out[0][good].isfinite().all()) and bool(out[0][[1, 5], :, :32].isnan().all())
        assert bool(out[0][[1, 5], :, 32:].isfinite().all())
        chosen = torch.zeros(6, 1, 1, device=DEV).index_fill_(0, torch.tensor([*good, 3, 4], device=DEV), 1.0)
        grads = torch.autograd.grad(out[0], (leaves[0], leaves[2]), (chosen * torch.ones_like(out[0])).to(q.dtype))
        assert not grads[0][[3, 4]].any() and bool(grads[0][good].any())
    alone = dart.rotate_heads(q[:1], k[:1], cos, sin, positions[:1], q_weight=w)
    assert torch.equal(alone[0], dart.rotate_heads(q, k, cos, sin, positions, q_weight=w)[0][:1])


@pytest.mark.gpu
def test_rows_of_zeros_of_large_and_of_infinite_values():
    import dartkv_amd as dart
    x = torch.zeros(5, 1, 64, device=DEV)
    x[1], x[2, 0, 3], x[3, 0, 5] = 1e18, float("inf"), float("nan")
    cos, sin = (t.to(DEV) for t in angles(5, 32, torch.float32, 14))
    w = torch.ones(64, device=DEV)
    out = dart.rotate_heads(x, x, cos, sin, q_weight=w, k_weight=w)[0]
    assert not out[0].any() and bool(out[1].isfinite().all())
    assert bool(out[2, 0].isnan().any()) and bool(out[3].isnan().all()) and not out[4].any()
    norm = torch.cat((cos[1] - sin[1], cos[1] + sin[1]))  # (1e36 in the mean of squares has room in fp32)
    assert bool(((out[1, 0] - norm).abs() <= 2.0 ** -18 * 2).all())


@pytest.mark.gpu
def test_more_rows_than_a_backward_pass_has_workgroups():
    """Each workgroup goes over its rows in turns; the weights' gradient is the same every time."""
    import dartkv_amd as dart
    T, H, D = 3000, 33, 64
    q, k = (t.to(DEV) for t in inputs(T, H, 1, D, torch.bfloat16, 15))
    cos, sin = (t.to(DEV) for t in angles(T, 32, torch.float32, 16))
    w = (torch.rand(D) + 0.5).to(DEV)
    g = torch.randn(T, H, D, generator=torch.Generator().manual_seed(17)).to(torch.bfloat16)
    first = None
    for _ in range(3):
        leaves = [q.clone().requires_grad_(), w.clone().requires_grad_()]
        out = dart.rotate_heads(leaves[0], k, cos, sin, q_weight=leaves[1])
        got = torch.autograd.grad(out[0], leaves, g.to(DEV))
        first = first or got
        assert all(torch.equal(x, y) for x, y in zip(got, first))
    dx, dw, dx_size, dw_size = gradients(q.double().cpu(), w.double().cpu(), cos.double().cpu(), sin.double().cpu(), False,
                                         g.double())
    close(first[0], dx, dx_size, 2.0 ** -17)
    close(first[1], dw, dw_size, 2.0 ** -16 + 2.0 ** -17)


@pytest.mark.gpu
def test_captured_forward_and_backward():
    """The graph's gradients equal the eager ones on every replay, with eager calls between."""
    import dartkv_amd as dart
    q, k = (t.to(DEV).clone() for t in inputs(40, 4, 2, 64, torch.bfloat16, 18))
    cos, sin = (t.to(DEV) for t in angles(64, 32, torch.float32, 19))
    positions = torch.arange(40, device=DEV)
    w = torch.rand(64, device=DEV) + 0.5
    g = torch.randn_like(q)

    def step(q, k, w):
        leaves = [t.detach().requires_grad_() for t in (q, k, w)]
        out = dart.rotate_heads(leaves[0], leaves[1], cos, sin, positions, q_weight=leaves[2], k_weight=leaves[2])
        return [t.detach() for t in out] + list(torch.autograd.grad(out, leaves, (g, torch.ones_like(k))))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(q, k, w)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(q, k, w)
    for i in range(4):
        q.normal_(generator=torch.Generator(DEV).manual_seed(i))
        positions.copy_(torch.randint(-1, 64, (40,)))
        want = step(q, k, w)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.gpu
def test_a_stream_of_its_own():
    import dartkv_amd as dart
    q, k = (t.to(DEV) for t in inputs(100, 4, 2, 64, torch.bfloat16, 20))
    cos, sin = (t.to(DEV) for t in angles(100, 32, torch.float32, 21))
    want = dart.rotate_heads(q, k, cos, sin)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = dart.rotate_heads(q, k, cos, sin)
    stream.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.gpu
def test_nothing_to_do():
    import dartkv_amd as dart
    w = torch.ones(64, device=DEV, requires_grad=True)
    for shape in ((0, 4, 64), (2, 4, 0, 64), (0, 4, 3, 64)):
        q = torch.zeros(shape, device=DEV, dtype=torch.bfloat16)
        tokens = shape[:1] if len(shape) == 3 else (shape[0], shape[2])
        angle = torch.zeros(*tokens, 32, device=DEV)
        out = dart.rotate_heads(q, q[:, :2], angle, angle, q_weight=w)
        assert out[0].shape == q.shape
        assert not torch.autograd.grad(out[0].float().sum(), w)[0].any()


@pytest.mark.gpu
def test_refusals():
    import torch.autograd.forward_ad as forward
    import dartkv_amd as dart
    q = torch.zeros(4, 2, 64, dtype=torch.bfloat16, device=DEV)
    c, w, p = torch.zeros(4, 32, device=DEV), torch.ones(64, device=DEV), torch.zeros(4, dtype=torch.int32, device=DEV)
    call = dart.rotate_heads
    for error, args, kwargs in (
            (TypeError, (q.double(), q.double(), c, c), {}), (TypeError, (q, q.float(), c, c), {}),
            (ValueError, (q, q[:3], c, c), {}), (ValueError, (q[..., :60], q[..., :60], c[:, :30], c[:, :30]), {}),
            (ValueError, (q, q, c[:3], c[:3]), {}), (ValueError, (q, q, c[:1], c[:1]), {}),
            (ValueError, (q, q, c, c[:, :16]), {}), (TypeError, (q, q, c, c.half()), {}),
            (ValueError, (q[..., :48], q[..., :48], c, c), {}), (TypeError, (q, q, c, c, p.float()), {}),
            (TypeError, (q, q, c, c, [0, 1, 2, 3]), {}), (ValueError, (q, q, c, c, p[:3]), {}),
            (ValueError, (q, q, c[None], c[None], p), {}), (ValueError, (q, q, c, c), dict(q_weight=w[:32])),
            (TypeError, (q, q, c, c), dict(q_weight=w, k_weight=w.half())), (TypeError, (q, q, c, c), dict(q_weight=w.double())),
            (ValueError, (q, q, c, c), dict(eps=-1.0)), (ValueError, (q, q, c, c), dict(eps=float("nan"))),
            (RuntimeError, (q, q, c.cpu(), c), {}), (RuntimeError, (q, q, c, c), dict(k_weight=w.cpu())),
            (ValueError, (q[0], q[0], c, c), {}), (ValueError, (q[:, :0], q, c, c), {}),
            (ValueError, (q[None], q[None], c[None, :3], c[None, :3]), {})):
        for _ in range(2):
            with pytest.raises(error):
                call(*args, **kwargs)
            call(q, q, c, c, p, q_weight=w)
    leaf = c.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no gradients of cos and sin"):
        call(q, q, leaf, c)
    x = q.float().requires_grad_()
    once = torch.autograd.grad(call(x, q.float(), c, c)[0].sum(), x, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        torch.autograd.grad(once.sum(), x)
    with forward.dual_level():
        dual = forward.make_dual(q.float(), torch.ones_like(q.float()))
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(dual, q.float(), c, c)


def test_refusals_of_the_c_entries():
    from dartkv_amd import _lib
    lib = _lib.load()
    good = dict(query=256, keys=256, q_out=256, k_out=256, q_grad=256, k_grad=256, q_st=256, q_sh=64, k_st=128, k_sh=64,
                qo_st=256, qo_sh=64, ko_st=128, ko_sh=64, cos=256, sin=256, c_st=32, table_rows=9, batch=1, tokens=4, Hq=4,
                Hkv=2, D=64, half=32, dtype=2, eps=1e-6)
    for change, text in ((dict(dtype=3), "bf16"), (dict(weight_dtype=9), "weights"), (dict(D=60), "head_dim"),
                         (dict(D=264), "head_dim"), (dict(half=33), "turned"), (dict(half=-1), "turned"), (dict(Hq=0), "counts"),
                         (dict(tokens=-1), "counts"), (dict(batch=1 << 20, tokens=1 << 20), "2^31"),
                         (dict(batch=1 << 62, tokens=4), "2^31"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
                         (dict(q_st=252), "aligned"), (dict(query=264), "aligned"), (dict(c_st=33), "cos"),
                         (dict(cos=260), "cos"), (dict(query=0), "NULL"), (dict(sin=0), "NULL"),
                         (dict(positions=256, table_rows=-1), "table")):
        a = _lib.RotateHeadsArgs(**{**good, **change})
        for entry in (lib.dkv_rotate_heads, lib.dkv_rotate_heads_backward):
            assert entry(a, None) != 0 and text in lib.dkv_last_error().decode(), (change, lib.dkv_last_error())
    for change, text in ((dict(q_grad=0), "NULL"), (dict(q_weight_grad=256), "not there"),
                         (dict(q_weight=256, q_weight_grad=256), "workspace")):
        a = _lib.RotateHeadsArgs(**{**good, **change})
        assert lib.dkv_rotate_heads_backward(a, None) != 0 and text in lib.dkv_last_error().decode()
    for entry in (lib.dkv_rotate_heads, lib.dkv_rotate_heads_backward):
        assert entry(None, None) == 1
        assert entry(_lib.RotateHeadsArgs(**{**good, "tokens": 0}), None) == 0  # nothing to do, nothing launched
    assert lib.dkv_rotate_heads_backward_workspace_bytes(_lib.RotateHeadsArgs(**good)) == (1 + 1) * 64 * 4
    assert lib.dkv_rotate_heads_backward_workspace_bytes(_lib.RotateHeadsArgs(**{**good, "tokens": 1 << 20})) == 2048 * 64 * 4


def test_operators_want_the_gpu():
    import dartkv_amd as dart
    q = torch.zeros(4, 2, 64)
    with pytest.raises(RuntimeError, match="ROCm"):
        dart.rotate_heads(q, q, q[:, 0, :32], q[:, 0, :32])
