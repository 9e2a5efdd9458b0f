"""prompt_attention against attention in 64 bits (GPU), and its refusals (CPU).

Tolerance.  Both inputs' products are exact in fp32 and sums are fp32 (errors of 2^-24 relative each, far below
what follows).  The weights p in [0, 2^8] are rounded to the type (half a step u = eps / 2 relative each), so a
weighted sum moves by at most u * sum(p |v|) / sum(p); the result is rounded once, u * |o|.  So
|error| <= u * (W + |o|), W = sum(p |v|) / sum(p).  One per cent of slack (2e-5 W for bf16, 5e-6 W for fp16) covers
the fp32 sums (2^-24 relative per term, of random sign) and the exponentials' last bits (2^-22 relative each).
"""

from __future__ import annotations

import math

import pytest
import torch

DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16]


def _reference(q, k, v, causal, scale):
    """(o, W) of one sequence, q [nq, Hq, D], k and v [nk, Hkv, D], in 64 bits; a hidden key takes no part."""
    nq, Hq, D = q.shape
    nk, Hkv = k.shape[:2]
    q, k, v = (t.double().cpu().transpose(0, 1) for t in (q, k, v))
    o = torch.zeros(Hq, nq, D, dtype=torch.float64)
    w = torch.zeros(Hq, nq, D, dtype=torch.float64)
    for h in range(Hq):
        kh, vh = k[h // (Hq // Hkv)], v[h // (Hq // Hkv)]
        s = (q[h] @ kh.t()) * scale
        for i in range(nq):
            n = min(nk, max(0, i + 1 + nk - nq)) if causal else nk
            if n == 0:
                continue
            p = torch.softmax(s[i, :n], 0)
            o[h, i] = p @ vh[:n]
            w[h, i] = p @ vh[:n].abs()
    return o.transpose(0, 1), w.transpose(0, 1)


def _check(got, o, w, dtype):
    u = torch.finfo(dtype).eps / 2
    err = (got.double().cpu() - o).abs()
    bound = 1.01 * u * (w + o.abs()) + 1e-6 * w + torch.finfo(dtype).tiny
    worst = float((err / bound).max()) if err.numel() else 0.0
    assert worst <= 1.0, f"error is {worst:.3f} of its bound"


def _rand(shape, dtype, seed, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=gen) * scale).to(dtype).to(DEV)


def _starts(lengths):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device=DEV)


def _packed_check(got, q, k, v, qn, kn, causal, scale, dtype):
    qa = ka = 0
    for nq, nk in zip(qn, kn):
        o, w = _reference(q[qa:qa + nq], k[ka:ka + nk], v[ka:ka + nk], causal, scale)
        _check(got[qa:qa + nq], o, w, dtype)
        qa, ka = qa + nq, ka + nk


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [8, 40, 64, 80, 96, 128, 136, 192, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_head_dims(dtype, D, causal):
    import dartkv_amd as dart
    lengths = [1, 63, 130]
    q, k, v = (_rand((sum(lengths), h, D), dtype, 10 * D + i) for i, h in enumerate((4, 2, 2)))
    got = dart.prompt_attention(q, k, v, _starts(lengths), causal=causal)
    _packed_check(got, q, k, v, lengths, lengths, causal, 1 / math.sqrt(D), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (3, 1), (8, 8), (12, 2), (16, 1), (40, 1)])
def test_head_layouts(Hq, Hkv):
    import dartkv_amd as dart
    lengths = [5, 0, 200, 64, 65, 0]
    q, k, v = (_rand((sum(lengths), h, 64), torch.bfloat16, 7 + i) for i, h in enumerate((Hq, Hkv, Hkv)))
    got = dart.prompt_attention(q, k, v, _starts(lengths))
    _packed_check(got, q, k, v, lengths, lengths, True, 0.125, torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_more_and_fewer_keys_than_queries(dtype, causal):
    """Keys of an earlier part, none at all, and fewer keys than queries (rows that see nothing are 0)."""
    import dartkv_amd as dart
    qn, kn = [3, 70, 10, 1, 130, 64], [300, 70, 0, 129, 40, 64]
    q = _rand((sum(qn), 6, 128), dtype, 1)
    k, v = _rand((sum(kn), 2, 128), dtype, 2), _rand((sum(kn), 2, 128), dtype, 3)
    got = dart.prompt_attention(q, k, v, _starts(qn), _starts(kn), causal=causal, scale=0.2)
    _packed_check(got, q, k, v, qn, kn, causal, 0.2, dtype)
    assert bool((got[73:83] == 0).all())
    if causal:
        assert bool((got[84:84 + 90] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["heads_first", "tokens_first", "wide", "shared_keys", "unaligned", "odd_last"])
def test_batch_and_strides(layout):
    import dartkv_amd as dart
    B, Hq, Hkv, Q, T, D = 2, 4, 2, 67, 90, 64
    dtype = torch.bfloat16
    if layout == "tokens_first":
        q, k, v = (_rand((B, n, h, D), dtype, n + h).transpose(1, 2) for n, h in ((Q, Hq), (T, Hkv), (T, Hkv)))
    elif layout == "wide":  # slices of a joint projection
        x = _rand((B, T, Hq + 2 * Hkv, D), dtype, 5)
        q, k, v = (t.transpose(1, 2) for t in (x[:, :Q, :Hq], x[:, :, Hq:Hq + Hkv], x[:, :, Hq + Hkv:]))
    elif layout == "shared_keys":  # one sequence's keys for the whole batch
        q = _rand((B, Hq, Q, D), dtype, 1)
        k, v = (_rand((1, Hkv, T, D), dtype, s).expand(B, -1, -1, -1) for s in (2, 3))
    elif layout == "unaligned":
        q, k, v = (_rand((B, h, n, D + 3), dtype, h + n)[..., 3:] for h, n in ((Hq, Q), (Hkv, T), (Hkv, T)))
    elif layout == "odd_last":
        q, k, v = (_rand((B, h, D, n), dtype, h + n).transpose(2, 3) for h, n in ((Hq, Q), (Hkv, T), (Hkv, T)))
    else:
        q, k, v = (_rand((B, h, n, D), dtype, h + n) for h, n in ((Hq, Q), (Hkv, T), (Hkv, T)))
    got = dart.prompt_attention(q, k, v)
    assert got.shape == q.shape and got.dtype == dtype
    for b in range(B):
        o, w = _reference(*(t[b].transpose(0, 1) for t in (q, k, v)), True, 0.125)
        _check(got[b].transpose(0, 1), o, w, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_large_and_small_logits(dtype):
    """Logits whose running maximum rises from tile to tile, and rows where one key takes all."""
    import dartkv_amd as dart
    n, D = 400, 64
    q, k, v = _rand((n, 2, D), dtype, 1, 4.0), _rand((n, 1, D), dtype, 2, 4.0), _rand((n, 1, D), dtype, 3)
    k *= torch.linspace(0.01, 4, n, device=DEV)[:, None, None].to(dtype)
    got = dart.prompt_attention(q, k, v, _starts([n]))
    # The logits' own fp32 sums matter here: with sum |q k| scale about 325 a logit is off by at most 64 * 2^-24 * 325
    # = 1.2e-3 = d, so weights and their sum by e^d each: |error| grows by (e^2d - 1) W < 2^-8 W.
    o, w = _reference(q, k, v, True, 0.125)
    u = torch.finfo(dtype).eps / 2
    err = (got.double().cpu() - o).abs()
    assert bool((err <= 1.01 * u * (w + o.abs()) + 2 ** -8 * w).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,lengths", [(64, [70, 5, 200]), (128, [300, 1]), (256, [100, 40])])
@pytest.mark.parametrize("causal", [True, False])
def test_keys_that_a_row_does_not_see_do_not_reach_it(dtype, D, lengths, causal):
    """Infinities and NaN among keys and values: rows before them are as without them, rows behind them show them."""
    import dartkv_amd as dart
    n = sum(lengths)
    q, k, v = (_rand((n, h, D), dtype, D + h) for h in (4, 2, 2))
    inf = float("inf")
    for t, h, ch, x in ((3, 0, 1, inf), (3, 1, 2, -inf), (66, 0, 5, float("nan")), (69, 1, 7, inf), (69, 1, 7, inf),
                        (n - 2, 0, D - 1, -inf), (n - 1, 0, D - 1, inf), (n - 1, 1, 0, float("nan"))):
        v[t, h, ch] = x
    k[n - 3, 1, 4] = float("nan")
    got = dart.prompt_attention(q, k, v, _starts(lengths), causal=causal).double().cpu()
    at = 0
    for m in lengths:
        part = slice(at, at + m)
        o, w = _reference(q[part], k[part], v[part], causal, 1 / math.sqrt(D))
        fine = torch.isfinite(o)
        assert torch.equal(torch.isnan(got[part]), torch.isnan(o))
        assert torch.equal(got[part][~fine & ~torch.isnan(o)], o[~fine & ~torch.isnan(o)])
        _check(got[part][fine], o[fine], w[fine], dtype)
        at += m


@pytest.mark.gpu
def test_long_sequence_against_64_bits():
    """Many tiles with eight waves a workgroup: rows of the beginning, the middle and the end."""
    import dartkv_amd as dart
    n, Hq, Hkv, D = 9003, 32, 8, 128
    q, k, v = (_rand((n, h, D), torch.bfloat16, h + i) for i, h in enumerate((Hq, Hkv, Hkv)))
    got = dart.prompt_attention(q, k, v, _starts([n]))
    for i in (0, 1, 63, 64, 1000, 2047, 2500, 4095, 5002, 8191, 9002):
        s = torch.einsum("hgd,jhd->hgj", q[i].double().cpu().view(Hkv, 4, D), k[:i + 1].double().cpu()) / math.sqrt(D)
        p = torch.softmax(s, -1)
        o = torch.einsum("hgj,jhd->hgd", p, v[:i + 1].double().cpu()).reshape(Hq, D)
        w = torch.einsum("hgj,jhd->hgd", p, v[:i + 1].double().cpu().abs()).reshape(Hq, D)
        _check(got[i], o, w, torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("qn,kn", [([3], [5000]), ([40, 1, 17], [2000, 700, 3001]), ([130], [1030])])
def test_few_queries_over_many_keys(dtype, D, qn, kn):
    """The keys come in parts that are joined; infinities in one part, and a part that some rows see nothing of."""
    import dartkv_amd as dart
    q = _rand((sum(qn), 4, D), dtype, 1)
    k, v = _rand((sum(kn), 2, D), dtype, 2), _rand((sum(kn), 2, D), dtype, 3)
    got = dart.prompt_attention(q, k, v, _starts(qn), _starts(kn))
    _packed_check(got, q, k, v, qn, kn, True, 1 / math.sqrt(D), dtype)
    v[5, 0, 3] = float("inf")
    again = dart.prompt_attention(q, k, v, _starts(qn), _starts(kn))
    hit = torch.zeros(q.shape, dtype=torch.bool, device=DEV)
    hit[max(0, 5 - kn[0] + qn[0]):qn[0], :2, 3] = True
    assert bool((again[hit] == float("inf")).all()) and torch.equal(again[~hit], got[~hit])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,Hkv,G,Q,T,D", [(3, 4, 4, 333, 333, 128), (2, 8, 4, 500, 500, 96), (1, 16, 1, 1300, 1300, 128),
                                           (1, 8, 4, 501, 903, 72), (1, 4, 4, 999, 901, 128)])
def test_batches_of_about_one_workgroup_a_cu(dtype, B, Hkv, G, Q, T, D):
    """128 to 256 tiles of 128 rows, odd and even counts of them for each sequence, head_dims that are not powers of two."""
    import dartkv_amd as dart
    q, k, v = (_rand((B, h, n, D), dtype, h + n) for h, n in ((Hkv * G, Q), (Hkv, T), (Hkv, T)))
    got = dart.prompt_attention(q, k, v)
    for b in range(B):
        o, w = _reference(*(t[b].transpose(0, 1) for t in (q, k, v)), True, 1 / math.sqrt(D))
        _check(got[b].transpose(0, 1), o, w, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("qn,kn", [([1, 0, 300, 77, 129], None), ([200, 130, 200], [200, 401, 160]), ([507], None)])
def test_packed_of_about_one_workgroup_a_cu(qn, kn):
    import dartkv_amd as dart
    kn = kn or qn
    dtype = torch.bfloat16
    q = _rand((sum(qn) + 70, 32, 128), dtype, 1)
    k, v = _rand((sum(kn) + 70, 8, 128), dtype, 2), _rand((sum(kn) + 70, 8, 128), dtype, 3)
    k[sum(kn):], v[sum(kn):] = float("nan"), float("nan")
    got = dart.prompt_attention(q, k, v, _starts(qn), _starts(kn))
    _packed_check(got, q, k, v, qn, kn, True, 1 / math.sqrt(128), dtype)
    assert bool((got[sum(qn):] == 0).all())


@pytest.mark.gpu
def test_out_and_rows_behind_the_last_sequence():
    import dartkv_amd as dart
    q, k, v = (_rand((90, h, 64), torch.bfloat16, h) for h in (4, 2, 2))
    starts = _starts([30, 40])
    got = dart.prompt_attention(q, k, v, starts)
    assert bool((got[70:] == 0).all())
    out = torch.full((90, 4, 96), 7.0, dtype=torch.bfloat16, device=DEV)
    assert dart.prompt_attention(q, k, v, starts, out=out[..., :64]).data_ptr() == out.data_ptr()
    assert torch.equal(out[:70, :, :64], got[:70]) and bool((out[70:] == 7).all()) and bool((out[..., 64:] == 7).all())
    assert dart.prompt_attention(q[:0], k[:0], v[:0], _starts([0])).shape == (0, 4, 64)


@pytest.mark.gpu
def test_starts_outside_the_tensors_are_clamped():
    import dartkv_amd as dart
    q, k, v = (_rand((50, 2, 64), torch.bfloat16, s) for s in (1, 2, 3))
    got = dart.prompt_attention(q, k, v, torch.tensor([0, 20, 500], device=DEV))
    want = dart.prompt_attention(q, k, v, torch.tensor([0, 20, 50], device=DEV))
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_replayed_graph_and_other_stream():
    import dartkv_amd as dart
    q, k, v = (_rand((300, h, 128), torch.bfloat16, h) for h in (8, 2, 2))
    starts = _starts([100, 150])
    want = dart.prompt_attention(q, k, v, starts)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = dart.prompt_attention(q, k, v, starts)
    torch.cuda.synchronize()
    assert torch.equal(again, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = dart.prompt_attention(q, k, v, starts)
    for lengths in ([100, 150], [1, 249], [300, 0], [0, 17]):
        starts.copy_(_starts(lengths))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, dart.prompt_attention(q, k, v, starts)), lengths


@pytest.mark.gpu
@pytest.mark.parametrize("change,error", [
    (dict(dtype=torch.float32), TypeError), (dict(kdtype=torch.float16), TypeError), (dict(D=60), ValueError),
    (dict(D=264), ValueError), (dict(Hq=5), ValueError), (dict(scale=0.0), ValueError),
    (dict(scale=float("inf")), ValueError), (dict(grad=True), RuntimeError), (dict(starts=[0]), ValueError),
    (dict(float_starts=True), TypeError), (dict(key_starts=[0, 1, 2]), ValueError), (dict(flat=True), ValueError),
])
def test_refusals(change, error):
    import dartkv_amd as dart
    D, Hq = change.get("D", 64), change.get("Hq", 4)
    q = torch.zeros(10, Hq, D, dtype=change.get("dtype", torch.bfloat16), device=DEV)
    k = torch.zeros(10, 2, D, dtype=change.get("kdtype", change.get("dtype", torch.bfloat16)), device=DEV)
    starts = torch.tensor(change.get("starts", [0, 10]), device=DEV)
    if change.get("float_starts"):
        starts = starts.float()
    if change.get("grad"):
        q.requires_grad_()
    more = torch.tensor(change["key_starts"], device=DEV) if "key_starts" in change else None
    with pytest.raises(error):
        if change.get("flat"):
            dart.prompt_attention(q, k, k)
        else:
            dart.prompt_attention(q, k, k, starts, more, scale=change.get("scale"))
    with torch.no_grad():
        dart.prompt_attention(torch.zeros(1, 1, 8, 64, dtype=torch.float16, device=DEV, requires_grad=True),
                              *[torch.zeros(1, 1, 8, 64, dtype=torch.float16, device=DEV)] * 2)


def test_cpu_tensors_are_refused():
    import dartkv_amd as dart
    x = torch.zeros(1, 2, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        dart.prompt_attention(x, x, x)


@pytest.mark.parametrize("field,value,code,text", [
    ("dtype", 0, 3, "bf16 or fp16"), ("Hq", 5, 1, "divisible"), ("D", 12, 1, "multiple of 8"), ("D", 264, 1, "256"),
    ("requests", 0, 1, "counts"), ("q_starts", 64, 1, "together"), ("q_tokens", 1 << 31, 1, "too many"),
    ("scale", 0.0, 1, "scale"), ("scale", float("nan"), 1, "scale"), ("query", None, 1, "NULL"),
    ("keys", 8, 1, "aligned"), ("q_st", 4, 1, "aligned"), ("o_sh", 2, 1, "aligned"), ("k_st", 1 << 23, 1, "strides"),
])
def test_c_entry_refuses_on_the_host(field, value, code, text):
    """Bad arguments return an error before anything is launched (no GPU)."""
    from dartkv_amd import _lib
    a = _lib.PromptAttentionArgs(query=256, keys=256, values=256, out=256, requests=1, Hq=4, Hkv=2, D=64, q_tokens=8,
                                 k_tokens=8, dtype=2, scale=0.125, causal=1)
    for n in "qkvo":
        setattr(a, n + "_st", 256), setattr(a, n + "_sh", 64)
    setattr(a, field, value)
    lib = _lib.load()
    assert lib.dkv_prompt_attention(a, None) == code
    assert text in lib.dkv_last_error().decode()
    assert lib.dkv_prompt_attention(None, None) == 1
