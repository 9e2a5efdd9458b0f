"""prompt_attention where its types' ranges and its parts show, against 64 bits.

Bounds are test_prompt_attention's, u (W + |o|) with u half a step of the type, and what is said at each test.
"""

from __future__ import annotations

import math

import pytest
import torch

from tests.test_prompt_attention import _check, _packed_check, _rand, _reference, _starts

DEV = "cuda"


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("drop", [12.5, 20.5, 26.5])
def test_small_weights_beside_one_dominant_key_in_fp16(D, causal, drop):
    """One key whose value is 0 has all the weight but 2^-drop for each other key, and the result is theirs alone.

    The kernel rounds 2^7 p to fp16, p = 2^(s - m) with m at most 8 under the row's maximum, so p of the dominant key is at
    least 1, as is the sum of weights.  2^7 p is normal from 2^-14 on (p from 2^-21): half a step u relative.  Under that
    the step is 2^-24, so p is off by at most 2^-32: |error| <= u (W + |o|) + 2^-32 sum |v|.
    """
    import dartkv_amd as dart
    n = 700
    q = torch.zeros(n, 2, D)
    q[..., 0] = 1.0
    k = torch.zeros(n, 1, D)
    k[0, 0, 0] = drop
    v = (torch.randn(n, 1, D, generator=torch.Generator().manual_seed(D)) + 2) * 1000
    v[0] = 0.0
    q, k, v = (t.half().to(DEV) for t in (q, k, v))
    got = dart.prompt_attention(q, k, v, _starts([n]), causal=causal, scale=math.log(2.0))
    o, w = _reference(q, k, v, causal, math.log(2.0))
    u = torch.finfo(torch.float16).eps / 2
    bound = 1.01 * u * (w + o.abs()) + 1e-6 * w
    # the result's own rounding, where it is subnormal in fp16
    bound = bound + 2.0 ** -25
    if drop > 21:
        bound = bound + 2.0 ** -32 * v.double().abs().sum(0).cpu()
    err = (got.double().cpu() - o).abs()
    assert bool((err <= bound).all()), f"error is {float((err / bound).max()):.3f} of its bound"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,drop", [(torch.bfloat16, 140.0), (torch.float16, 60.0)])
@pytest.mark.parametrize("n", [40, 300])
def test_an_infinite_value_under_a_small_weight(dtype, drop, n):
    """Without the causal mask every row sees every key: a positive weight times an infinity is one, however small."""
    import dartkv_amd as dart
    q, k, v = (_rand((n, h, 64), dtype, h, 0.5) for h in (4, 2, 2))
    q[..., 0], k[..., 0] = 1.0, 0.0
    k[17, 0, 0] = -drop
    v[17, 0, 3], v[17, 0, 9] = float("inf"), float("-inf")
    got = dart.prompt_attention(q, k, v, _starts([n]), causal=False, scale=math.log(2.0)).double().cpu()
    assert bool((got[:, :2, 3] == math.inf).all()) and bool((got[:, :2, 9] == -math.inf).all())
    v[17, 0, 3], v[17, 0, 9] = 0.0, 0.0
    o, w = _reference(q, k, v, False, math.log(2.0))
    got[:, :2, 3], got[:, :2, 9] = o[:, :2, 3], o[:, :2, 9]
    _check(got, o, w, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128, 256])
def test_large_values_in_a_part_without_weight(D):
    """The keys come in parts; some parts' values are large and their weights 2^-400 of the dominant key's: they
    add nothing, an infinity among them apart."""
    import dartkv_amd as dart
    nq, nk = 3, 5000
    q, k, v = _rand((nq, 4, D), torch.bfloat16, 1, 0.1), _rand((nk, 2, D), torch.bfloat16, 2), _rand((nk, 2, D), torch.bfloat16, 3)
    q[..., 0] = 1.0
    k[..., 0] = 0.0
    k[:2048, :, 0] = -300.0
    v[:2048] = 1e34
    k[4800, :, 0] = 100.0
    got = dart.prompt_attention(q, k, v, _starts([nq]), _starts([nk]), scale=math.log(2.0))
    o, w = _reference(q, k, v, True, math.log(2.0))
    _check(got, o, w, torch.bfloat16)
    v[5, 0, 3] = float("inf")  # in the first part, which the last one outweighs
    again = dart.prompt_attention(q, k, v, _starts([nq]), _starts([nk]), scale=math.log(2.0))
    assert bool((again[:, :2, 3] == math.inf).all())
    again[:, :2, 3] = got[:, :2, 3]
    assert torch.equal(again, got)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("first,lengths,behind", [(10, [30, 40], 20), (200, [1], 0), (1, [300, 0, 77], 130), (64, [0], 0),
                                                  (7, [1200], 3)])
def test_rows_before_the_first_sequence(D, first, lengths, behind):
    """0 in a new tensor like the rows behind the last, untouched in a given one."""
    import dartkv_amd as dart
    total = first + sum(lengths) + behind
    q, k, v = (_rand((total, h, D), torch.bfloat16, h) for h in (4, 2, 2))
    starts = _starts(lengths) + first
    held = torch.full_like(q, float("nan"))
    del held  # (what a new tensor is likely to hold)
    got = dart.prompt_attention(q, k, v, starts)
    real = slice(first, first + sum(lengths))
    assert bool((got[:first] == 0).all()) and bool((got[real.stop:] == 0).all())
    _packed_check(got[real], q[real], k[real], v[real], lengths, lengths, True, 1 / math.sqrt(D), torch.bfloat16)
    out = torch.full((total, 4, D), 7.0, dtype=torch.bfloat16, device=DEV)
    dart.prompt_attention(q, k, v, starts, out=out)
    assert torch.equal(out[real], got[real]) and bool((out[:first] == 7).all()) and bool((out[real.stop:] == 7).all())


@pytest.mark.gpu
@pytest.mark.parametrize("many", [False, True])
def test_rows_before_the_first_request_of_a_block_cache(many):
    import dartkv_amd as dart
    from tests.test_blocks import _cache, _check_attention, _query
    new, lengths, first, behind = ([70, 1, 33] if many else [2, 1, 3]), [100, 300, 40], 5, 4
    cache = _cache(lengths, 2, 64, 32, 7)
    total = first + sum(new) + behind
    q = _query(total, 4, 64, torch.bfloat16, 7)
    held = torch.full_like(q, float("nan"))
    del held
    got = dart.block_attention(q, *cache, _starts(new) + first, max_tokens=None if many else 3)
    real = slice(first, first + sum(new))
    assert bool((got[:first] == 0).all()) and bool((got[real.stop:] == 0).all())
    _check_attention(got[real], q[real], cache, new, torch.bfloat16, chunk=many)
    out = torch.full((total, 4, 64), 7.0, dtype=torch.bfloat16, device=DEV)
    dart.block_attention(q, *cache, _starts(new) + first, max_tokens=None if many else 3, out=out)
    assert torch.equal(out[real], got[real]) and bool((out[:first] == 7).all()) and bool((out[real.stop:] == 7).all())
