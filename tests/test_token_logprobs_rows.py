"""token_logprobs: what the tests of its values do not reach."""

from __future__ import annotations

import math

import pytest
import torch

import dartkv_amd as dart

from tests.test_token_logprobs import DEV, expected, rows


@pytest.mark.gpu
@pytest.mark.parametrize("T", [3, 700, 2100])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_moments_are_a_reference_and_its_sum(T, dtype):
    """m + ln(2) log2 s is the row's log of the sum of e^x, wherever its maximum lies: s as in expected(), log2 s (at most
    17 + 16) and its product off by 2^-22 of theirs, m exact, one rounding of none of them on the host."""
    x, tokens = rows(T, 20_011, dtype, 40)
    x[0] = 0
    x[0, -1] = 7  # (under what raises the reference by itself)
    x[1] += torch.linspace(0, 60, 20_011).to(dtype)
    moments = dart.torch_ops.token_logprobs(x.to(DEV), tokens.to(DEV), 2)[4].double().cpu()
    x = x.double()
    _, _, _, _, e = expected(x, tokens)
    got = moments[:, 0] + math.log(2) * moments[:, 1]
    assert bool(((got - x.logsumexp(-1)).abs() <= e + 2.0 ** -22 * moments[:, 1].abs()).all())
    assert bool((moments[:, 0] <= x.amax(-1)).all())
