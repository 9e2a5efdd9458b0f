"""More rows than one launch has room for: a launch holds fewer than 2^32 threads."""

from __future__ import annotations

import math

import pytest
import torch

import dartkv_amd as dart
from dartkv_amd import _lib

DEV = "cuda"
ROTATE = dict(query=256, keys=256, q_out=256, k_out=256, q_st=320, q_sh=80, k_st=160, k_sh=80, qo_st=320, qo_sh=80, ko_st=160,
              ko_sh=80, cos=256, sin=256, c_st=5, table_rows=9, batch=1, Hq=4, Hkv=2, D=80, half=5, dtype=2, eps=1e-6)


def test_rotations_of_more_rows_than_a_launch_holds_are_refused():
    """Odd counts of angles: a row for each wave, two steps, so 8 rows a workgroup: 2^24 of them for 2^27 rows."""
    lib = _lib.load()
    for tokens in (1 << 25, (1 << 27) // 6 + 8):
        assert lib.dkv_rotate_heads(_lib.RotateHeadsArgs(**ROTATE, tokens=tokens), None) == 1
        assert "rows" in lib.dkv_last_error().decode()


def test_appends_of_more_tokens_than_a_launch_holds_are_refused():
    lib = _lib.load()
    append = dict(keys=256, values=256, k_st=32, k_sh=16, v_st=32, v_sh=16, slots=256, key_codes=256, value_codes=256,
                  key_scale=256, value_scale=256, tokens=1 << 30, H=4, D=16, blocks=1, block_size=16, dtype=2)
    assert lib.dkv_append_blocks(_lib.AppendBlocksArgs(**append), None) == 1
    assert "too many tokens" in lib.dkv_last_error().decode()
    # 2^29 rows of queries of 256, 32 a workgroup, beside the append
    append = {**append, "tokens": 1 << 19, "D": 256, "k_st": 1024, "k_sh": 256, "v_st": 1024, "v_sh": 256}
    rotate = {**ROTATE, "D": 256, "half": 128, "c_st": 128, "Hq": 1024, "Hkv": 4, "positions": 256, "q_st": 1 << 18, "q_sh": 256,
              "qo_st": 1 << 18, "qo_sh": 256, "tokens": 1 << 19}
    assert lib.dkv_append_rotated_blocks(_lib.AppendBlocksArgs(**append), _lib.RotateHeadsArgs(**rotate), None) == 1
    assert "too many tokens" in lib.dkv_last_error().decode()


def test_copies_of_more_heads_than_a_launch_holds_are_refused():
    lib = _lib.load()
    a = _lib.CopyBlocksArgs(copies=256, count=1, layers=1 << 10, blocks=1, H=1 << 18, block_size=256, D=512, key_codes=256,
                            value_codes=256, key_scale=256, value_scale=256)
    assert lib.dkv_copy_blocks(a, None) == 1 and "too many layers" in lib.dkv_last_error().decode()


@pytest.mark.gpu
def test_gradients_of_more_rows_than_a_launch_holds():
    """2^24 + 3 rows of two logits: in 64 bits log p of the larger is -log1p(e^-d), H = log1p(e^-d) + d / (1 + e^d)."""
    rows = (1 << 24) + 3
    x = torch.empty(rows, 2, dtype=torch.float32, device=DEV)
    x[:, 0] = torch.arange(rows, device=DEV) % 8191 / 512.0 - 8
    x[:, 1] = 1
    tokens = torch.arange(rows, device=DEV, dtype=torch.int32) % 2
    leaf = x.requires_grad_()
    out = dart.token_logprobs(leaf, tokens, top=1)
    grad = torch.autograd.grad((out.logprobs, out.entropy), leaf, (torch.ones(rows, device=DEV), 2 * torch.ones(rows, device=DEV)))[0]
    index = torch.arange(rows, device=DEV)
    for part in index.split(1 << 22):
        p = torch.softmax(x.detach()[part].double(), -1)
        logp = p.log()
        entropy = -(p * logp).sum(-1, keepdim=True)
        want = -p * (1 + 2 * (logp + entropy)) + torch.nn.functional.one_hot(tokens[part].long(), 2)
        got = logp.gather(1, tokens[part, None].long()).squeeze(1)
        # (two terms: each off by 2^-22 (|z| + 2) with |z| <= 25; the formula's products as much again)
        assert bool(((out.logprobs[part].double() - got).abs() <= 2.0 ** -17).all())
        assert bool(((out.entropy[part].double() - entropy.squeeze(1)).abs() <= 2.0 ** -16).all())
        assert bool(((grad[part].double() - want).abs() <= 2.0 ** -14).all())
        first = x.detach()[part].argmax(-1)
        assert torch.equal(out.top_tokens[part].squeeze(1), first)


@pytest.mark.gpu
def test_more_rows_than_a_forward_launch_holds():
    rows = (1 << 26) + 5
    x = torch.zeros(rows, 2, dtype=torch.bfloat16, device=DEV)
    x[:, 1] = torch.arange(rows, device=DEV) % 3
    tokens = torch.ones(rows, device=DEV, dtype=torch.int32)
    tokens[-1] = -1
    out = dart.token_logprobs(x, tokens)
    want = torch.tensor([-math.log1p(math.exp(-d)) for d in range(3)], device=DEV)[torch.arange(rows, device=DEV) % 3]
    want[-1] = 0
    assert bool(((out.logprobs - want).abs() <= 2.0 ** -20).all())  # (at most 0.7, two terms)
    assert bool((out.entropy > 0.3).all())
