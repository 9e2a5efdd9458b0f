"""Calls of several threads: what one thread's launches leave for each other belongs to that thread."""

from __future__ import annotations

import gc
import threading
import weakref

import pytest
import torch

import dartkv_amd as dart
from dartkv_amd import attention

CPU = torch.device("cpu")


@pytest.fixture
def no_capture(monkeypatch):
    """Workspaces without a GPU: nothing is being captured."""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    attention.release_workspaces()
    yield
    attention.release_workspaces()


def _in_thread(f):
    """f() in a thread that lives until the returned function is called, and its result."""
    out, done, stop = [], threading.Event(), threading.Event()

    def body():
        try:
            out.append(f())
        finally:
            done.set()
            stop.wait(30)

    thread = threading.Thread(target=body, daemon=True)
    thread.start()
    assert done.wait(30)

    def end():
        stop.set()
        thread.join(30)

    return out[0], end


def test_threads_of_one_stream_have_workspaces_of_their_own(no_capture):
    """A call's launches pass records through its workspace, and another thread's launches may come between them."""
    mine = attention._workspace(CPU, 1 << 12, 7)
    assert attention._workspace(CPU, 1 << 12, 7) is mine
    other, end = _in_thread(lambda: attention._workspace(CPU, 1 << 12, 7))
    end()
    assert other.data_ptr() != mine.data_ptr()
    assert attention._workspace(CPU, 1 << 12, 7) is mine


def test_another_threads_streams_do_not_displace_a_workspace(no_capture):
    mine = attention._workspace(CPU, 256, 0)
    _, end = _in_thread(lambda: [attention._workspace(CPU, 256, s) for s in range(1, 40)])
    end()
    assert attention._workspace(CPU, 256, 0) is mine
    for s in range(1, 40):
        attention._workspace(CPU, 256, s)
    assert attention._workspace(CPU, 256, 0) is not mine


def test_released_workspaces_are_those_of_all_threads(no_capture):
    mine = weakref.ref(attention._workspace(CPU, 256, 0))
    other, end = _in_thread(lambda: weakref.ref(attention._workspace(CPU, 256, 0)))
    try:
        assert mine() is not None and other() is not None
        attention.release_workspaces()
        gc.collect()
        assert mine() is None and other() is None
    finally:
        end()


def test_a_thread_that_ends_keeps_no_workspace(no_capture):
    other, end = _in_thread(lambda: weakref.ref(attention._workspace(CPU, 256, 0)))
    assert other() is not None
    end()
    gc.collect()
    assert other() is None


@pytest.mark.gpu
def test_calls_of_three_threads_on_one_stream_give_what_they_give_alone():
    """Log probabilities whose parts are joined by a second launch, the weights' gradients of a rotation, forks and
    compactions of tables that one workgroup does not do alone: sums and tables have one order, so results are equal."""
    torch.manual_seed(0)
    dev = "cuda"
    logits = torch.randn(9, 151_936, device=dev, dtype=torch.bfloat16)
    tokens = torch.randint(0, 151_936, (9,), device=dev)
    q = torch.randn(700, 6, 64, device=dev, dtype=torch.bfloat16)
    k, cos, sin = q[:, 4:].contiguous(), torch.rand(700, 32, device=dev), torch.rand(700, 32, device=dev)
    weight, g = torch.rand(64, device=dev) + 0.5, torch.randn(700, 6, 64, device=dev, dtype=torch.bfloat16)
    sources = torch.arange(256, device=dev, dtype=torch.int32) // 8 * 8
    more = torch.full((256,), 3, device=dev, dtype=torch.int32)

    def probabilities():
        return tuple(dart.token_logprobs(logits, tokens, top=20))

    def rotation():
        w = weight.clone().requires_grad_()
        a, b = dart.rotate_heads(q, k, cos, sin, q_weight=w, k_weight=w)
        return torch.autograd.grad((a, b), w, (g, g[:, 4:]))

    def tables():
        cache = dart.BlockKVCache(256, 20_000, 1, 16, block_size=16, max_blocks=80, sharing=True, device=dev)
        prompts = torch.full((256,), 1000, device=dev, dtype=torch.int32)
        prompts[1::2] = 5
        cache.reserve(prompts, int(128 * 1005))
        cache.fork(sources)
        cache.reserve(more, 768)
        cache.release(more)
        cache.compact()
        return cache.table, cache.lengths, cache.free, cache.state, cache.shares

    jobs = (probabilities, rotation, tables)
    alone = [[t.clone() for t in job()] for job in jobs]
    torch.cuda.synchronize()
    results, errors, gate = [[] for _ in jobs], [], threading.Barrier(len(jobs))

    def run(i):
        try:
            gate.wait(30)
            for _ in range(20):
                results[i].append(jobs[i]())
        except Exception as e:  # (for the test's own thread)
            errors.append(e)

    threads = [threading.Thread(target=run, args=(i,), daemon=True) for i in range(len(jobs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not errors and [len(r) for r in results] == [20] * len(jobs)
    torch.cuda.synchronize()
    for want, got in zip(alone, results):
        for once in got:
            assert all(torch.equal(a, b) for a, b in zip(want, once))
