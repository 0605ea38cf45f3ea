"""Compiled models that the collector finds while a graph is captured elsewhere in the process."""

from __future__ import annotations

import gc
import threading

import pytest
import torch

import mlc
from mlc import ops
from mlc.runtime import hip_runtime
from test_decoder_operators import Step, step_inputs

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("where", ("another thread", "another stream"))
def test_a_compiled_step_that_is_collected_beside_a_capture(where):
    """The thread that frees its memory captures nothing itself, or not on its current stream."""
    model, args = Step().cuda(), step_inputs(tokens=3)
    held = [mlc.compile(model, args)]
    held[0](*args)
    want = model(*args)
    gc.collect()
    torch.cuda.synchronize()

    def drop():
        held.clear()
        gc.collect()

    g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(g):
        got = model(*args)
        if where == "another thread":
            thread = threading.Thread(target=drop)
            thread.start()
            thread.join()
        else:
            with torch.cuda.stream(side):
                drop()
        twice = got[1] * 2.0
    for _ in range(3):
        g.replay()
        eager = model(*args)
        assert all(torch.equal(x, y) for x, y in zip(got, want))
        assert all(torch.equal(x, y) for x, y in zip(eager, want)) and torch.equal(twice, want[1] * 2.0)
    ops.check_errors()
    assert not hip_runtime._late


def _runtime(close):
    r = hip_runtime.HipRuntime.__new__(hip_runtime.HipRuntime)
    r.close = close
    return r


def test_runtimes_are_closed_by_whoever_comes_first(monkeypatch):
    """Another thread may take the last one between a look and the taking."""
    class Taken(list):
        def __len__(self):
            return 1

    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(hip_runtime, "_late", Taken())
    hip_runtime.close_late()


def test_a_runtime_that_does_not_close_is_nobody_elses_matter(monkeypatch):
    closed, late = [], []

    def fails():
        raise RuntimeError("not closed")

    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(hip_runtime, "_late", late)
    held = [_runtime(lambda: closed.append(1)), _runtime(fails), _runtime(lambda: closed.append(2))]
    late += held  # what is held does not end by itself, which would swallow the failure
    hip_runtime.close_late()
    assert sorted(closed) == [1, 2] and not late


def test_late_runtimes_are_closed_by_a_wait_outside_of_captures(monkeypatch):
    """Where nothing is compiled any more their memory would stay."""
    closed, late, capturing = [], [], [True]
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    monkeypatch.setattr(hip_runtime, "_late", late)
    late.append(_runtime(lambda: closed.append(1)))
    ops.check_errors()
    assert not closed
    capturing[0] = False
    ops.check_errors()
    assert closed and not late


@gpu
def test_late_runtimes_are_closed_by_a_compiled_call():
    args = step_inputs(tokens=3)
    kept, held = mlc.compile(Step().cuda(), args), [mlc.compile(Step().cuda(), args)]
    for compiled in (kept, *held):
        compiled(*args)
    compiled = None
    x = torch.ones(4, device="cuda")
    x * 2.0
    gc.collect()
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        x * 2.0
        held.clear()
        gc.collect()
    assert hip_runtime._late
    kept(*args)
    assert not hip_runtime._late


@gpu
@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two devices")
def test_a_runtime_that_is_closed_leaves_the_current_device():
    last = torch.device("cuda", torch.cuda.device_count() - 1)
    model = torch.nn.Sequential(torch.nn.Linear(64, 64), torch.nn.ReLU()).to(last)
    with torch.cuda.device(last):
        held = [mlc.compile(model, (torch.ones(2, 64, device=last),))]
        held[0](torch.ones(2, 64, device=last))
    torch.cuda.set_device(0)
    held.clear()
    gc.collect()
    assert torch.cuda.current_device() == 0
