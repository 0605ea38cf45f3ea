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
