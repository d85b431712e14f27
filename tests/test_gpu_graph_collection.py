"""Captured graphs that nobody holds any more are gone before another capture begins (tests/conftest.py)."""
import gc
import weakref

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_dead_graphs_are_collected_before_a_capture():
    x = torch.zeros(64, device='cuda')

    class Holder:
        pass

    def held_by_a_cycle():
        holder = Holder()
        holder.me, holder.graph = holder, torch.cuda.CUDAGraph()
        with torch.cuda.graph(holder.graph):
            x.add_(1)
        return weakref.ref(holder)

    gc.disable()                 # (its own moment to run must not decide this)
    try:
        holder = held_by_a_cycle()
        assert holder() is not None
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            dead = holder() is None
            x.add_(1)
    finally:
        gc.enable()
    assert dead
    graph.replay()
    torch.cuda.synchronize()
    assert float(x[0]) == 1.0
