"""Captures of the engine beside graphs that nobody holds any more."""
import gc

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_capture_outlives_forgotten_graphs():
    """A cycle that holds a graph, and a collector that would run at the next allocation: the capture ends well, and the collector is as it was."""
    from rexl3_b200.engine.gpu_backend import capturing
    x = torch.zeros(8, device="cuda")

    class Holder:
        pass
    x.add_(1)
    torch.cuda.synchronize()
    before = gc.get_threshold()
    for on in (True, False):
        gc.collect()
        h = Holder()
        h.graph, h.me = torch.cuda.CUDAGraph(), h
        with capturing(h.graph):
            x.add_(1)
        g = torch.cuda.CUDAGraph()
        try:
            gc.enable() if on else gc.disable()
            gc.set_threshold(100000, 1, 1)                     # (nothing runs until the capture has begun)
            del h
            with capturing(g):
                gc.set_threshold(1, 1, 1)
                keep = [[i] for i in range(1000)]
                x.add_(2)
            gc.set_threshold(*before)
            assert gc.isenabled() == on and len(keep) == 1000
        finally:
            gc.set_threshold(*before)
            gc.enable()
        x.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert bool((x == 2).all())


def test_the_collector_comes_back_after_a_capture_that_failed():
    from rexl3_b200.engine.gpu_backend import capturing
    x = torch.zeros(8, device="cuda")
    with pytest.raises(ZeroDivisionError):
        with capturing(torch.cuda.CUDAGraph()):
            x.add_(1)
            1 // 0
    assert gc.isenabled()
    torch.cuda.synchronize()
