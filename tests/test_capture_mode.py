"""CPU: a process group's watchdog thread queries events at any time, so what is captured beside one forbids such calls in the
capturing thread only."""
import contextlib

import torch
import torch.distributed as dist

from pde_amd.pinn import PhysicsInformedNN


def test_capture_beside_a_process_group(monkeypatch, tmp_path):
    modes = []

    @contextlib.contextmanager
    def graph(g, pool=None, stream=None, capture_error_mode="global"):
        modes.append(capture_error_mode)
        yield
    monkeypatch.setattr(torch.cuda, "CUDAGraph", object)
    monkeypatch.setattr(torch.cuda, "graph", graph)
    model = object.__new__(PhysicsInformedNN)
    assert not dist.is_initialized()
    assert model._capture(lambda: 5)[1] == 5 and modes == ["global"]
    dist.init_process_group("gloo", init_method="file://%s" % (tmp_path / "store"), rank=0, world_size=1)
    try:
        assert model._capture(lambda: 6)[1] == 6 and modes == ["global", "thread_local"]
    finally:
        dist.destroy_process_group()
    assert model._capture(lambda: 7)[1] == 7 and modes[2] == "global"
