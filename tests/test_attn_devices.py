"""Attention's workspaces by device, without a GPU: how a call is cut goes by the CUs of the device that it runs on, so that the
bytes asked for have to be that device's, whichever device is the current one and whichever asked before."""

from __future__ import annotations

import importlib
from types import SimpleNamespace

import pytest
import torch

CUS = {0: 256, 1: 32}  # of two devices that are not alike


def _tensors(index: int):
    """A tensor type whose tensors say that they lie on GPU `index` (their data is never read)."""

    class OnGpu(torch.Tensor):
        is_cuda = property(lambda self: True)
        device = property(lambda self: torch.device("cuda", index))

        def get_device(self):
            return index

    return lambda *shape, dtype=torch.bfloat16: torch.zeros(*shape, dtype=dtype).as_subclass(OnGpu)


@pytest.fixture
def launches(gdn, monkeypatch):
    """Records (device, entry point, workspace bytes) of the calls; the library's sizes stand for the current device."""
    ops = importlib.import_module("zonos3-mini_amd.ops")
    current, made = [0], []

    class Device:
        def __init__(self, device):
            self.index = device if isinstance(device, int) else device.index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *_):
            current[0] = self.before

    size = lambda *sizes: 64 * CUS[current[0]] + len(sizes)  # noqa: E731
    library = SimpleNamespace(zattn_window_fwd_workspace_bytes=size, zattn_window_step_workspace_bytes=size)
    monkeypatch.setattr(ops._native, "lib", lambda: library)
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(ops, "_launch", lambda index, dev, name, *args: made.append((index, name, args[-1])))
    yield made
    for kept in vars(ops).values():  # (no size of these devices is left for other tests)
        if hasattr(kept, "cache_clear"):
            kept.cache_clear()


@pytest.mark.parametrize("order", [(0, 1, 0), (1, 0, 1)])
def test_workspaces_go_by_the_tensors_device(gdn, launches, order):
    for index in order:
        z = _tensors(index)
        q, k, c = z(1, 20 + order[0], 4, 64), z(1, 20 + order[0], 2, 64), z(2, 48 + order[0], 2, 64)
        gdn.window_attn_fwd(q, k, k, window=9, sinks=1)
        gdn.window_attn_step(q[0, :2], c, c, z(2, dtype=torch.int32), window=9)
    assert launches == [(i, n, 64 * CUS[i] + s) for i in order for n, s in (("zattn_window_fwd", 10), ("zattn_window_step", 8))]


@pytest.mark.gpu
def test_sizes_first_met_in_a_capture(gdn, cuda):
    """A workspace's size is asked for, and its device made current, while a graph is captured: sizes that no call had before."""
    importlib.import_module("zonos3-mini_amd.ops")._attn_workspace.cache_clear()
    g = torch.Generator().manual_seed(91)
    r = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).to(cuda)  # noqa: E731
    q, k, v, n = r(1, 11, 8, 128), r(1, 2900, 2, 128), r(1, 2900, 2, 128), torch.tensor([2801], dtype=torch.int32, device=cuda)
    calls = lambda: (gdn.window_attn_fwd(q, k, v), gdn.window_attn_step(q[:, -1], k, v, n))  # noqa: E731
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = calls()
    want = calls()
    for _ in range(3):
        for o in out:
            o.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        want = calls()
