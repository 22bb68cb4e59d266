"""Rules of FieldOps that hold without a GPU."""
import ctypes

import pytest
import torch

from gsplat_tt_amd import field


class _Library:
    """Stands for the library: keeps the context pointer of each call."""

    def __init__(self):
        self.handles = []

    def gs_lookup_dev(self, handle, *rest):
        self.handles.append(handle.value)
        return 0


class _Context:
    device_index = -1  # what CPU tensors say

    def __init__(self, lib):
        self._L, self.handle = lib, ctypes.c_void_p(0x1000)

    def close(self):
        self.handle = ctypes.c_void_p()


def test_a_closed_context_is_not_used(monkeypatch):
    """After Context.close() a call passes the null pointer that the library refuses,
    never the freed one."""
    lib = _Library()
    ctx = _Context(lib)
    real = torch.device
    monkeypatch.setattr(field.torch, "device", lambda *a: real("cpu"))
    monkeypatch.setattr(field.torch.cuda, "current_stream", lambda *a: _Stream())
    ops = field.FieldOps(ctx)
    table, ids = torch.ones(3, 4), torch.zeros(2, dtype=torch.int64)
    ops.lookup(table, ids)
    ctx.close()
    ops.lookup(table, ids)
    assert lib.handles == [0x1000, None]


class _Stream:
    cuda_stream = 0

    def synchronize(self):
        pass


def test_label_loss_sizes_past_a_launch_are_refused():
    lib = field.L.load_library()
    assert lib.gs_label_loss_workspace(2 ** 31 - 256, 2, 1, 1, 0) > 0
    assert lib.gs_label_loss_workspace(2 ** 31 - 255, 2, 1, 1, 0) == -1
