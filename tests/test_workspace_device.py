"""Workspace sizes go by the device that a call's tensors are on: they are asked for with it current,
whichever device was so before.  Devices and the library stand in here, so this needs no GPU."""

import contextlib

import pytest
import torch

from pytorch_morlet_fdwt_b200 import _lib
from pytorch_morlet_fdwt_b200.causal_conv import _describe as _describe_convolution
from pytorch_morlet_fdwt_b200.linear_attention import _describe as _describe_attention
from pytorch_morlet_fdwt_b200.selective_scan import _describe as _describe_scan

F32 = torch.float32


class _Library:
    """Its workspaces are as many bytes as the current device's number and 100; others as the
    library's."""

    def __init__(self, real, devices):
        self.real, self.devices, self.asked = real, devices, []

    def __getattr__(self, name):
        if not name.endswith(("_workspace", "_bytes")):
            return getattr(self.real, name)

        def size(desc):
            self.asked.append(name)
            return 100 + self.devices[-1]
        return size


@pytest.fixture
def library(monkeypatch):
    devices = [0]  # the current one last

    @contextlib.contextmanager
    def device(d):
        devices.append(torch.device(d).index)
        try:
            yield
        finally:
            devices.pop()

    fake = _Library(_lib.load(), devices)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: devices[-1])
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(_lib, "load", lambda: fake)
    plans = (_describe_convolution, _describe_attention, _describe_scan)
    for plan in plans:
        plan.cache_clear()
    yield fake
    for plan in plans:
        plan.cache_clear()


def _stride(shape):
    return torch.empty(shape, device="meta").stride()


def _scan(index):
    x, bc = torch.Size((2, 30, 8)), torch.Size((2, 30, 1, 4))
    shapes = (x, x, bc, bc, None)
    return _describe_scan(("B", "L"), (F32,) * 4 + (None,), shapes,
                          tuple(s and _stride(s) for s in shapes), torch.Size((8, 4)), None, True,
                          index)[2:5]


def _convolution(index):
    return _describe_convolution(F32, torch.Size((2, 30, 8)), (240, 8, 1), None, F32,
                                 torch.Size((8, 4)), None, "silu", index)[2:]


def _attention(index):
    shape = torch.Size((2, 30, 2, 16))
    return _describe_attention(("B", "L", "H", "D"), (F32,) * 3, (shape,) * 3,
                               (_stride(shape),) * 3, None, None, index)[2:4]


@pytest.mark.parametrize("plan", [_scan, _convolution, _attention])
def test_sizes_are_those_of_the_tensors_device(plan, library):
    for index in (0, 1, 3):
        sizes = plan(index)
        assert sizes and all(n == 100 + index for n in sizes)
        assert library.devices == [0]
        asked = len(library.asked)
        assert plan(index) == sizes and len(library.asked) == asked  # kept
