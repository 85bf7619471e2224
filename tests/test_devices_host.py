"""Operands on a device that is not the current one: every launch makes it current, or leaves the call to a path that does.
On the CPU, with the device queries and the library stood in for."""

import contextlib

import pytest
import torch

from trnblas_amd.hip import _lib, dispatch, grouped_kernels, kernels


class _Tensor:
    """What the wrappers ask of a device tensor."""

    is_cuda = True
    requires_grad = False

    def __init__(self, shape, dtype, index):
        self.shape, self.dtype, self.device = torch.Size(shape if isinstance(shape, tuple) else (shape,)), dtype, torch.device("cuda", index)

    dim = lambda self: len(self.shape)
    stride = lambda self, i=None: torch.empty(self.shape, device="meta").stride(*(() if i is None else (i,)))
    get_device = lambda self: self.device.index
    data_ptr = lambda self: 4096
    is_neg = lambda self: False
    new_empty = lambda self, shape, dtype=None: _Tensor(shape, dtype or self.dtype, self.device.index)


@pytest.fixture
def device(monkeypatch):
    """The current device, and the calls that the library gets: (name, device current in it, arguments)."""
    state = {"current": 0, "calls": []}

    @contextlib.contextmanager
    def current(index):
        was, state["current"] = state["current"], index
        try:
            yield
        finally:
            state["current"] = was

    class Library:
        def __getattr__(self, name):
            return lambda *args: state["calls"].append((name, state["current"], args)) or 0

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: state["current"], raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0, raising=False)
    monkeypatch.setattr(grouped_kernels, "_raw_stream", lambda index: 0)
    monkeypatch.setattr(grouped_kernels, "_current_device", lambda: state["current"])
    monkeypatch.setattr(torch.cuda, "device", current)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: state["current"])
    monkeypatch.setattr(_lib, "load", Library)
    monkeypatch.setattr(grouped_kernels, "_fns", {})
    return state


@pytest.mark.parametrize("probed", [False, True])
def test_a_launch_makes_its_device_current(device, monkeypatch, probed):
    if probed:
        monkeypatch.setattr(kernels, "_launch_probe", lambda *_: None)
    for index in (1, 0):
        kernels._probed_call("k", "some_kernel", 5, _lib.stream_of(torch.device("cuda", index)))
    assert device["calls"] == [("some_kernel", 1, (5, 0)), ("some_kernel", 0, (5, 0))] and device["current"] == 0
    _lib.call("no_stream", 3)
    assert device["calls"][-1] == ("no_stream", 0, (3,))


def test_the_short_paths_serve_the_current_device_only(device, monkeypatch):
    monkeypatch.setattr(dispatch, "_backend", "hip")
    bf16, off = torch.bfloat16, torch.int32
    for index in (1, 0):
        t = lambda *shape, dtype=bf16: _Tensor(shape, dtype, index)
        codes = t(8, 16, dtype=torch.uint8), t(1, 1, 256, dtype=torch.uint8)
        got = [
            grouped_kernels.grouped_gemm_fast(1.0, t(4, 32), t(2, 32, 16), t(3, dtype=off), False, None),
            grouped_kernels.grouped_rank_k_fast(1.0, t(4, 32), t(4, 16), t(3, dtype=off), None),
            grouped_kernels.mx_gemm_fast(1.0, t(4, 32), codes, None, None),
            grouped_kernels.mx_quantize_fast(t(4, 32)),
            grouped_kernels.mx_dequantize_fast(*codes, 32, bf16),
        ]
        assert all((x is None) == (index == 1) for x in got)
        assert len(device["calls"]) == (0 if index else len(got))
    f32 = lambda *shape: _Tensor(shape, torch.float32, 1)
    assert dispatch.gemm_fast(1.0, f32(4, 32), f32(32, 16), 0.0, None, False, False) is None
