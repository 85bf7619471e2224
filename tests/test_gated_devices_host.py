"""Gated projections and 4-bit weights on a device that is not the current one, as in `test_devices_host.py`: the short paths
leave it to the others, and the launches that have one way make it current."""

import torch
from test_devices_host import _Tensor, device  # noqa: F401

from trnblas_amd.hip import gated_kernels, int4_kernels
from trnblas_amd.int4 import Int4Matrix

F32, BF16, U8 = torch.float32, torch.bfloat16, torch.uint8


def _matrix(index, *lead, n=32, k=128):
    t = lambda *shape, dtype: _Tensor(shape, dtype, index)
    parts = t(*lead, n // 16, 1, 1024, dtype=U8), t(*lead, n // 16, 1, 16, 1, dtype=BF16), None
    return Int4Matrix._of(parts, (*lead, n, k), 128)


def test_the_short_paths_serve_the_current_device_only(device, monkeypatch):  # noqa: F811
    monkeypatch.setattr(int4_kernels, "_partial_bytes", lambda *_: 64)
    for index in (1, 0):
        t = lambda *shape, dtype=BF16: _Tensor(shape, dtype, index)
        off, E, Q = t(3, dtype=torch.int32), _matrix(index, 2), _matrix(index)
        q = Q.codes, Q.scales, Q.zeros
        got = [
            gated_kernels.gated_gemm_fast(t(4, 32), t(32, 16), None, "silu", False, None),
            gated_kernels.gated_gemm_fast(t(4, 32), t(2, 16, 32), off, "gelu", True, None, True),
            gated_kernels.gated_gemm_fast(t(4, 33), t(2, 33, 16), off, "gelu", False, None),
            gated_kernels.gated_gemm_fast(t(4, 32), t(2, 32, 16), off, "relu", False, F32, True),
            int4_kernels.int4_gemm_fast(1.0, t(4, 128), Q, None, None),
            int4_kernels.int4_gemm_fast(1.0, t(4, 128), E, off, F32, "silu"),
            int4_kernels.quantize_fast(t(4, 32), 64, True, BF16),
            int4_kernels.dequantize_fast(q, (32, 128), 128, BF16),
        ]
        assert all((x is None) == (index != 0) for x in got), (index, got)
    names = [name.removeprefix("trnblas_hip_") for name, _, _ in device["calls"]]
    assert names == ["gated_gemm", "gated_gemm", "grouped_gemm", "gate", "grouped_gemm", "gate", "int4_gemm", "int4_gemm",
                     "int4_quantize", "int4_dequantize"]  # fmt: skip


def test_offsets_on_another_device_take_the_general_path(device):  # noqa: F811
    t = lambda *shape, dtype=BF16, index=0: _Tensor(shape, dtype, index)
    off = t(3, dtype=torch.int32, index=1)
    assert gated_kernels.gated_gemm_fast(t(4, 32), t(2, 32, 16), off, "silu", False, None) is None
    assert gated_kernels.gated_gemm_fast(t(4, 32), t(32, 16, index=1), None, "silu", False, None) is None
    assert int4_kernels.int4_gemm_fast(1.0, t(4, 128), _matrix(0, 2), off, None) is None
    assert int4_kernels.int4_gemm_fast(1.0, t(4, 128), _matrix(1), None, None) is None
    assert not device["calls"]


def test_the_gate_makes_its_device_current(device):  # noqa: F811
    for index in (1, 0):
        P, dH = _Tensor((4, 16), F32, index), _Tensor((4, 8), F32, index)
        H, S = gated_kernels.gate(P, "silu", BF16, True)
        dP = gated_kernels.gate_backward(P, dH, "silu")
        assert (H.dtype, S.dtype, dP.dtype) == (BF16, BF16, F32) and H.get_device() == S.get_device() == dP.get_device() == index
    assert [(name, at) for name, at, _ in device["calls"]] == [(f"trnblas_hip_{n}", i) for i in (1, 0) for n in ("gate", "gate_backward")]
