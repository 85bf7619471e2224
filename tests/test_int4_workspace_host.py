"""The workspaces of 4-bit products go by the plan, and the plan by the compute units of the device that runs it."""

import torch
from test_devices_host import _Tensor, device  # noqa: F401
from test_gated_devices_host import _matrix

from trnblas_amd.hip import int4_kernels

BF16 = torch.bfloat16


def test_each_device_has_a_size_of_its_own(device, monkeypatch):  # noqa: F811
    bytes_of = {0: 1 << 20, 1: 3 << 20}  # beside the rows as the kernels read them
    asked = []

    def library(name):
        if name != "trnblas_hip_int4_gemm_workspace":
            return lambda *args: device["calls"].append((name, device["current"], args)) or 0

        def workspace(code, gated, groups, R, N, K, group):
            asked.append(device["current"])
            return bytes_of[device["current"]] + R * (-(-K // 128) * 128) * 2

        return workspace

    monkeypatch.setattr(int4_kernels, "_fn", library)
    int4_kernels._partial_bytes.cache_clear()
    try:
        for index in (0, 1, 0, 1):
            with torch.cuda.device(index):
                assert int4_kernels.int4_gemm_fast(1.0, _Tensor((200, 4096), BF16, index), _matrix(index, n=4096, k=4096), None, None) is not None
            sizes = [args[-2] for name, at, args in device["calls"] if at == index]
            assert sizes and all(n == bytes_of[index] for n in sizes)
        assert asked == [0, 1]  # once for each
    finally:
        int4_kernels._partial_bytes.cache_clear()
