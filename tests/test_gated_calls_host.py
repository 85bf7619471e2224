"""Which calls of the gated projections and 4-bit products take the short path, with the library stood in for."""

import pytest
import torch
from test_devices_host import _Tensor, device  # noqa: F401

import trnblas_amd as tb
from trnblas_amd import gated
from trnblas_amd.hip import _lib, gated_kernels


class _Short:
    """The short path, which takes whatever it is given."""

    def __init__(self):
        self.calls = []

    def gated_gemm_fast(self, A, B, offsets, activation, transB, dtype):
        self.calls.append((tuple(B.shape), offsets is not None))
        return A.new_zeros(A.shape[0], B.shape[-1] // 2)


@pytest.fixture
def short(monkeypatch):
    path = _Short()
    monkeypatch.setattr(gated, "_gk", lambda: path)
    monkeypatch.setattr(gated, "_fast_call", lambda *_: True)
    return path


def test_the_short_path_takes_operands_of_the_documented_dimensions(short):
    A, B, off = torch.zeros(6, 4), torch.zeros(1, 4, 6), torch.tensor([0, 6])
    with pytest.raises(ValueError, match="2-D"):
        tb.gated_gemm(A, B)  # a stack of one is no matrix
    with pytest.raises(ValueError, match="3-D"):
        tb.grouped_gated_gemm(A, B[0], off)
    assert not short.calls
    tb.gated_gemm(A, B[0])
    tb.grouped_gated_gemm(A, B, off)
    assert short.calls == [((4, 6), False), ((1, 4, 6), True)]


class TestFarRows:
    """Leading dimensions past the 32-bit offsets of the fused kernels: the product goes to fp32 by the grouped kernels, which take any, and
    the gate is a launch of its own, or the operand is copied first."""

    # (dtype, strides of A (4, 64), strides of op(B) stored (64, 32) or (32, 64), transB): 256 rows of A or of a transposed B, 128 bytes of k of
    # the other kind, lie within 2^31 bytes
    FAR = [
        (torch.bfloat16, (1 << 22, 1), (32, 1), False),
        (torch.float32, (1 << 21, 1), (32, 1), False),
        (torch.float16, (64, 1), (1 << 22, 1), True),
        (torch.float32, (64, 1), (1 << 21, 1), True),
        (torch.bfloat16, (64, 1), (1 << 24, 1), False),
        (torch.float32, (64, 1), (1 << 24, 1), False),
    ]
    NEAR = [
        (torch.bfloat16, ((1 << 22) - 8, 1), (32, 1), False),
        (torch.float32, ((1 << 21) - 8, 1), (32, 1), False),
        (torch.float16, (64, 1), ((1 << 22) - 8, 1), True),
        (torch.float32, (64, 1), ((1 << 21) - 8, 1), True),
        (torch.bfloat16, (64, 1), ((1 << 24) - 16, 1), False),
        (torch.float32, (64, 1), ((1 << 24) - 16, 1), False),
    ]

    @staticmethod
    def _call(device, dtype, a, b, transB, rows=4):
        class T(_Tensor):
            def __init__(self, shape, dtype, strides):
                super().__init__(shape, dtype, 0)
                self.strides = strides

            stride = lambda self, i=None: self.strides if i is None else self.strides[i]
            unsqueeze = lambda self, _: T((1, *self.shape), self.dtype, (0, *self.strides))
            new_empty = lambda self, shape, dtype=None: _Tensor(shape, dtype or self.dtype, 0)

        A, B = T((rows, 64), dtype, a), T((32, 64) if transB else (64, 32), dtype, b)
        device["calls"].clear()
        assert gated_kernels.gated_gemm_fast(A, B, None, "silu", transB, None) is not None
        return [(name.removeprefix("trnblas_hip_"), args) for name, _, args in device["calls"]]

    def test_kernels(self, device):  # noqa: F811
        for case in self.FAR:
            assert [name for name, _ in self._call(device, *case)] == ["grouped_gemm", "gate"], case
        for case in self.NEAR:
            assert [name for name, _ in self._call(device, *case)] == ["gated_gemm"], case

    def test_one_row_is_never_far(self, device):  # noqa: F811
        for dtype in (torch.float32, torch.bfloat16):
            ((name, args),) = self._call(device, dtype, (1 << 40, 1), (32, 1), False, rows=1)
            assert name == "gated_gemm" and args[8] == 64

    def test_one_row_without_values(self, device):  # noqa: F811
        # no operand to read: not the fused kernels
        A, B, off = _Tensor((1, 0), torch.bfloat16, 0), _Tensor((1, 0, 32), torch.bfloat16, 0), _Tensor(2, torch.int32, 0)
        assert gated_kernels.gated_gemm_fast(A, B, off, "silu", False, None) is not None
        assert [name.removeprefix("trnblas_hip_") for name, _, _ in device["calls"]] == ["grouped_gemm", "gate"]

    def test_the_library_refuses_them(self):
        # so none may reach it
        if not _lib.LIB_PATH.exists():
            pytest.skip("library not built")
        lib = _lib.load()
        for dtype, (lda, _), (ldb, _), transB in self.FAR:
            code = _lib.DTYPE_CODES[dtype]
            rc = lib.trnblas_hip_gated_gemm(0, code, transB, 1, 4, 16, 64, 4096, lda, 4096, ldb, 0, 16 * ldb if transB else 16, None, 0, 4096, 16,
                                            None, 32, 0, None)  # fmt: skip
            assert rc == _lib.E_ARG and b"16 bytes" in lib.trnblas_hip_last_error()
