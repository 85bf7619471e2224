"""Which calls of the gated projections and 4-bit products take the short path, with the library stood in for."""

import pytest
import torch

import trnblas_amd as tb
from trnblas_amd import gated


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
