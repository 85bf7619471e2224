"""Calls of the gated projections that the short paths leave to the others."""

import pytest
import torch

import trnblas_amd as tb

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_a_stack_of_one_is_no_matrix(dev, dtype):
    for K in (64, 33):
        A, B = torch.ones(6, K, dtype=dtype, device=dev), torch.ones(1, K, 16, dtype=dtype, device=dev)
        for transB in (False, True):
            with pytest.raises(ValueError, match="2-D"):
                tb.gated_gemm(A, B.mT.contiguous() if transB else B, transB=transB)
        with pytest.raises(ValueError, match="3-D"):
            tb.grouped_gated_gemm(A, B[0], torch.tensor([0, 6], device=dev))
        assert torch.equal(tb.gated_gemm(A, B[0]), tb.grouped_gated_gemm(A, B, torch.tensor([0, 6], device=dev)))
