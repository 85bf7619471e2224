"""4-bit products of rows at the end of their range: a group's fp32 sum is taken before its scale."""

import pytest
import torch

import trnblas_amd as tb
from trnblas_amd.int4 import Int4Matrix

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_of_2_to_116(dev, dtype, group):
    # one sign, and the largest distance from a zero point: 128 * 255 / 16 * 2^116 lies below 2^127
    for K, N, R in ((128, 48, 1), (1024, 48, 40), (1024, 512, 300)):
        zeros = torch.full((N, K // group), 255, dtype=torch.uint8)
        scales = torch.full((N, K // group), 2.0**-14, dtype=BF16)
        Q = Int4Matrix.from_parts(torch.zeros(N, K // 2, dtype=torch.uint8), scales, K, group, zeros).to(dev)
        A = torch.full((R, K), 2.0**116, dtype=dtype, device=dev)
        D = tb.int4_gemm(1.0, A, Q, dtype=F32)
        assert (D == -255.0 * K * 2.0**102).all(), (K, N, R)  # every partial sum is a number of at most 24 bits


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_the_smallest_rows(dev, dtype):
    # and the least normal values: what is lost lies below them
    tiny = torch.finfo(dtype).tiny
    g = torch.Generator().manual_seed(1)
    for K, N, R in ((128, 48, 1), (1024, 48, 40), (1024, 512, 300)):
        Q = tb.int4_quantize(torch.randn(N, K, generator=g).to(dev), 128, zeros=True)
        A = (torch.randint(1, 64, (R, K), generator=g) * tiny * 64).to(dtype).to(dev)
        W = Q.dequantize().double()
        ref, den = A.double() @ W.T, A.double().abs() @ W.abs().T
        D = tb.int4_gemm(1.0, A, Q, dtype=F32).double()
        # products and pieces of rows below 2^-126 may go: K of them, each within 2^-126 of 16 (values enter in sixteenths)
        assert ((D - ref).abs() <= (K + 2) * 2.0**-23 * den + 3 * K * 16 * 2.0**-126).all()
