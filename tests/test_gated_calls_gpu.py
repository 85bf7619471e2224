"""Calls of the gated projections that the short paths leave to the others."""

import pytest
import test_gated_shared_host
import torch
from test_gated_shared_host import CASES

import trnblas_amd as tb
from oracle import gated as og

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


def _apart(X, step, dev):
    """X (rows, columns) with `step` values from row to row, one device buffer."""
    return torch.zeros((X.shape[0] - 1) * step + X.shape[1], dtype=X.dtype, device=dev).as_strided(X.shape, (step, 1)).copy_(X)


def _holds(H, A, B, transB, dtype):
    P, den = og.products(A, B[None], torch.tensor([0, A.shape[0]]), transB)
    return og.ratio(H.detach().cpu(), *og.forward("silu", P, den, A.shape[1], dtype)) <= 1


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_rows_far_apart(dev, dtype):
    # on both sides of what the fused kernels reach: small products, and ones whose operands are copied first; one row alone
    es = 4 if dtype == F32 else 2
    g = torch.Generator().manual_seed(1)
    for R, K, N in ((1, 64, 40), (40, 64, 40), (70, 72, 33), (300, 1024, 2056)):
        A = torch.randn(R, K, generator=g).to(dtype)
        for transB in (False, True):
            B = (torch.randn(*((2 * N, K) if transB else (K, 2 * N)), generator=g) * K**-0.5).to(dtype)
            near = 2**31 // (256 * es)
            for step in (near - 8, near, 2 * near + 3):
                a = _apart(A, step, dev).requires_grad_()
                H = tb.gated_gemm(a, B.to(dev), transB=transB)
                assert H.dtype == dtype and _holds(H, A, B, transB, dtype), (R, K, N, transB, step)
                assert torch.equal(tb.gated_gemm(a.detach(), B.to(dev), transB=transB), H)
                if step == near:
                    dH = torch.ones_like(H)
                    c = A.to(dev).requires_grad_()
                    (want,) = torch.autograd.grad(tb.gated_gemm(c, B.to(dev), transB=transB), c, dH)
                    (dA,) = torch.autograd.grad(H, a, dH)
                    # P may be summed by another kernel: dP differs by its roundings and one of its type, and each product by its own
                    size = float(want.abs().max())
                    assert float((dA - want).abs().max()) <= 8 * og.EPS[dtype] * size + 2.0**-18 * size
                del a, H


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_weights_far_apart(dev, dtype):
    es = 4 if dtype == F32 else 2
    g = torch.Generator().manual_seed(2)
    for R in (1, 40):
        for transB, (K, N) in ((False, (9, 33)), (False, (16, 40)), (True, (64, 24)), (True, (33, 24))):
            A = torch.randn(R, K, generator=g).to(dtype)
            B = (torch.randn(*((2 * N, K) if transB else (K, 2 * N)), generator=g) * K**-0.5).to(dtype)
            near = 2**31 // (256 * es) if transB else 2**31 // 128
            for step in (near - 16, near):
                assert _holds(tb.gated_gemm(A.to(dev), _apart(B, step, dev), transB=transB), A, B, transB, dtype), (R, transB, K, N, step)


def test_rows_longer_than_reach(dev):
    # K past 2^31 / 512 values: no copy brings the rows together
    K = (1 << 22) + 8
    A = torch.randint(-1, 2, (3, K), generator=torch.Generator().manual_seed(3)).to(BF16)
    B = (torch.randint(-1, 2, (16, K), generator=torch.Generator().manual_seed(4)) * 2.0**-10).to(BF16)
    # whole numbers of 2^-10 below 2^12: every order of summation gives the same sums
    assert _holds(tb.gated_gemm(A.to(dev), B.to(dev), transB=True), A, B, True, BF16)


def test_the_last_tokens_of_sequences(dev):
    x = torch.randn(6, 1100, 4096, generator=torch.Generator(device=dev).manual_seed(5), device=dev).to(BF16)
    W = (torch.randn(512, 4096, generator=torch.Generator().manual_seed(6)) / 64).to(BF16)
    last = x[:, -1]
    assert last.stride(0) > 1 << 22
    H = tb.gated_gemm(last, W.to(dev), transB=True)
    assert _holds(H, last.cpu(), W, True, BF16)


def test_one_row_of_no_values(dev):
    for dtype in (F32, BF16, F16):
        for N in (16, 5):
            H = tb.gated_gemm(torch.ones(1, 0, dtype=dtype, device=dev), torch.zeros(0, 2 * N, dtype=dtype, device=dev))
            assert H.shape == (1, N) and not H.any()


@pytest.mark.parametrize("name", list(CASES))
def test_operands_that_depend_on_each_other(dev, name, monkeypatch):
    # first and second derivatives, fp32 on the GPU against 64 bits on the host
    leaves, own, plain = CASES[name]

    def second(f, device, dtype):
        x = [(t / 4).to(device, dtype).requires_grad_() for t in leaves]
        first = torch.autograd.grad(f(*x).square().sum(), x, create_graph=True)
        return [t.detach() for t in first] + list(torch.autograd.grad(sum(g.square().sum() for g in first), x))

    want = second(plain, "cpu", torch.float64)
    monkeypatch.setattr(test_gated_shared_host, "OFF", test_gated_shared_host.OFF.to(dev))
    for got, ref in zip(second(own, dev, F32), want):
        # some hundred fp32 operations
        assert torch.allclose(got.double().cpu(), ref, rtol=1e-4, atol=1e-4 * float(ref.abs().max())), name


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_a_step_repeats_itself(dev, dtype):
    g = torch.Generator(device=dev).manual_seed(8)
    off = torch.tensor([0, 300, 300, 1100], device=dev)
    for K, N in ((264, 520), (261, 515)):
        a = torch.randn(1100, K, generator=g, device=dev).to(dtype).requires_grad_()
        b = (torch.randn(3, K, 2 * N, generator=g, device=dev) / 16).to(dtype).requires_grad_()
        dH = torch.randn(1100, N, generator=g, device=dev).to(dtype)

        def step():
            H = tb.grouped_gated_gemm(a, b, off)
            return (H.detach(), *torch.autograd.grad(H, (a, b), dH))

        first = step()
        for _ in range(4):
            assert all(torch.equal(x, y) for x, y in zip(first, step()))
