"""Gated projections whose sums lie past the range of a 16-bit type while results and gradients do not."""

import pytest
import torch

import trnblas_amd as tb
from oracle import gated as og

# (rows, gate weights, up weights): sums of two products each
FAR = {
    "gates far below zero": ([300.0, 300.0], [-150.0, -150.0], [0.5, 0.25]),
    "ups past the range, gates far below zero": ([300.0, 300.0], [-30.0, -31.0], [200.0, 150.0]),
    "ups past the range, gates below zero": ([300.0, 300.0], [-0.03125, -0.015625], [200.0, 150.0]),
    "ups past the range, gates near zero": ([300.0, 300.0], [2.0**-14, -(2.0**-15)], [200.0, 150.0]),
}


def _case(name, device):
    x, g, u = (torch.tensor(v, dtype=torch.float16, device=device) for v in FAR[name])
    # three rows and eight columns of H of the same values
    return x.expand(3, 2).contiguous(), torch.cat([g[:, None].expand(2, 8), u[:, None].expand(2, 8)], 1).contiguous()


def check(name, act, device, transB=False):
    A, B = _case(name, device)
    dH = (torch.arange(24, device=device).reshape(3, 8) - 12).half() * 2.0**-15
    a, b = A.clone().requires_grad_(), (B.mT.contiguous() if transB else B.clone()).requires_grad_()
    H = tb.gated_gemm(a, b, act, transB=transB)
    dA, dB = torch.autograd.grad(H, (a, b), dH)
    A, B, dH, dA, dB = (t.cpu() for t in (A, B, dH, dA, dB.mT if transB else dB))
    P, den = og.products(A, B[None], torch.tensor([0, 3]))
    assert og.ratio(H.cpu(), *og.forward(act, P, den, 2, torch.float16)) <= 1
    # P in fp32; dP rounded to fp16; products of at most sixteen terms summed in fp32, rounded once
    dP, e = og.backward(act, P, dH), og.gradient_bounds(act, P, den, dH, 2, torch.float32)
    e = e + og.EPS[torch.float16] * (dP.abs() + e) + og.TINY[torch.float16]
    A, B = A.double(), B.double()
    for got, ref, err, size in ((dA, dP @ B.T, e @ B.abs().T, dP.abs() @ B.abs().T), (dB, A.T @ dP, A.abs().T @ e, A.abs().T @ dP.abs())):
        err = err + 18 * 2.0**-23 * (size + err)
        err = err + og.EPS[torch.float16] * (ref.abs() + err) + og.TINY[torch.float16]
        assert ref.abs().max() < 65504 and got.isfinite().all(), (name, act)
        assert og.ratio(got, ref, err) <= 1, (name, act)


@pytest.mark.parametrize("act", og.ACTS)
@pytest.mark.parametrize("name", list(FAR))
def test_gradients_of_far_sums(name, act):
    check(name, act, "cpu")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16, torch.float64])
def test_sums_are_kept_in_32_bits_or_more(dtype):
    from trnblas_amd import gated

    A = torch.tensor([[1.0, 2.0**-12]], dtype=dtype)
    B = torch.tensor([[1.0, 1.0], [0.0, 1.0]], dtype=dtype)  # G = 1, U = 1 + 2^-12, which has more than 16 bits
    H, P = gated._forward(A, B[None], None, "relu", dtype, True)
    want = torch.tensor([[1.0, 1.0 + 2.0**-12]], dtype=torch.promote_types(dtype, torch.float32))
    assert H.dtype == dtype and P.dtype == want.dtype and torch.equal(P, want)
    assert gated._backward(P, torch.ones(1, 1, dtype=dtype), "relu").dtype == dtype
