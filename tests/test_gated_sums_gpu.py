"""The fp32 sums that a gated projection keeps for its gradient, and the gradient taken from them, on the GPU. Bounds: `oracle.gated`'s."""

import pytest
import torch
from test_gated_gpu import REACH, _operands
from test_gated_sums_host import FAR, check

from oracle import gated as og
from oracle.grouped import uneven as _uneven
from trnblas_amd.hip import _lib, gated_kernels

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.mark.parametrize("kernel", list(REACH))
def test_each_kernel_keeps_its_sums(dev, kernel):
    for i, (dtype, transB, G, R, N, K) in enumerate(REACH[kernel]):
        A, B = _operands(i, dtype, R, K, N, G, transB, dev)
        off = _uneven(G, R, i) if R > 4 * G else torch.arange(G + 1) * (R // G)
        for n in (N, N - 3) if K % 8 == 0 and transB else (N,):  # columns that are no multiple of four: value by value
            b = B if n == N else B[:, : 2 * n].contiguous()
            H, S = gated_kernels.gated_gemm(A, b.mT if transB else b, off.to(dev), "silu", dtype, True)
            P, den = og.products(A, b, off, transB)
            assert H.dtype == dtype and S.dtype == F32 and S.shape == (R, 2 * n)
            e = (K + 2) * 2.0**-23 * den
            assert og.ratio(S, P, e + og.TINY[F32]) <= 1, (dtype, transB, G, R, n, K)
            assert og.ratio(H, *og.forward("silu", P, den, K, dtype)) <= 1


@pytest.mark.parametrize("act", og.ACTS)
@pytest.mark.parametrize("name", list(FAR))
def test_gradients_of_far_sums(dev, name, act):
    for transB in (False, True):
        check(name, act, dev, transB)


@pytest.mark.parametrize("act", og.ACTS)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_gate_backward(dev, dtype, act):
    g = torch.Generator().manual_seed(6)
    for R, N in ((1, 8), (5, 64), (130, 520), (3, 1), (7, 61), (131, 515), (2, 4096)):
        P = torch.randn(R, 2 * N, generator=g) * 3
        dH = torch.randn(R, N, generator=g).to(dtype)
        dP = gated_kernels.gate_backward(P.to(dev), dH.to(dev), act)
        wide = torch.full((R, N + 9), float("nan"), dtype=dtype, device=dev)
        wide[:, 1 : N + 1] = dH.to(dev)  # rows that start anywhere
        # (these go one value at a time, by a kernel of its own: the compiler may round a product to fp32 and then to 16 bits in one,
        # at once in the other, which differ by a unit where the first lies halfway; both lie within the bound below)
        dP = dP, gated_kernels.gate_backward(P.to(dev), wide[:, 1 : N + 1], act)
        G, U = P.double().chunk(2, -1)
        # act and act' within FN (1 + |G|), two products
        e = dH.double().abs().repeat(1, 2) * torch.cat([U.abs(), torch.ones_like(U)], 1) * (og.FN * (1.0 + G.abs())).repeat(1, 2)
        want = og.backward(act, P.double(), dH)
        e = e + 2.0**-22 * (want.abs() + e)
        for got in dP:
            assert got.dtype == dtype and og.ratio(got.cpu(), want, e + og.EPS[dtype] * (want.abs() + e) + og.TINY[dtype]) <= 1, (R, N)


@pytest.mark.parametrize("act", og.ACTS)
@pytest.mark.parametrize("dtype, out", [(BF16, BF16), (F16, F16), (F32, BF16), (F32, F16), (F32, F32)])
def test_gate_of_every_type(dev, dtype, out, act):
    # the C entry, of P in 16 bits too: alone, and with P as it goes into the result's type; rows that start anywhere
    g = torch.Generator().manual_seed(7)
    codes = _lib.DTYPE_CODES
    for R, N, gap in ((1, 8, 0), (130, 520, 0), (7, 61, 0), (5, 64, 3), (33, 72, 8)):
        P = torch.full((R, 2 * N + gap), float("nan"), dtype=dtype)
        P[:, : 2 * N] = (torch.randn(R, 2 * N, generator=g) * 3).to(dtype)
        G, U = P[:, : 2 * N].double().chunk(2, -1)
        want = og.gate(act, G)[0] * U
        e = U.abs() * og.FN * (1.0 + G.abs()) + 2.0**-23 * want.abs()
        for keep in (False, True):
            p = P.to(dev)
            H = torch.full((R, N + gap), 7.0, dtype=out, device=dev)
            S = torch.full((R, 2 * N + gap), 7.0, dtype=out, device=dev)
            stream = torch.cuda.current_stream().cuda_stream
            _lib.call("trnblas_hip_gate", gated_kernels.ACTS[act], codes[dtype], codes[out], R, N, p.data_ptr(), 2 * N + gap, H.data_ptr(),
                      N + gap, S.data_ptr() if keep else None, 2 * N + gap, stream)  # fmt: skip
            assert og.ratio(H[:, :N].cpu(), want, e + og.EPS[out] * (want.abs() + e) + og.TINY[out]) <= 1, (R, N)
            assert (H[:, N:] == 7.0).all() and (S[:, 2 * N :] == 7.0).all()
            assert torch.equal(S[:, : 2 * N], p[:, : 2 * N].to(out)) if keep else (S == 7.0).all()
