"""Microscaled 4-bit floats on host tensors: values, layout, products, refusals."""

import pytest
import torch

import trnblas_amd as tb
from oracle import grouped as og
from oracle import mx as om
from oracle.mx import wide as _wide


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(1, 1), (3, 32), (17, 33), (16, 512), (5, 1030), (2, 19, 70)])
def test_quantize(shape, dtype):
    X = _wide(torch.Generator().manual_seed(0), *shape, dtype=dtype)
    Q = tb.mx_quantize(X)
    want, code, byte = om.quantize(X)
    assert Q.shape == X.shape
    assert torch.equal(Q.dequantize().double(), want)
    assert torch.equal(Q.block_scales().long(), byte)
    got = torch.stack([Q.codes & 7, Q.codes >> 4 & 7], -1).flatten(-2)
    assert torch.equal(got.long(), code)
    again = tb.MXMatrix.from_parts(Q.codes, Q.block_scales(), X.shape[-1])
    assert torch.equal(again.scales, Q.scales)
    T = tb.mx_quantize(X.mT.contiguous(), trans=True)
    assert torch.equal(T.codes, Q.codes) and torch.equal(T.scales, Q.scales)
    if X.dim() == 3:
        assert torch.equal(Q[1].dequantize(), Q.dequantize()[1])


def test_scale_bytes_are_where_the_layout_says():
    X = torch.ones(40, 1200)
    X *= torch.exp2(torch.arange(40).float() % 7)[:, None] * torch.exp2((torch.arange(1200) // 32).float() % 5)
    Q = tb.mx_quantize(X)
    for r, b in ((0, 0), (1, 0), (15, 3), (16, 4), (39, 37), (20, 17)):
        want = 127 - 2 + r % 7 + b % 5
        bb = b % 16
        assert int(Q.scales[r // 16, b // 16, 64 * (bb % 4) + 4 * (r % 16) + bb // 4]) == want


def test_values_at_the_ends():
    big, tiny = torch.finfo(torch.float32).max, 2.0**-149
    X = torch.zeros(6, 64)
    X[0, 3], X[0, 40] = big, -big
    X[1, 0], X[1, 1], X[1, 33] = tiny, 2.0**-126, 2.0**-128
    X[2, 5] = float("inf")
    X[3, 5], X[3, 6] = float("nan"), float("-inf")
    X[4, 1] = -0.0
    X[5, :8] = torch.tensor([7.99, 7.0, 5.0, 5.01, 3.5, 2.5, 0.25, 0.2501])
    Q = tb.mx_quantize(X)
    want, _, byte = om.quantize(X)
    V = Q.dequantize()
    assert torch.equal(V.double().nan_to_num(-1.0), want.nan_to_num(-1.0)) and torch.equal(V.isnan(), want.isnan())
    assert V[2, :32].isnan().all() and not V[2, 32:].any() and V[3, :32].isnan().all()
    assert torch.equal(Q.block_scales().long(), byte)
    assert V[5, :8].tolist() == [6, 6, 4, 6, 4, 2, 0, 0.5]


def test_products():
    g = torch.Generator().manual_seed(1)
    A, W, C = _wide(g, 9, 70), _wide(g, 5, 70), torch.randn(9, 5, generator=g)
    Q = tb.mx_quantize(W)
    a, w = om.quantize(A)[0], om.quantize(W)[0]
    for x in (A, tb.mx_quantize(A)):
        D = tb.mx_gemm(1.5, x, Q, 0.5, C, dtype=torch.float32)
        assert og.excess(D, *om.product(1.5, a, w, None, 0.5, C), 70) <= 1
    assert tb.mx_gemm(1.0, tb.mx_quantize(A), Q).dtype == torch.bfloat16
    assert tb.mx_gemm(1.0, A.half(), Q).dtype == torch.float16
    E = _wide(g, 3, 5, 70)
    off = torch.tensor([1, 4, 4, 8])
    D = tb.mx_grouped_gemm(1.0, A, tb.mx_quantize(E), off)
    assert og.excess(D, *om.product(1.0, a, om.quantize(E)[0], off), 70) <= 1
    assert not D[0].any() and not D[8].any()


def test_refusals():
    A, W = torch.zeros(4, 64), tb.mx_quantize(torch.zeros(3, 64))
    E = tb.mx_quantize(torch.zeros(2, 3, 64))
    off = torch.tensor([0, 1, 4])
    with pytest.raises(TypeError, match="floating"):
        tb.mx_quantize(torch.zeros(2, 2, dtype=torch.int32))
    with pytest.raises(ValueError, match="2-D or 3-D"):
        tb.mx_quantize(torch.zeros(5))
    with pytest.raises(TypeError, match="dtype"):
        W.dequantize(torch.float64)
    with pytest.raises(ValueError, match="MXMatrix"):
        tb.mx_gemm(1.0, A, torch.zeros(3, 64))
    with pytest.raises(ValueError, match="3 dimensions"):
        tb.mx_grouped_gemm(1.0, A, W, off)
    with pytest.raises(ValueError, match="inner dimensions"):
        tb.mx_gemm(1.0, torch.zeros(4, 32), W)
    with pytest.raises(TypeError, match="float64"):
        tb.mx_gemm(1.0, A.double(), W)
    with pytest.raises(NotImplementedError, match="no gradient"):
        tb.mx_gemm(1.0, A.requires_grad_(), W)
    A = A.detach()
    with pytest.raises(ValueError, match="need 3 offsets"):
        tb.mx_grouped_gemm(1.0, A, E, torch.tensor([0, 4]))
    with pytest.raises(ValueError, match="offsets"):
        tb.mx_grouped_gemm(1.0, A, E, None)
    with pytest.raises(ValueError, match="needs C"):
        tb.mx_gemm(1.0, A, W, 1.0)
    with pytest.raises(TypeError, match="result dtype"):
        tb.mx_gemm(1.0, A, W, dtype=torch.float64)
    with pytest.raises(ValueError, match="codes must be"):
        tb.MXMatrix(W.codes[:2], W.scales, W.shape)
    with pytest.raises(ValueError, match="block_scales"):
        tb.MXMatrix.from_parts(W.codes, torch.zeros(3, 3, dtype=torch.uint8), 64)


def test_tangents_are_refused():
    from torch.autograd import forward_ad as fwd

    A, C = torch.ones(4, 64), torch.ones(4, 3)
    W, E, off = tb.mx_quantize(torch.ones(3, 64)), tb.mx_quantize(torch.ones(2, 3, 64)), torch.tensor([0, 1, 4])
    with fwd.dual_level():
        dual, c = fwd.make_dual(A, A), fwd.make_dual(C, C)
        for call in (lambda: tb.mx_gemm(1.0, dual, W), lambda: tb.mx_grouped_gemm(1.0, dual, E, off),
                     lambda: tb.mx_gemm(1.0, A, W, 1.0, c), lambda: tb.mx_grouped_gemm(1.0, A, E, off, 1.0, c)):  # fmt: skip
            with pytest.raises(NotImplementedError, match="no gradient"):
                call()
        assert torch.equal(tb.mx_gemm(1.0, A, W), torch.full((4, 3), 64.0))


def test_c_abi_refusals():
    from trnblas_amd.hip import _lib

    if not _lib.LIB_PATH.exists():
        pytest.skip("library not built")
    lib = _lib.load()
    p = 4096  # never dereferenced: every call fails its argument checks
    err = lib.trnblas_hip_last_error
    assert lib.trnblas_hip_mx_quantize(3, 4, 64, p, 64, 1, 0, p, p, 1, None) == _lib.E_ARG and b"dtype" in err()
    assert lib.trnblas_hip_mx_quantize(0, 4, 64, p, -1, 1, 0, p, p, 1, None) == _lib.E_ARG and b"stride" in err()
    assert lib.trnblas_hip_mx_quantize(0, 4, 64, p, 64, 1, 0, p + 4, p, 1, None) == _lib.E_ARG and b"aligned" in err()
    assert lib.trnblas_hip_mx_quantize(0, 1 << 30, 1 << 20, p, 1 << 20, 1, 0, p, p, 1, None) == _lib.E_ARG
    assert lib.trnblas_hip_mx_quantize(0, 0, 64, p, 64, 1, 0, p, p, 1, None) == 0
    assert lib.trnblas_hip_mx_dequantize(0, 4, 64, p, p, p, 63, 0, 1, None) == _lib.E_ARG and b"leading" in err()
    rc = lib.trnblas_hip_mx_gemm(1, 2, 4, 8, 64, 1.0, p, p, p, p, None, 0, 0.0, None, 8, p, 8, None)
    assert rc == _lib.E_ARG and b"offsets" in err()
    rc = lib.trnblas_hip_mx_gemm(1, 1, 4, 8, 64, 1.0, p, p, p, p + 8, None, 0, 0.0, None, 8, p, 8, None)
    assert rc == _lib.E_ARG and b"aligned" in err()
    rc = lib.trnblas_hip_mx_gemm(1, 1, 4, 8, 64, 1.0, p, p, p, p, None, 0, 1.0, None, 8, p, 8, None)
    assert rc == _lib.E_ARG and b"without C" in err()
