"""grouped_gemm / grouped_rank_k on host tensors: values, gradients against differences, refusals."""

import pytest
import torch

import trnblas_amd as tb
from oracle import grouped as og


def _offsets(*o, dtype=torch.int32):
    return torch.tensor(o, dtype=dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("transB", [False, True])
def test_values(dtype, transB):
    g = torch.Generator().manual_seed(0)
    A = torch.randn(20, 9, generator=g).to(dtype)
    B = torch.randn(4, *((5, 9) if transB else (9, 5)), generator=g).to(dtype)
    C = torch.randn(20, 5, generator=g).to(dtype)
    off = _offsets(1, 4, 4, 17, 18)  # rows 0, 18, 19 of no group, group 1 empty
    D = tb.grouped_gemm(1.5, A, B, off, 0.5, C, transB=transB)
    ref, den = og.grouped_gemm(1.5, A, B, off, 0.5, C, transB)
    assert D.dtype == dtype and og.excess(D, ref, den, 9) <= 1
    W = torch.randn(20, 5, generator=g).to(dtype)
    P = tb.grouped_rank_k(2.0, A, W, off, dtype=torch.float32)
    ref, den = og.grouped_rank_k(2.0, A, W, off)
    assert P.dtype == torch.float32 and og.excess(P, ref, den, 20) <= 1
    assert not P[1].any()


def test_gradients_against_differences():
    g = torch.Generator().manual_seed(1)
    off = _offsets(0, 3, 3, 6, dtype=torch.int64)
    A, B, C = (torch.randn(s, generator=g, dtype=torch.float64, requires_grad=True) for s in ((7, 4), (3, 4, 5), (7, 5)))
    W = torch.randn(7, 5, generator=g, dtype=torch.float64, requires_grad=True)
    row = torch.randn(5, generator=g, dtype=torch.float64, requires_grad=True)
    assert torch.autograd.gradcheck(lambda a, b, c: tb.grouped_gemm(0.7, a, b, off, 0.3, c), (A, B, C))
    # C broadcast over the rows, B given transposed, and a view of one matrix for all groups
    assert torch.autograd.gradcheck(
        lambda a, b, c: tb.grouped_gemm(0.7, a, b.mT.contiguous(), off, 0.3, c, transB=True), (A, B, row)
    )
    one = torch.randn(4, 5, generator=g, dtype=torch.float64, requires_grad=True)
    assert torch.autograd.gradcheck(lambda a, b: tb.grouped_gemm(1.0, a, b.expand(3, 4, 5), off), (A, one))
    acc = torch.randn(3, 4, 5, generator=g, dtype=torch.float64, requires_grad=True)
    assert torch.autograd.gradcheck(lambda a, w, c: tb.grouped_rank_k(0.7, a, w, off, 1.0, c), (A, W, acc))
    assert torch.autograd.gradgradcheck(lambda a, b: tb.grouped_gemm(0.7, a, b, off), (A, B))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gradient_of_an_fp32_result_is_not_rounded(dtype):
    # its values pass the range of fp16 and fall below it, and have more bits than a 16-bit type holds
    rows, K, N = 60, 24, 40
    off = _offsets(0, 9, 30, 30, 55)
    g = torch.Generator().manual_seed(12)
    A, B = (torch.randn(rows, K, generator=g) * 1e-3).to(dtype), (torch.randn(4, K, N, generator=g) * 2e-3).to(dtype)
    dD = torch.randn(rows, N, generator=g) * torch.tensor([1e5, 1e-5]).repeat_interleave(rows // 2)[:, None]
    for transB in (False, True):
        b0 = B.mT.contiguous() if transB else B
        a, b = A.clone().requires_grad_(), b0.clone().requires_grad_()
        D = tb.grouped_gemm(2.0, a, b, off, transB=transB, dtype=torch.float32)
        dA, dB = torch.autograd.grad(D, (a, b), dD)
        assert dA.dtype == dB.dtype == dtype
        assert og.excess(dA, *og.grouped_gemm(2.0, dD, b0, off, transB=not transB), N) <= 1
        assert og.excess(dB, *og.grouped_rank_k(2.0, *((dD, A) if transB else (A, dD)), off), rows) <= 1
    W, dP = (torch.randn(rows, N, generator=g) * 1e-3).to(dtype), torch.randn(4, K, N, generator=g) * 1e5
    a, w = A.clone().requires_grad_(), W.clone().requires_grad_()
    dA, dW = torch.autograd.grad(tb.grouped_rank_k(1.0, a, w, off, dtype=torch.float32), (a, w), dP)
    assert og.excess(dA, *og.grouped_gemm(1.0, W, dP.mT, off), N) <= 1
    assert og.excess(dW, *og.grouped_gemm(1.0, A, dP, off), K) <= 1


def _products(off):
    return (
        lambda a, b, c, w, s: tb.grouped_gemm(0.7, a, b, off, 0.3, c),
        lambda a, b, c, w, s: tb.grouped_gemm(0.7, a, b.mT.contiguous(), off, 0.3, c, transB=True),
        lambda a, b, c, w, s: tb.grouped_rank_k(0.7, a, w, off, 0.5, s),
    )


def test_tangents_against_differences():
    g = torch.Generator().manual_seed(3)
    off = _offsets(0, 3, 3, 6)
    args = tuple(torch.randn(s, generator=g, dtype=torch.float64, requires_grad=True)
                 for s in ((7, 4), (3, 4, 5), (7, 5), (7, 5), (3, 4, 5)))  # fmt: skip
    for f in _products(off):
        used = lambda *x, f=f: f(*x) + 0.0 * sum(v.sum() for v in x)
        assert torch.autograd.gradcheck(used, args, check_forward_ad=True, check_backward_ad=False)
        assert torch.autograd.gradgradcheck(used, args, check_fwd_over_rev=True, check_rev_over_rev=False, check_undefined_grad=False)


def test_tangents_of_each_operand_alone():
    from torch.autograd import forward_ad as fwd

    g = torch.Generator().manual_seed(4)
    off = _offsets(1, 3, 3, 6)
    X = [torch.randn(s, generator=g, dtype=torch.float64) for s in ((7, 4), (3, 4, 5), (7, 5), (7, 5), (3, 4, 5))]
    T = [torch.randn(x.shape, generator=g, dtype=torch.float64) for x in X]
    for f in _products(off):
        for i in range(5):
            step = lambda h: f(*(x + h * t if i == j else x for j, (x, t) in enumerate(zip(X, T))))
            with fwd.dual_level():
                got = fwd.unpack_dual(f(*(fwd.make_dual(x, t) if i == j else x for j, (x, t) in enumerate(zip(X, T)))))
                got = got.tangent
            # the products are linear in each operand: a difference is exact but for rounding
            assert (got is None) == torch.equal(step(1.0), step(-1.0))
            if got is not None:
                assert torch.allclose(got, (step(1.0) - step(-1.0)) / 2, rtol=0, atol=1e-13)


def test_sizes_of_zero():
    off = _offsets(0, 0, 0)
    assert tb.grouped_gemm(1.0, torch.zeros(0, 4), torch.zeros(2, 4, 3), off).shape == (0, 3)
    D = tb.grouped_gemm(1.0, torch.zeros(5, 0), torch.zeros(2, 0, 3), _offsets(0, 2, 5))
    assert D.shape == (5, 3) and not D.any()
    assert tb.grouped_rank_k(1.0, torch.zeros(0, 4), torch.zeros(0, 3), off).shape == (2, 4, 3)
    assert tb.grouped_gemm(1.0, torch.zeros(3, 4), torch.zeros(0, 4, 3), _offsets(0)).shape == (3, 3)


def test_refusals():
    A, B, off = torch.zeros(6, 4), torch.zeros(2, 4, 3), _offsets(0, 2, 6)
    with pytest.raises(ValueError, match="inner dimensions"):
        tb.grouped_gemm(1.0, A, B, off, transB=True)
    with pytest.raises(ValueError, match="need 3 offsets"):
        tb.grouped_gemm(1.0, A, B, _offsets(0, 6))
    with pytest.raises(TypeError, match="int32 or int64"):
        tb.grouped_gemm(1.0, A, B, off.float())
    with pytest.raises(ValueError, match="1-D"):
        tb.grouped_gemm(1.0, A, B, [0, 2, 6])
    with pytest.raises(TypeError, match="mixed dtypes"):
        tb.grouped_gemm(1.0, A.bfloat16(), B, off)
    with pytest.raises(TypeError, match="floating"):
        tb.grouped_gemm(1.0, A.int(), B.int(), off)
    with pytest.raises(ValueError, match="3-D"):
        tb.grouped_gemm(1.0, A, B[0], off)
    with pytest.raises(ValueError, match="needs C"):
        tb.grouped_gemm(1.0, A, B, off, beta=1.0)
    with pytest.raises(ValueError, match="broadcast"):
        tb.grouped_gemm(1.0, A, B, off, 1.0, torch.zeros(5, 3))
    with pytest.raises(TypeError, match="C is"):
        tb.grouped_gemm(1.0, A, B, off, 1.0, torch.zeros(6, 3).double())
    with pytest.raises(TypeError, match="result dtype"):
        tb.grouped_gemm(1.0, A, B, off, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="rows"):
        tb.grouped_rank_k(1.0, A, torch.zeros(5, 3), off)
    with pytest.raises(ValueError, match="transB"):
        tb.grouped_gemm(1.0, A, B, off, transB="x")


def test_c_abi_refusals():
    from trnblas_amd.hip import _lib

    if not _lib.LIB_PATH.exists():
        pytest.skip("library not built")
    lib = _lib.load()

    def gemm(dtype=0, groups=2, rows=6, n=3, k=4, lda=4, ldb=3, off=4096, beta=0.0, c=None, ldd=3):
        # the pointers are never dereferenced: every call fails its argument checks
        return lib.trnblas_hip_grouped_gemm(dtype, 0, 0, groups, rows, n, k, 1.0, 4096, lda, 4096, ldb, 12, off, 0, beta, c,
                                            3, 4096, ldd, 0, None)  # fmt: skip

    for bad, word in ((dict(dtype=7), b"dtype"), (dict(rows=-1), b"sizes"), (dict(groups=1 << 24), b"sizes"),
                      (dict(lda=3), b"leading"), (dict(ldd=2), b"leading"), (dict(off=None), b"offsets"),
                      (dict(off=4098), b"offsets"), (dict(beta=1.0), b"without C"), (dict(k=1 << 31), b"sizes")):  # fmt: skip
        assert gemm(**bad) == _lib.E_ARG and word in lib.trnblas_hip_last_error(), bad
    assert gemm(rows=0) == 0  # nothing to do
    rc = lib.trnblas_hip_grouped_rank_k(1, 0, 2, 6, 4, 3, 1.0, 4096, 3, 4096, 3, 4096, 0, 0.0, None, 3, 0, 4096, 3, 12, 0, None)
    assert rc == _lib.E_ARG and b"leading" in lib.trnblas_hip_last_error()


def test_rows_plan_refusals():
    import ctypes

    from trnblas_amd.hip import _lib

    if not _lib.LIB_PATH.exists():
        pytest.skip("library not built")
    lib = _lib.load()
    out = (ctypes.c_int32 * 3)(7, 7, 7)
    for bad in ((1, 1, 0, 2, 6, 4, 3), (3, 1, 0, 2, 6, 4, 3), (0, 3, 0, 2, 6, 4, 3), (0, 1, 0, 0, 6, 4, 3), (0, 1, 0, 2, 6, 0, 3)):
        assert lib.trnblas_hip_grouped_rows_plan(*bad, out) == _lib.E_ARG and b"bad arguments" in lib.trnblas_hip_last_error()
    assert lib.trnblas_hip_grouped_rows_plan(0, 1, 0, 2, 6, 64, 64, None) == _lib.E_ARG
    assert lib.trnblas_hip_grouped_rows_plan(0, 1, 0, 1, 30000, 4096, 4096, out) == 0 and not any(out)


def test_the_plan_asks_for_forms_that_exist():
    # fewer than eight waves along K: one row block of a K-contiguous 16-bit matrix; wide short matrices of many groups came to
    # one wave elsewhere, and eight ran
    from oracle.grouped import rows_plan
    from trnblas_amd.hip import _lib

    if not _lib.LIB_PATH.exists():
        pytest.skip("library not built")
    seen = set()
    for G in (1, 5, 16, 50, 64):
        for R in sorted({G, 2 * G + 6, 8 * G, 18 * G + 7, 40 * G}):
            for N in (72, 520, 2056, 28376, 32160):
                for K in (40, 96, 520, 2056):
                    for transB in (0, 1):
                        blocks, waves, inside = rows_plan(0, torch.bfloat16, transB, G, R, N, K)
                        assert not inside and (waves in (0, 8) or (blocks == 1 and transB))
                        seen.add((blocks, waves, transB))
    assert {(1, 8, 0), (2, 8, 0), (1, 1, 1), (1, 2, 1), (1, 4, 1), (1, 8, 1), (2, 8, 1)} <= seen


def test_the_fp32_plan_follows_fp32_costs():
    # few rows: the weights straight into registers, not a tile per CU; large products: the ring kernel; between them 32 x 64 tiles
    from oracle.grouped import plan, rows_plan
    from trnblas_amd.hip import _lib

    if not _lib.LIB_PATH.exists():
        pytest.skip("library not built")
    f32 = torch.float32
    for transB in (0, 1):
        for G, R, N, K in ((2, 32, 1536, 4096), (64, 64, 1024, 4096), (1, 1, 8192, 4096)):
            want = "rows_kernel" if G < 64 or not transB else "grouped_any_kernel"
            assert plan(0, f32, transB, G, R, 0, N, K) == want, (transB, G, R, N, K)
        for G, R, N, K in ((16, 512, 4096, 2048), (64, 2048, 1536, 2056), (64, 1024, 2048, 1024)):
            assert plan(0, f32, transB, G, R, 0, N, K) == "grouped_any_kernel", (transB, G, R, N, K)
        for G, R, N, K in ((4, 8192, 4096, 2048), (1, 4096, 1024, 4096)):
            assert plan(0, f32, transB, G, R, 0, N, K) == "ring_kernel 64 x 128", (transB, G, R, N, K)
    assert plan(1, f32, 0, 8, 4096, 2048, 2048, 0) == "ring_kernel 64 x 128"
    for G in (1, 6, 12, 20, 33):
        for R in (G, 8 * G, 24 * G):
            for N in (520, 856, 3028, 18400):
                for K in (40, 132, 1412, 3052):
                    for transB in (0, 1):
                        blocks, waves, _ = rows_plan(0, f32, transB, G, R, N, K)
                        assert (blocks, waves) in ((0, 0), (1, 8)) or (transB and (blocks, waves) in ((1, 4), (1, 1)))
