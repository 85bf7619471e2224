"""gated_gemm / grouped_gated_gemm on host tensors: values, gradients against differences, refusals."""

import pytest
import torch

import trnblas_amd as tb
from oracle import gated as og


def _offsets(*o, dtype=torch.int32):
    return torch.tensor(o, dtype=dtype)


@pytest.mark.parametrize("act", og.ACTS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("transB", [False, True])
def test_values(dtype, transB, act):
    g = torch.Generator().manual_seed(0)
    A = torch.randn(20, 9, generator=g).to(dtype)
    B = torch.randn(4, *((14, 9) if transB else (9, 14)), generator=g).to(dtype)
    off = _offsets(1, 4, 4, 17, 18)  # rows 0, 18, 19 of no group, group 1 empty
    H = tb.grouped_gated_gemm(A, B, off, act, transB=transB)
    P, den = og.products(A, B, off, transB)
    assert H.dtype == dtype and H.shape == (20, 7)
    assert og.ratio(H, *og.forward(act, P, den, 9, dtype)) <= 1 and not H[18:].any() and not H[0].any()
    H = tb.gated_gemm(A, B[2], act, transB=transB, dtype=torch.float32)
    P, den = og.products(A, B[2:3], _offsets(0, 20), transB)
    assert H.dtype == torch.float32 and og.ratio(H, *og.forward(act, P, den, 9, torch.float32)) <= 1


@pytest.mark.parametrize("act", og.ACTS)
def test_gradients_against_differences(act):
    g = torch.Generator().manual_seed(1)
    off = _offsets(0, 3, 3, 6, dtype=torch.int64)
    A, B = (torch.randn(s, generator=g, dtype=torch.float64, requires_grad=True) for s in ((7, 4), (3, 4, 10)))
    check = torch.autograd.gradcheck
    assert check(lambda a, b: tb.grouped_gated_gemm(a, b, off, act), (A, B), check_forward_ad=True)
    assert check(lambda a, b: tb.grouped_gated_gemm(a, b.mT.contiguous(), off, act, transB=True), (A, B))
    assert check(lambda a, b: tb.gated_gemm(a, b[1], act), (A, B), check_forward_ad=True)
    assert check(lambda a, b: tb.gated_gemm(a, b[1].mT.contiguous(), act, True), (A, B))
    one = torch.randn(4, 10, generator=g, dtype=torch.float64, requires_grad=True)
    assert check(lambda a, b: tb.grouped_gated_gemm(a, b.expand(3, 4, 10), off, act), (A, one))
    if act != "relu":  # differences across its kink say nothing
        assert torch.autograd.gradgradcheck(lambda a, b: tb.grouped_gated_gemm(a, b, off, act), (A, B))
        assert torch.autograd.gradgradcheck(lambda a, b: tb.gated_gemm(a, b[0], act), (A, B))


@pytest.mark.parametrize("which", [0, 1])
def test_gradient_of_one_operand_alone(which):
    g = torch.Generator().manual_seed(2)
    X = [torch.randn(5, 6, generator=g, dtype=torch.float64), torch.randn(6, 8, generator=g, dtype=torch.float64)]
    X[which].requires_grad_()
    assert torch.autograd.gradcheck(lambda x: tb.gated_gemm(*(x if i == which else X[i] for i in (0, 1))), (X[which],))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gradient_of_an_fp32_result_is_not_rounded(dtype):
    # gradients past the range of fp16 and below it: rounded to 16 bits they would be infinite, or nothing
    g = torch.Generator().manual_seed(12)
    A, B = (torch.randn(40, 24, generator=g) * 1e-3).to(dtype), (torch.randn(1, 24, 32, generator=g) * 2e-3).to(dtype)
    dH = torch.randn(40, 16, generator=g) * torch.tensor([1e9, 1e-3]).repeat_interleave(20)[:, None]
    a, b = A.clone().requires_grad_(), B[0].clone().requires_grad_()
    dA, dB = torch.autograd.grad(tb.gated_gemm(a, b, dtype=torch.float32), (a, b), dH)
    P, _ = og.products(A, B, _offsets(0, 40))
    dP = og.backward("silu", P, dH)
    want = dP @ B[0].double().T, A.double().T @ dP
    assert dA.dtype == dB.dtype == dtype
    for got, ref, den in zip((dA, dB), want, (dP.abs() @ B[0].double().abs().T, A.double().abs().T @ dP.abs())):
        assert ((got.double() - ref).abs() <= og.EPS[dtype] * ref.abs() + 1e-5 * den + 2 * og.TINY[dtype]).all()


def test_activations_far_from_zero():
    # finite values and slopes at the ends of the range, NaN where the argument is one
    x = torch.tensor([-3e38, -1e20, -700.0, -90.0, -20.0, 0.0, 20.0, 90.0, 700.0, 1e20, 3e38])
    for act in og.ACTS:
        A, B = x[:, None], torch.tensor([[1.0, 0.0]])
        up = torch.cat([torch.ones_like(A), A], 1)[:, [1, 0]]  # columns (x, 1)
        B = torch.eye(2)
        a = up.clone().requires_grad_()
        H = tb.gated_gemm(a, B, act)
        ref = og.gate(act, x.double())[0]
        assert torch.allclose(H.detach()[:, 0].double(), ref, rtol=1e-5, atol=1e-30)


def test_sizes_of_zero():
    off = _offsets(0, 0, 0)
    assert tb.grouped_gated_gemm(torch.zeros(0, 4), torch.zeros(2, 4, 6), off).shape == (0, 3)
    H = tb.grouped_gated_gemm(torch.zeros(5, 0), torch.zeros(2, 0, 6), _offsets(0, 2, 5))
    assert H.shape == (5, 3) and not H.any()
    assert tb.grouped_gated_gemm(torch.zeros(3, 4), torch.zeros(0, 4, 6), _offsets(0)).shape == (3, 3)
    assert tb.gated_gemm(torch.zeros(3, 4), torch.zeros(4, 0)).shape == (3, 0)
    assert tb.gated_gemm(torch.zeros(0, 4), torch.zeros(4, 2)).shape == (0, 1)


def test_refusals():
    A, B, off = torch.zeros(6, 4), torch.zeros(2, 4, 6), _offsets(0, 2, 6)
    with pytest.raises(ValueError, match="inner dimensions"):
        tb.grouped_gated_gemm(A, B, off, transB=True)
    with pytest.raises(ValueError, match="as many again"):
        tb.gated_gemm(A, B[0, :, :5])
    with pytest.raises(ValueError, match="activation"):
        tb.gated_gemm(A, B[0], "swish")
    with pytest.raises(ValueError, match="activation"):
        tb.gated_gemm(A, B[0], None)
    with pytest.raises(ValueError, match="2-D"):
        tb.gated_gemm(A, B)
    with pytest.raises(ValueError, match="3-D"):
        tb.grouped_gated_gemm(A, B[0], off)
    with pytest.raises(ValueError, match="need 3 offsets"):
        tb.grouped_gated_gemm(A, B, _offsets(0, 6))
    with pytest.raises(ValueError, match="1-D"):
        tb.grouped_gated_gemm(A, B, None)
    with pytest.raises(TypeError, match="mixed dtypes"):
        tb.gated_gemm(A.bfloat16(), B[0])
    with pytest.raises(TypeError, match="floating"):
        tb.gated_gemm(A.int(), B[0].int())
    with pytest.raises(TypeError, match="result dtype"):
        tb.gated_gemm(A, B[0], dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="transB"):
        tb.gated_gemm(A, B[0], transB="x")


def test_c_abi_refusals():
    from trnblas_amd.hip import _lib

    if not _lib.LIB_PATH.exists():
        pytest.skip("library not built")
    lib = _lib.load()

    # the pointers are never dereferenced: every call fails its argument checks
    def gate(act=0, dtype=1, out=1, rows=6, n=8, p=4096, ldp=16, ldh=8, s=None, lds=16):
        return lib.trnblas_hip_gate(act, dtype, out, rows, n, p, ldp, 4096, ldh, s, lds, None)

    for bad, word in ((dict(act=5), b"activation"), (dict(act=-1), b"activation"), (dict(dtype=3), b"dtype"),
                      (dict(out=0), b"result dtype"), (dict(rows=-1), b"sizes"), (dict(n=1 << 30), b"sizes"),
                      (dict(ldp=15), b"leading"), (dict(ldh=7), b"leading"), (dict(s=4096, lds=15), b"leading"),
                      (dict(p=None), b"null")):  # fmt: skip
        assert gate(**bad) == _lib.E_ARG and word in lib.trnblas_hip_last_error(), bad
    assert gate(rows=0) == 0 and gate(n=0, ldp=0) == 0

    def back(act=0, dtype=1, rows=6, n=8, ldp=16, ldg=8, d=4096, ldd=16):
        return lib.trnblas_hip_gate_backward(act, dtype, rows, n, 4096, ldp, 4096, ldg, d, ldd, None)

    for bad, word in ((dict(act=9), b"activation"), (dict(dtype=7), b"dtype"), (dict(ldg=7), b"leading"),
                      (dict(ldd=15), b"leading"), (dict(d=None), b"null")):  # fmt: skip
        assert back(**bad) == _lib.E_ARG and word in lib.trnblas_hip_last_error(), bad
    assert back(rows=0) == 0

    def product(act=0, dtype=1, groups=2, rows=6, n=8, k=16, a=4096, lda=16, b=4096, ldb=16, sb=128, su=8, off=4096, h=4096, ldh=8,
                p=None, ldp=16):  # fmt: skip
        return lib.trnblas_hip_gated_gemm(act, dtype, 0, groups, rows, n, k, a, lda, b, ldb, sb, su, off, 0, h, ldh, p, ldp, 0, None)

    for bad, word in ((dict(act=5), b"activation"), (dict(dtype=3), b"dtype"), (dict(groups=-1), b"sizes"), (dict(rows=1 << 31), b"sizes"),
                      (dict(k=1 << 31), b"sizes"), (dict(lda=15), b"leading"), (dict(ldb=7), b"leading"), (dict(su=-8), b"leading"),
                      (dict(ldh=7), b"leading"), (dict(p=4096, ldp=15), b"leading"), (dict(off=None), b"offsets"),
                      (dict(off=4098), b"offsets"), (dict(a=None), b"null"), (dict(h=None), b"null"), (dict(a=4098), b"16 bytes"),
                      (dict(lda=17), b"16 bytes"), (dict(su=9), b"16 bytes"), (dict(sb=129), b"16 bytes"), (dict(k=15), b"16 bytes"),
                      (dict(n=7), b"16 bytes")):  # fmt: skip
        assert product(**bad) == _lib.E_ARG and word in lib.trnblas_hip_last_error(), bad
    assert product(rows=0) == 0 and product(n=0) == 0
    for bad in ((3, 0, 1, 6, 8, 8), (1, 0, 0, 6, 8, 8), (1, 0, 1, 0, 8, 8), (1, 0, 1, 6, 0, 8), (1, 0, 1, 6, 8, -1)):
        assert lib.trnblas_hip_gated_plan(*bad) is None and b"bad arguments" in lib.trnblas_hip_last_error()


@pytest.mark.parametrize("source", ["gated_bf16.hip", "gated_f16.hip"])
def test_wait_states_before_matrix_instructions(source):
    from test_wait_states_host import _assembly, hazards

    r = _assembly(source)
    assert r.returncode == 0, r.stderr
    assert "v_mfma" in r.stdout and not hazards(r.stdout)
