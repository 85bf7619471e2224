"""4-bit integer weights on host tensors: codes and scales by the definition, products, layout, refusals."""

import pytest
import torch

import trnblas_amd as tb
from oracle import gated as oa
from oracle import grouped as og
from oracle import int4 as oi

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _same(Q, X, group, zeros, scale_dtype):
    W, q, s, z = oi.quantize(X, group, zeros, scale_dtype)
    V = Q.dequantize().double().cpu()
    W = W.float().double()  # past the largest number: a scale rounded up, times fifteen
    assert torch.equal(V.isnan(), W.isnan()) and torch.equal(V.nan_to_num(-1.0), W.nan_to_num(-1.0))
    codes, scales, z2 = (None if t is None else t.cpu() for t in Q.parts())
    assert scales.dtype == scale_dtype and torch.equal(scales.double().nan_to_num(-1.0), s.nan_to_num(-1.0))
    assert (z2 is None) == (not zeros) and (z2 is None or torch.equal(z2.double(), z))
    got = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)[..., : X.shape[-1]]
    assert torch.equal(got.double(), q)


@pytest.mark.parametrize("scale_dtype", [BF16, F16])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantize(group, zeros, scale_dtype):
    for i, shape in enumerate([(1, 1), (3, 32), (17, 33), (16, 128), (40, 300), (2, 19, 70)]):
        for dtype in (F32, BF16, F16):
            X = oi.wide(torch.Generator().manual_seed(i), *shape, dtype=dtype)
            Q = tb.int4_quantize(X, group, zeros, scale_dtype=scale_dtype)
            assert Q.shape == X.shape and Q.group == group
            _same(Q, X, group, zeros, scale_dtype)
            T = tb.int4_quantize(X.mT.contiguous(), group, zeros, trans=True, scale_dtype=scale_dtype)
            assert torch.equal(T.codes, Q.codes) and torch.equal(T.scales, Q.scales)


@pytest.mark.parametrize("zeros", [False, True])
def test_values_at_the_ends(zeros):
    for dtype in (F32, BF16, F16):
        f = torch.finfo(dtype)
        X = torch.zeros(12, 96, dtype=dtype)
        X[0, 3], X[0, 40] = f.max, -f.max
        X[1, 0], X[1, 1], X[1, 33] = f.smallest_normal / 4, f.smallest_normal, f.smallest_normal / 2
        X[2, 5], X[3, 6], X[3, 70] = float("inf"), float("-inf"), float("nan")
        X[4, 1], X[5, 0], X[6, 0] = -0.0, 1.0, -1.0
        X[7], X[8] = 3.0, -3.0
        for scale_dtype in (BF16, F16):
            _same(tb.int4_quantize(X, 32, zeros, scale_dtype=scale_dtype), X, 32, zeros, scale_dtype)


@pytest.mark.parametrize("group", [32, 64, 128])
def test_layout_goes_there_and_back(group):
    g = torch.Generator().manual_seed(group)
    for shape in ((1, 1), (5, 33), (16, 128), (33, 257), (3, 18, 200)):
        for zeros in (False, True):
            Q, W = oi.random_matrix(g, *shape, group=group, zeros=zeros, scale_dtype=F16, z_max=255)
            assert torch.equal(Q.dequantize().double(), W)
            codes, scales, z = Q.parts()
            P = tb.Int4Matrix.from_parts(codes, scales, shape[-1], group, z)
            assert torch.equal(P.codes, Q.codes) and torch.equal(P.scales, Q.scales) and (z is None or torch.equal(P.zeros, Q.zeros))
            if len(shape) == 3:
                assert torch.equal(Q[2].dequantize().double(), W[2])
    # the layout itself, as include/trnblas_hip.h has it: value (r, k) of a matrix with one nibble set
    for r, k in ((0, 0), (3, 1), (17, 45), (31, 255), (20, 130), (9, 78)):
        codes = torch.full((32, 128), 0x88, dtype=torch.uint8)
        codes[r, k // 2] = 0x89 if k % 2 == 0 else 0x98
        Q = tb.Int4Matrix.from_parts(codes, torch.ones(32, 256 // group, dtype=BF16), 256, group)
        c, t, e = k // 128, k % 128, k % 8
        at, nibble = 16 * (16 * (t % 32 // 8) + r % 16) + 4 * (t // 32), e // 2 + 4 * (e % 2)
        want = torch.zeros(2, 2, 1024, dtype=torch.uint8)
        want[r // 16, c, at + nibble // 2] = 1 << 4 * (nibble % 2)
        assert torch.equal(Q.codes, want), (r, k)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_products(dtype):
    g = torch.Generator().manual_seed(1)
    off = og.split(30, [4, 0, 21, 2], 2)
    for zeros in (False, True):
        E, W = oi.random_matrix(g, 4, 20, 70, group=32, zeros=zeros, scale_dtype=BF16)
        A, C = torch.randn(30, 70, generator=g).to(dtype), torch.randn(30, 20, generator=g).to(dtype)
        D = tb.int4_grouped_gemm(-1.5, A, E, off, 0.5, C)
        assert D.dtype == dtype and og.excess(D, *oi.product(-1.5, A, W, off, 0.5, C), 70) <= 1
        D = tb.int4_gemm(2.0, A, E[2], 0.5, C[0])
        assert og.excess(D, *oi.product(2.0, A, W[2], None, 0.5, C[0]), 70) <= 1
        D = tb.int4_gemm(2.0, A, E[2], dtype=F32)
        assert D.dtype == F32 and og.excess(D, *oi.product(2.0, A, W[2]), 70) <= 1
        for act in oa.ACTS:
            H = tb.grouped_gated_gemm(A, E, off, act)
            P, den = oa.products(A, W, off, True)
            assert H.shape == (30, 10) and oa.ratio(H, *oa.forward(act, P, den, 70, dtype)) <= 1
            H = tb.gated_gemm(A, E[1], act, dtype=F32)
            P, den = oa.products(A, W[1:2], torch.tensor([0, 30]), True)
            assert H.dtype == F32 and oa.ratio(H, *oa.forward(act, P, den, 70, F32)) <= 1


def test_sizes_of_zero():
    for shape in ((0, 40), (5, 0), (0, 0)):
        Q = tb.int4_quantize(torch.zeros(shape))
        assert Q.shape == shape and Q.dequantize().shape == shape
        D = tb.int4_gemm(1.0, torch.ones(3, shape[1]), Q)
        assert D.shape == (3, shape[0]) and not D.any()
    Q = tb.int4_quantize(torch.ones(2, 4, 8))
    off = torch.tensor([0, 0, 0])
    assert tb.int4_grouped_gemm(1.0, torch.zeros(0, 8), Q, off).shape == (0, 4)
    assert not tb.int4_grouped_gemm(1.0, torch.ones(3, 8), Q, off).any()
    assert tb.grouped_gated_gemm(torch.ones(3, 8), Q, off).shape == (3, 2)


def test_refusals():
    X = torch.zeros(4, 64)
    Q = tb.int4_quantize(X)
    E = tb.int4_quantize(torch.zeros(2, 5, 64))
    off = torch.tensor([0, 1, 4])
    for call, error, match in (
        (lambda: tb.int4_quantize(X, 16), ValueError, "group"),
        (lambda: tb.int4_quantize(X, 64.0), ValueError, "group"),
        (lambda: tb.int4_quantize(X[0]), ValueError, "2-D or 3-D"),
        (lambda: tb.int4_quantize(X.int()), TypeError, "floating"),
        (lambda: tb.int4_quantize(X, scale_dtype=F32), TypeError, "scale_dtype"),
        (lambda: tb.int4_dequantize(X), TypeError, "Int4Matrix is needed"),
        (lambda: tb.int4_dequantize(Q, torch.float64), TypeError, "dtype"),
        (lambda: tb.int4_gemm(1.0, X, X), ValueError, "Int4Matrix of 2"),
        (lambda: tb.int4_gemm(1.0, X, E), ValueError, "Int4Matrix of 2"),
        (lambda: tb.int4_grouped_gemm(1.0, X, Q, off), ValueError, "Int4Matrix of 3"),
        (lambda: tb.int4_gemm(1.0, X[0], Q), ValueError, "2-D"),
        (lambda: tb.int4_gemm(1.0, X.double(), Q), TypeError, "A is"),
        (lambda: tb.int4_gemm(1.0, X[:, :63], Q), ValueError, "inner dimensions"),
        (lambda: tb.int4_gemm(1.0, X, Q, 1.0), ValueError, "needs C"),
        (lambda: tb.int4_gemm(1.0, X, Q, 1.0, torch.zeros(3, 4)), ValueError, "broadcast"),
        (lambda: tb.int4_gemm(1.0, X, Q, 1.0, torch.zeros(4, 4).half()), TypeError, "C is"),
        (lambda: tb.int4_gemm(1.0, X, Q, dtype=torch.float64), TypeError, "result dtype"),
        (lambda: tb.int4_gemm(1.0, X.clone().requires_grad_(), Q), NotImplementedError, "no gradient"),
        (lambda: tb.int4_gemm(1.0, X, Q, 1.0, torch.zeros(4, 4, requires_grad=True)), NotImplementedError, "no gradient"),
        (lambda: tb.int4_grouped_gemm(1.0, X, E, off[:2]), ValueError, "need 3 offsets"),
        (lambda: tb.int4_grouped_gemm(1.0, X, E, None), ValueError, "1-D"),
        (lambda: tb.grouped_gated_gemm(X, E, off), ValueError, "as many again"),
        (lambda: tb.grouped_gated_gemm(X, Q, off), ValueError, "Int4Matrix of 3"),
        (lambda: tb.gated_gemm(X, E), ValueError, "Int4Matrix of 2"),
        (lambda: tb.gated_gemm(X, Q, "tanh"), ValueError, "activation"),
        (lambda: tb.gated_gemm(X.clone().requires_grad_(), Q), NotImplementedError, "no gradient"),
        (lambda: Q[0], ValueError, "stack"),
        (lambda: tb.Int4Matrix(Q.codes, Q.scales, None, (4, 64), 64), ValueError, "scales must be"),
        (lambda: tb.Int4Matrix(Q.codes[..., :512], Q.scales, None, (4, 64), 128), ValueError, "codes must be"),
        (lambda: tb.Int4Matrix(Q.codes, Q.scales, Q.scales, (4, 64), 128), ValueError, "zeros must be"),
        (lambda: tb.Int4Matrix(Q.codes, Q.scales, None, (64,), 128), ValueError, "shape must be"),
        (lambda: tb.Int4Matrix.from_parts(torch.zeros(4, 31, dtype=torch.uint8), Q.scales, 64, 128), ValueError, "codes must be"),
        (lambda: tb.Int4Matrix.from_parts(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 1), 64, 128), ValueError, "scales must be"),
        (lambda: tb.Int4Matrix.from_parts(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 1).half(), 64, 128, torch.zeros(4, 1)), ValueError, "zeros must be"),
    ):  # fmt: skip
        with pytest.raises(error, match=match):
            call()
    from torch.autograd import forward_ad as fwd

    with fwd.dual_level():
        with pytest.raises(NotImplementedError, match="no gradient"):
            tb.int4_gemm(1.0, fwd.make_dual(X, X), Q)


def test_c_abi_refusals():
    from trnblas_amd.hip import _lib

    if not _lib.LIB_PATH.exists():
        pytest.skip("library not built")
    lib = _lib.load()

    # the pointers are never dereferenced: every call fails its argument checks
    def quant(dtype=1, st=1, r=5, k=70, group=64, x=4096, sr=70, codes=4096, scales=4096, zeros=None, batch=1):
        return lib.trnblas_hip_int4_quantize(dtype, st, r, k, group, x, sr, 1, 0, codes, scales, zeros, batch, None)

    for bad, word in ((dict(dtype=3), b"dtype"), (dict(st=0), b"scale dtype"), (dict(r=-1), b"sizes"), (dict(group=16), b"group"),
                      (dict(sr=-1), b"stride"), (dict(x=None), b"null"), (dict(codes=4104), b"aligned"), (dict(scales=4098), b"aligned"),
                      (dict(zeros=4097), b"aligned"), (dict(batch=65536), b"sizes")):  # fmt: skip
        assert quant(**bad) == _lib.E_ARG and word in lib.trnblas_hip_last_error(), bad
    assert quant(r=0) == 0 and quant(k=0) == 0 and quant(batch=0) == 0

    def dequant(dtype=1, ldd=70, d=4096):
        return lib.trnblas_hip_int4_dequantize(dtype, 1, 5, 70, 64, 4096, 4096, None, d, ldd, 350, 1, None)

    for bad, word in ((dict(dtype=9), b"dtype"), (dict(ldd=69), b"leading"), (dict(d=None), b"null")):
        assert dequant(**bad) == _lib.E_ARG and word in lib.trnblas_hip_last_error(), bad

    def gemm(dtype=1, out=1, gated=0, act=0, groups=1, rows=3, n=8, k=64, group=32, alpha=1.0, a=4096, sr=64, sk=1, codes=4096,
             scales=4096, zeros=None, st=1, off=None, beta=0.0, c=None, ldd=8, ws=None, size=0):  # fmt: skip
        return lib.trnblas_hip_int4_gemm(dtype, out, gated, act, groups, rows, n, k, group, alpha, a, sr, sk, codes, scales, zeros, st,
                                         off, 0, beta, c, 8, 4096, ldd, ws, size, None)  # fmt: skip

    for bad, word in ((dict(dtype=3), b"dtype"), (dict(out=3), b"result dtype"), (dict(gated=1, act=5), b"activation"),
                      (dict(gated=1, alpha=2.0), b"alpha"), (dict(gated=1, beta=1.0, c=4096), b"beta"), (dict(group=48), b"group"),
                      (dict(n=1 << 31), b"sizes"), (dict(k=(1 << 22) + 1, sr=1 << 23), b"sizes"), (dict(groups=2), b"offsets"), (dict(off=4098), b"offsets"), (dict(beta=1.0), b"without C"),
                      (dict(sk=-1), b"stride"), (dict(ldd=7), b"leading"), (dict(a=None), b"null"), (dict(codes=8), b"aligned")):  # fmt: skip
        assert gemm(**bad) == _lib.E_ARG and word in lib.trnblas_hip_last_error(), bad
    # rows that are not read in place need a workspace
    need = lib.trnblas_hip_int4_gemm_workspace(0, 0, 1, 3, 8, 64, 32)
    assert need == 3 * 128 * 2 * 3 and lib.trnblas_hip_int4_gemm_workspace(1, 0, 1, 3, 8, 130, 64) == 3 * 256 * 2
    assert lib.trnblas_hip_int4_gemm_workspace(1, 0, 1, 0, 8, 130, 64) == 0
    for how in (dict(dtype=0), dict(sk=2), dict(a=4098), dict(sr=65)):
        assert gemm(**how) == _lib.E_WORKSPACE and b"workspace" in lib.trnblas_hip_last_error(), how
    assert gemm(dtype=0, ws=4096, size=need - 1) == _lib.E_WORKSPACE and gemm(dtype=0, ws=4104, size=need) == _lib.E_WORKSPACE
    assert gemm(rows=0) == 0 and gemm(n=0, ldd=0) == 0
