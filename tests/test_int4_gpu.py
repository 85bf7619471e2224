"""4-bit integer weights on the GPU: codes and scales equal to the definition's, products within what fp32 sums allow."""

import pytest
import torch

import trnblas_amd as tb
from oracle import gated as oa
from oracle import grouped as og
from oracle import int4 as oi
from oracle.grouped import GROUPS
from oracle.grouped import split as _split
from test_int4_host import _same

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
DTYPES = [F32, BF16, F16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantize(dev, group, zeros, dtype):
    for i, shape in enumerate([(1, 1), (1, 4096), (3, 32), (17, 33), (16, 512), (64, 128), (130, 1032), (2, 19, 70), (3, 65, 520), (257, 130)]):
        X = oi.wide(torch.Generator().manual_seed(i), *shape, dtype=dtype)
        scale_dtype = (BF16, F16)[i % 2]
        how = dict(group=group, zeros=zeros, scale_dtype=scale_dtype)
        Q = tb.int4_quantize(X.to(dev), **how)
        _same(Q, X, group, zeros, scale_dtype)
        H = tb.int4_quantize(X, **how)  # on the host: the same buffers, what lies outside the matrix included
        assert torch.equal(H.codes, Q.codes.cpu()) and torch.equal(H.scales.view(torch.int16), Q.scales.cpu().view(torch.int16))
        assert not zeros or torch.equal(H.zeros, Q.zeros.cpu())
        P = torch.full((*X.shape[:-1], X.shape[-1] + 5), float("nan"), dtype=dtype, device=dev)
        P[..., 3:-2] = X
        T = torch.full((*X.shape[:-2], X.shape[-1], X.shape[-2] + 7), float("nan"), dtype=dtype, device=dev)
        T[..., 1:-6] = X.mT
        for Y, trans in ((X.mT.contiguous().to(dev), True), (P[..., 3:-2], False), (T[..., 1:-6], True),
                         (torch.stack([X, X * 0 + 9], -1).to(dev)[..., 0], False)):  # fmt: skip
            S = tb.int4_quantize(Y, trans=trans, **how)
            assert torch.equal(S.codes, Q.codes) and torch.equal(S.scales.view(torch.int16), Q.scales.view(torch.int16))
            assert not zeros or torch.equal(S.zeros, Q.zeros)


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_values_at_the_ends(dev, dtype, trans, zeros):
    f = torch.finfo(dtype)
    X = torch.zeros(70, 160, dtype=dtype)
    X[0, 3], X[0, 40] = f.max, -f.max
    X[1, 0], X[1, 1], X[1, 33] = f.smallest_normal / 4, f.smallest_normal, f.smallest_normal / 2
    X[2, 5], X[3, 6], X[3, 70] = float("inf"), float("-inf"), float("nan")
    X[4, 1], X[5, 0], X[6, 0] = -0.0, 1.0, -1.0
    X[7], X[8] = 3.0, -3.0
    X[69, 159] = float("nan")
    X[9:40] = oi.wide(torch.Generator().manual_seed(1), 31, 160, dtype=dtype) * f.smallest_normal * 16
    for group in (32, 64, 128):
        for scale_dtype in (BF16, F16):
            Y = (X.mT.contiguous() if trans else X).to(dev)
            _same(tb.int4_quantize(Y, group, zeros, trans, scale_dtype), X, group, zeros, scale_dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("zeros", [False, True])
def test_quotients_near_halfway(dev, zeros, dtype):
    # a group per leading value with each of a type's significands; the rest nearest to (n + 1/2) scales, and one step each way
    bits = {F32: 10, BF16: 7, F16: 10}[dtype]
    for scale_dtype in (BF16, F16):
        for exponent in (-14, -3, 0, 11) if F16 in (dtype, scale_dtype) else (-100, -3, 0, 100):
            top = ((1 + torch.arange(2**bits) * 2.0**-bits) * 2.0**exponent).to(dtype)
            low = torch.where(torch.arange(2**bits) % 3 == 0, top.float() * 0, -top.float() / 4).to(dtype)
            s = (((top.float() - low.float()) / 15 if zeros else top.float() / 7).to(scale_dtype)).double()
            half = torch.arange(-8, 16) + 0.5
            mid = (s[:, None] * half).to(dtype)
            mid = torch.maximum(torch.minimum(mid, top[:, None]), low[:, None] if zeros else -top[:, None])
            x = torch.stack([mid, torch.nextafter(mid, low[:, None]), torch.nextafter(mid, top[:, None])], -1).flatten(1)
            x = torch.where(x.float().abs() <= top.float()[:, None], x, top[:, None])
            x = torch.where(x < low[:, None], low[:, None], x) if zeros else x
            X = torch.cat([top[:, None], low[:, None], x, x[:, :54]], 1)
            assert X.shape[1] == 128
            _same(tb.int4_quantize(X.to(dev), 128, zeros, scale_dtype=scale_dtype), X, 128, zeros, scale_dtype)
            _same(tb.int4_quantize(X.to(dev), 32, zeros, scale_dtype=scale_dtype), X, 32, zeros, scale_dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_dequantize_and_layout(dev, dtype):
    g = torch.Generator().manual_seed(0)
    for group in (32, 64, 128):
        for shape in ((1, 1), (5, 33), (16, 128), (33, 257), (3, 18, 200)):
            for zeros in (False, True):
                Q, W = oi.random_matrix(g, *shape, group=group, zeros=zeros, scale_dtype=(BF16, F16)[group == 64], z_max=255)
                D = Q.to(dev).dequantize(dtype)
                assert D.dtype == dtype and torch.equal(D.cpu(), W.float().to(dtype))
                parts = Q.to(dev).parts()
                assert all(a is None or torch.equal(a, b.cpu()) for a, b in zip(Q.parts(), parts))


SIZES = [(1, 1), (1, 40), (5, 33), (16, 16), (33, 70), (64, 128), (100, 61), (136, 264), (257, 520)]


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("K", [1, 32, 100, 128, 512, 520, 1030, 2080])
def test_int4_gemm(dev, K, group):
    for i, (M, N) in enumerate(SIZES):
        g = torch.Generator().manual_seed(i)
        for zeros in (False, True):
            Q, W = oi.random_matrix(g, N, K, group=group, zeros=zeros, scale_dtype=(BF16, F16)[i % 2])
            Q = Q.to(dev)
            A = torch.randn(M, K, generator=g)
            for dtype in DTYPES:
                a = A.to(dtype)
                ref, den = oi.product(1.0, a, W)
                for out in {dtype, F32}:
                    D = tb.int4_gemm(1.0, a.to(dev), Q, dtype=out)
                    assert D.dtype == out and og.excess(D, ref, den, K) <= 1, (M, N, zeros, dtype, out)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", list(GROUPS))
def test_grouped(dev, shape, dtype):
    rows, sizes, lead = GROUPS[shape]
    off = _split(rows, sizes, lead)
    for i, (K, N) in enumerate([(40, 33), (512, 128), (1032, 72), (200, 264), (256, 520)]):
        g = torch.Generator().manual_seed(i)
        A = torch.randn(rows, K, generator=g).to(dtype)
        E, W = oi.random_matrix(g, len(sizes), N, K, group=(32, 64, 128)[i % 3], zeros=bool(i % 2), scale_dtype=BF16)
        D = tb.int4_grouped_gemm(1.0, A.to(dev), E.to(dev), off.to(dev))
        ref, den = oi.product(1.0, A, W, off)
        assert D.dtype == dtype and og.excess(D, ref, den, K) <= 1, (K, N)


@pytest.mark.parametrize("act", oa.ACTS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_gated(dev, dtype, act):
    for i, (shape, K, N) in enumerate([("one", 40, 8), ("token", 130, 24), ("gaps", 264, 17), ("small", 520, 72), ("uneven", 128, 136),
                                       ("single", 200, 61)]):  # fmt: skip
        rows, sizes, lead = GROUPS[shape]
        off = _split(rows, sizes, lead)
        g = torch.Generator().manual_seed(i)
        A = torch.randn(rows, K, generator=g).to(dtype)
        E, W = oi.random_matrix(g, len(sizes), 2 * N, K, group=(32, 64, 128)[i % 3], zeros=bool(i % 2), scale_dtype=F16)
        for out in {dtype, F32, F16}:
            H = tb.grouped_gated_gemm(A.to(dev), E.to(dev), off.to(dev), act, dtype=out)
            P, den = oa.products(A, W, off, True)
            assert H.dtype == out and oa.ratio(H, *oa.forward(act, P, den, K, out)) <= 1, (shape, K, N, out)
        H = tb.gated_gemm(A.to(dev), E[0].to(dev), act, transB=True)
        P, den = oa.products(A, W[:1], torch.tensor([0, rows]), True)
        assert oa.ratio(H, *oa.forward(act, P, den, K, dtype)) <= 1, (shape, K, N)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group", [32, 64, 128])
def test_many_rows(dev, group, dtype):
    # tiles of 128 rows that end inside, columns that end inside a tile and a block, chunks of 128 values cut short
    for i, (G, R, K, N) in enumerate([(1, 65, 128, 16), (1, 300, 1160, 400), (1, 513, 72, 1000), (2, 390, 2056, 264), (3, 1200, 515, 333), (1, 129, 4100, 48)]):
        g = torch.Generator(device=dev).manual_seed(i)
        off = torch.tensor([0, R]) if G == 1 else og.uneven(G, R, i)
        A = torch.randn(R, K, generator=g, device=dev).to(dtype)
        E, W = oi.random_matrix(g, G, N, K, group=group, zeros=bool(i % 2), scale_dtype=(BF16, F16)[i % 2], device=dev)
        ref, den = torch.zeros(2, R, N, dtype=torch.float64, device=dev)
        for j, a, b in og.rows_of(off, R):
            V = W[j].T.contiguous()
            ref[a:b], den[a:b] = A[a:b].double() @ V, A[a:b].double().abs() @ V.abs()
        for out in {dtype, F32}:
            D = tb.int4_grouped_gemm(1.0, A, E, off.to(dev), dtype=out)
            assert og.excess(D.cpu(), ref.cpu(), den.cpu(), K) <= 1, (G, R, K, N, out)
        # the same matrix as gates and ups, where their rows start on a block of sixteen and where they do not
        if N % 2 == 0:
            P, d = oa.products(A, W, off, True)
            act = oa.ACTS[i % 3]
            for out in {dtype, F32}:
                H = tb.grouped_gated_gemm(A, E, off.to(dev), act, dtype=out)
                assert oa.ratio(H, *oa.forward(act, P, d, K, out)) <= 1, (G, R, K, N, out)


def _plan(dtype, gated, groups, rows, N, K, group):
    """(rows of a tile, parts of K, blocks of rows, blocks of columns, waves along K)"""
    import ctypes

    from trnblas_amd.hip import _lib

    out = (ctypes.c_int32 * 5)()
    _lib.call("trnblas_hip_int4_plan", _lib.DTYPE_CODES[dtype], gated, groups, rows, N, K, group, out)
    return tuple(out)


# (dtype, gated, groups, rows, N, K) that each form of the kernels serves with each length of group
FORMS = {
    (0, 1, 1, 1, 1): [(F32, 0, 8, 8, 2158, 17)],
    (0, 1, 1, 1, 2): [(BF16, 0, 1, 1, 9316, 135), (F32, 0, 2, 2, 4179, 17)],
    (0, 1, 1, 1, 4): [(BF16, 0, 2, 2, 2077, 133), (F32, 0, 1, 1, 4138, 16)],
    (0, 1, 1, 1, 8): [(F16, 0, 1, 1, 16, 141), (F32, 0, 1, 1, 19, 17)],
    (0, 1, 1, 2, 1): [(F16, 0, 33, 44, 1942, 16), (F32, 0, 16, 87, 2319, 16), (F16, 1, 2, 2126, 67, 17), (F32, 1, 4, 2021, 66, 19)],
    (0, 1, 1, 2, 2): [(F16, 0, 8, 2193, 67, 135), (F32, 0, 33, 71, 1853, 20), (F16, 1, 64, 1605, 40, 20), (F32, 1, 2, 2197, 35, 18)],
    (0, 1, 1, 2, 4): [(F16, 0, 1, 2076, 33, 278), (F32, 0, 64, 1652, 34, 278), (F16, 1, 2, 9, 2179, 17), (F32, 1, 1, 2151, 17, 17)],
    (0, 1, 1, 2, 8): [(F16, 0, 1, 1, 4105, 540), (F32, 0, 1, 1, 4492, 525), (BF16, 1, 1, 1, 18, 16), (F32, 1, 1, 2, 18, 16)],
    (0, 1, 2, 2, 1): [(F16, 0, 64, 908, 1344, 16), (F32, 0, 16, 138, 3852, 21), (BF16, 1, 64, 1993, 132, 18), (F32, 1, 64, 2004, 132, 19)],
    (0, 1, 2, 2, 2): [(BF16, 0, 64, 974, 335, 701), (F32, 0, 64, 872, 293, 169), (BF16, 1, 16, 4254, 33, 17), (F32, 1, 64, 4487, 43, 17)],
    (0, 1, 2, 2, 4): [(BF16, 0, 64, 3763, 38, 257), (F32, 0, 64, 1595, 152, 133), (BF16, 1, 64, 3763, 18, 17), (F32, 1, 64, 3604, 25, 17)],
    (0, 1, 2, 2, 8): [(BF16, 0, 4, 4246, 18, 259), (F32, 0, 2, 4508, 17, 287), (F16, 1, 33, 3879, 16, 277), (F32, 1, 8, 4119, 16, 268)],
    (0, 1, 4, 2, 1): [(F16, 0, 64, 1259, 2032, 16), (BF16, 1, 64, 3859, 156, 16)],
    (0, 1, 4, 2, 2): [(BF16, 1, 8, 4809, 141, 19)],
    (0, 1, 4, 2, 4): [(F16, 0, 8, 203, 1935, 427), (F16, 1, 8, 215, 945, 323)],
    (0, 1, 4, 2, 8): [(BF16, 0, 64, 2424, 80, 548), (F16, 1, 64, 3742, 27, 540)],
    (64, 1, 0, 0, 0): [(F16, 0, 1, 4, 16, 17), (F32, 0, 1, 4285, 16, 17), (BF16, 1, 1, 1, 16, 16), (F32, 1, 1, 10, 16, 16)],
    (64, 2, 0, 0, 0): [(F16, 0, 64, 1938, 207, 1243), (F32, 0, 33, 805, 407, 564), (BF16, 1, 64, 1547, 112, 1223), (F32, 1, 64, 2863, 80, 416)],
    (64, 4, 0, 0, 0): [(BF16, 0, 16, 4157, 33, 1030), (F32, 0, 1, 4100, 65, 268), (F16, 1, 1, 4167, 32, 1577), (F32, 1, 1, 18, 4448, 561)],
    (64, 8, 0, 0, 0): [(F16, 0, 8, 2347, 34, 3389), (F32, 0, 4, 2270, 33, 1037), (BF16, 1, 1, 16, 16, 10816), (F32, 1, 1, 18, 2320, 1064)],
    (128, 1, 0, 0, 0): [(F16, 0, 64, 2971, 786, 17), (F32, 0, 64, 2617, 1015, 17), (F16, 1, 64, 3743, 336, 17), (F32, 1, 4, 145, 7984, 16)],
}


@pytest.mark.parametrize("form", list(FORMS))
def test_each_form(dev, form):
    for i, (dtype, gated, G, R, N, K) in enumerate(FORMS[form]):
        g = torch.Generator(device=dev).manual_seed(i)
        off = og.uneven(G, R, i) if R > 4 * G else torch.arange(G + 1) * (R // G)
        A = torch.randn(R, K, generator=g, device=dev).to(dtype)
        for group, zeros in ((128, False), (32, True), (64, False)):
            assert _plan(dtype, gated, G, R, N, K, group) == form, (dtype, gated, G, R, N, K, group)
            E, W = oi.random_matrix(g, G, 2 * N if gated else N, K, group=group, zeros=zeros, scale_dtype=BF16 if zeros else F16, device=dev)
            if gated:
                P, d = oa.products(A, W, off, True)
                H = tb.grouped_gated_gemm(A, E, off.to(dev), "gelu")
                assert oa.ratio(H, *oa.forward("gelu", P, d, K, dtype)) <= 1, (G, R, N, K, group)
            else:
                C = torch.randn(N, generator=g, device=dev).to(dtype)
                P, d = oa.products(A, W, off, True)
                D = tb.int4_grouped_gemm(2.0, A, E, off.to(dev), 0.5, C)
                ref, den = 2.0 * P + 0.5 * C.double(), 2.0 * d + 0.5 * C.double().abs()
                assert og.excess(D.cpu(), ref.cpu(), den.cpu(), K) <= 1, (G, R, N, K, group)


@pytest.mark.parametrize("out", DTYPES)
def test_alpha_beta_and_result_type(dev, out):
    rows, sizes, lead = GROUPS["gaps"]
    off = _split(rows, sizes, lead).to(torch.int64)
    g = torch.Generator().manual_seed(2)
    A = torch.randn(rows, 200, generator=g)
    E, W = oi.random_matrix(g, len(sizes), 72, 200, group=64, zeros=True, scale_dtype=BF16)
    E = E.to(dev)
    for C in (torch.randn(rows, 72, generator=g).to(out), torch.randn(72, generator=g).to(out),
              torch.randn(rows, 145, generator=g).to(out)[:, 1:73]):  # fmt: skip
        for dtype in DTYPES:
            a = A.to(dtype)
            D = tb.int4_grouped_gemm(-1.5, a.to(dev), E, off.to(dev), 0.25, C.to(dev), dtype=out)
            assert og.excess(D, *oi.product(-1.5, a, W, off, 0.25, C), 200) <= 1
            D = tb.int4_gemm(-1.5, a.to(dev), E[1], 0.25, C.to(dev), dtype=out)
            assert og.excess(D, *oi.product(-1.5, a, W[1], None, 0.25, C), 200) <= 1


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(dev, dtype):
    # rows inside larger buffers, at any column and leading dimension, with NaN around them; one value of a pair; columns
    g = torch.Generator().manual_seed(3)
    for M, K, N in ((1, 136, 40), (40, 136, 40), (40, 61, 33), (7, 64, 24)):
        Q, W = oi.random_matrix(g, N, K, group=32, zeros=True, scale_dtype=BF16)
        Q = Q.to(dev)
        A = torch.randn(M, K, generator=g).to(dtype)
        ref, den = oi.product(1.0, A, W)
        for left in (0, 1, 8):
            X = torch.full((M, K + 24), float("nan"), dtype=dtype, device=dev)
            X[:, left : left + K] = A
            assert og.excess(tb.int4_gemm(1.0, X[:, left : left + K], Q), ref, den, K) <= 1, (M, K, left)
        assert og.excess(tb.int4_gemm(1.0, torch.stack([A, A * 0 + 9], -1).to(dev)[..., 0], Q), ref, den, K) <= 1
        assert og.excess(tb.int4_gemm(1.0, A.mT.contiguous().to(dev).mT, Q), ref, den, K) <= 1
        assert og.excess(tb.int4_gemm(1.0, A[:1].to(dev).expand(M, K), Q), *oi.product(1.0, A[:1].expand(M, K), W), K) <= 1


def test_negated_views(dev):
    g = torch.Generator().manual_seed(4)
    for M, K in ((1, 40), (17, 33), (130, 520)):
        x, c = torch.randn(M, K, 2, generator=g), torch.randn(M, 24, 2, generator=g)
        conj = lambda t: torch.view_as_complex(t.to(dev)).conj().imag
        A, C = conj(x), conj(c)
        assert A.is_neg() and C.is_neg()
        _same(tb.int4_quantize(A, 64), -x[..., 1], 64, False, BF16)
        _same(tb.int4_quantize(A.mT, 64, trans=True), -x[..., 1], 64, False, BF16)
        Q, W = oi.random_matrix(g, 24, K, group=64, zeros=False, scale_dtype=BF16)
        assert og.excess(tb.int4_gemm(1.0, A, Q.to(dev)), *oi.product(1.0, -x[..., 1], W), K) <= 1
        assert og.excess(tb.int4_gemm(1.0, A, Q.to(dev), 0.5, C), *oi.product(1.0, -x[..., 1], W, None, 0.5, -c[..., 1]), K) <= 1


def test_fp32_rows_are_not_rounded(dev):
    # values over the whole range of fp32, each with all its bits: sums of one term, and of terms that cancel
    g = torch.Generator().manual_seed(5)
    A = torch.zeros(200, 128)
    A[torch.arange(200), torch.arange(200) % 128] = torch.randn(200, generator=g) * torch.exp2(torch.randint(-96, 96, (200,), generator=g).float())
    Q, W = oi.random_matrix(g, 16, 128, group=128, zeros=False, scale_dtype=BF16)
    D = tb.int4_gemm(1.0, A.to(dev), Q.to(dev)).double().cpu()
    ref = A.double() @ W.T
    # three pieces: the products with q - z are exact, three additions, and the scale
    assert ((D - ref).abs() <= 5 * 2.0**-24 * ref.abs()).all()
    big = torch.tensor([[3e38, float("inf"), 1.0], [1.0, float("nan"), 2.0], [-float("inf"), 0.0, 1.0], [1e-30, 2.0, 1.0]])
    codes = torch.full((1, 2), 0x99, dtype=torch.uint8)  # weights of one
    one = tb.Int4Matrix.from_parts(codes, torch.ones(1, 1, dtype=BF16), 3, 32).to(dev)
    D = tb.int4_gemm(1.0, big.to(dev), one).cpu()[:, 0]
    assert D[0] == float("inf") and D[1].isnan() and D[2] == -float("inf") and D[3] == 3.0


@pytest.mark.parametrize("dtype", DTYPES)
def test_nan_groups_reach_their_results_only(dev, dtype):
    g = torch.Generator().manual_seed(6)
    A, X = torch.randn(40, 300, generator=g).to(dtype), torch.randn(3, 50, 300, generator=g)
    off = _split(40, [10, 12, 8], 5)
    call = lambda a, x: tb.int4_grouped_gemm(1.0, a.to(dev), tb.int4_quantize(x.to(dev), 64), off.to(dev)).cpu()
    want = call(A, X)
    Ab, Xb = A.clone(), X.clone()
    Ab[2, 7], Ab[9, 299], Xb[1, 4, 0], Xb[1, 49, 200] = (float(x) for x in ("nan", "nan", "nan", "-inf"))
    got = call(Ab, Xb)
    bad = torch.zeros(40, 50, dtype=torch.bool)
    bad[9], bad[15:27, 4], bad[15:27, 49] = True, True, True
    assert torch.equal(got.isnan(), bad) and torch.equal(got[~bad], want[~bad])


def test_sizes_of_zero(dev):
    for shape in ((0, 40), (5, 0)):
        Q = tb.int4_quantize(torch.zeros(shape, device=dev))
        assert Q.dequantize().shape == shape
        D = tb.int4_gemm(1.0, torch.ones(3, shape[1], device=dev), Q)
        assert D.shape == (3, shape[0]) and not D.any()
    C = torch.ones(3, 5, device=dev)
    assert torch.equal(tb.int4_gemm(1.0, torch.ones(3, 0, device=dev), Q, 2.0, C), 2.0 * C)
    E = tb.int4_quantize(torch.ones(2, 4, 8, device=dev))
    off = torch.tensor([0, 0, 0], device=dev)
    assert tb.int4_grouped_gemm(1.0, torch.zeros(0, 8, device=dev), E, off).shape == (0, 4)
    assert not tb.int4_grouped_gemm(1.0, torch.ones(3, 8, device=dev), E, off).any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_captured_graph_serves_any_routing(dev, dtype):
    g = torch.Generator().manual_seed(9)
    A = torch.randn(96, 512, generator=g).to(dev, dtype)
    E, _ = oi.random_matrix(g, 6, 128, 512, group=64, zeros=True, scale_dtype=F16)
    E = E.to(dev)
    one = E[0]
    off = _split(96, [16] * 6).to(dev)
    calls = lambda: (tb.int4_grouped_gemm(1.0, A, E, off), tb.int4_gemm(1.0, A, one), tb.int4_gemm(1.0, A[:2], one),
                     tb.grouped_gated_gemm(A, E, off), tb.gated_gemm(A[:1], one))  # fmt: skip
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        calls()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = calls()
    for i, sizes in enumerate(([16] * 6, [0, 0, 96, 0, 0, 0], [1, 2, 3, 4, 5, 6], [40, 0, 40, 0, 1, 0])):
        off.copy_(_split(96, sizes))
        A.mul_(1.0 + i)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, calls()))


def test_two_streams_at_once(dev):
    # fp32 rows go through a workspace: each call has its own
    g = torch.Generator().manual_seed(10)
    A = torch.randn(300, 520, generator=g).to(dev)
    Q, _ = oi.random_matrix(g, 264, 520, group=32, zeros=True, scale_dtype=BF16)
    Q = Q.to(dev)
    B = A * 3 + 1
    want = tb.int4_gemm(1.0, A, Q), tb.int4_gemm(1.0, B, Q)
    streams, out = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for i, s in enumerate(streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            out[i] += [tb.int4_gemm(1.0, (A, B)[i], Q) for _ in range(6)]
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(x, want[i]) for i in range(2) for x in out[i])


def test_a_block_trained_and_served(dev):
    # gated projections in a training step, their weights quantised, and the same block from 4 bits: both against 64 bits
    g = torch.Generator().manual_seed(11)
    x, W, V = torch.randn(20, 256, generator=g), torch.randn(2 * 192, 256, generator=g) / 16, torch.randn(256, 192, generator=g) / 14
    w = W.to(dev).requires_grad_()
    (dW,) = torch.autograd.grad(tb.gated_gemm(x.to(dev), w, transB=True).square().sum(), w)
    W = (w - 1e-3 * dW).detach()
    Qw, Qv = tb.int4_quantize(W, 64, zeros=True), tb.int4_quantize(V.to(dev), 32)
    got = tb.int4_gemm(1.0, tb.gated_gemm(x.to(dev), Qw), Qv).double().cpu()
    G, U = (x.double() @ oi.quantize(W.cpu(), 64, True, BF16)[0].T).chunk(2, -1)
    H = torch.nn.functional.silu(G) * U
    Vq = oi.quantize(V, 32, False, BF16)[0]
    ref, den = H @ Vq.T, H.abs() @ Vq.abs().T
    assert ((got - ref).abs() <= 1e-5 * den).all()
    full = torch.nn.functional.silu((x.double() @ W.cpu().double().T)[:, :192]) * (x.double() @ W.cpu().double().T)[:, 192:] @ V.double().T
    assert float((got - full).norm() / full.norm()) < 0.25  # 4 bits: an eighth of a weight's size each, three products deep
