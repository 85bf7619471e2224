"""Microscaled 4-bit floats on the GPU: codes and scales equal to the definition's, products within what fp32 sums allow."""

import pytest
import torch

import trnblas_amd as tb
from oracle import grouped as og
from oracle import mx as om
from oracle.grouped import GROUPS, plan, rows_plan, uneven
from oracle.grouped import split as _split
from oracle.mx import wide as _wide

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
DTYPES = [F32, BF16, F16]


def _same(Q, X):
    want, code, byte = om.quantize(X)
    V = Q.dequantize().double().cpu()
    assert torch.equal(V.isnan(), want.isnan()) and torch.equal(V.nan_to_num(-1.0), want.nan_to_num(-1.0))
    assert torch.equal(Q.block_scales().long().cpu(), byte)
    H = tb.mx_quantize(X)  # on the host
    assert torch.equal(H.scales, Q.scales.cpu())
    assert torch.equal(H.codes & 0x77, Q.codes.cpu() & 0x77)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (1, 4096), (3, 32), (17, 33), (16, 512), (64, 512), (130, 1032), (2, 19, 70),
                                   (257, 130), (3, 65, 520)])  # fmt: skip
def test_quantize(dev, shape, dtype):
    X = _wide(torch.Generator().manual_seed(0), *shape, dtype=dtype)
    _same(tb.mx_quantize(X.to(dev)), X)
    _same(tb.mx_quantize(X.mT.contiguous().to(dev), trans=True), X)
    P = torch.full((*X.shape[:-1], X.shape[-1] + 5), float("nan"), dtype=dtype, device=dev)
    P[..., 3:-2] = X
    _same(tb.mx_quantize(P[..., 3:-2]), X)
    if X.dim() == 2:
        _same(tb.mx_quantize(torch.stack([X, X * 0 + 9], -1).to(dev)[..., 0]), X)
        P = torch.full((X.shape[1], X.shape[0] + 7), float("nan"), dtype=dtype, device=dev)
        P[:, 1:-6] = X.mT
        _same(tb.mx_quantize(P[:, 1:-6], trans=True), X)


@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_values_at_the_ends(dev, dtype, trans):
    f = torch.finfo(dtype)
    X = torch.zeros(70, 96, dtype=dtype)
    X[0, 3], X[0, 40] = f.max, -f.max
    X[1, 0], X[1, 1], X[1, 33] = f.smallest_normal / 4, f.smallest_normal, f.smallest_normal / 2
    X[2, 5] = float("inf")
    X[3, 5], X[3, 6] = float("nan"), float("-inf")
    X[4, 1] = -0.0
    X[5, :8] = torch.tensor([7.99, 7.0, 5.0, 5.01, 3.5, 2.5, 0.25, 0.2501])
    X[69, 95] = float("nan")
    X[6:40] = _wide(torch.Generator().manual_seed(1), 34, 96, dtype=dtype) * f.smallest_normal * 16
    Xd = X.mT.contiguous().to(dev) if trans else X.to(dev)
    _same(tb.mx_quantize(Xd, trans=trans), X)


def test_every_code_and_scale(dev):
    # all 16 codes under all 256 scale bytes, into each type
    codes = torch.arange(16, dtype=torch.uint8).repeat(2)
    packed = (codes[::2] | codes[1::2] << 4).expand(256, 16).contiguous()
    Q = tb.MXMatrix.from_parts(packed, torch.arange(256, dtype=torch.uint8)[:, None].contiguous(), 32)
    for dtype in DTYPES:
        host, gpu = Q.dequantize(dtype), Q.to(dev).dequantize(dtype).cpu()
        assert torch.equal(host.isnan(), gpu.isnan()) and torch.equal(host.nan_to_num(7.0), gpu.nan_to_num(7.0))


SIZES = [(1, 1), (1, 40), (5, 33), (16, 16), (33, 70), (64, 128), (100, 61), (136, 264), (257, 520)]


@pytest.mark.parametrize("K", [1, 32, 100, 128, 512, 520, 1030, 2080])
def test_mx_gemm(dev, K):
    for i, (M, N) in enumerate(SIZES):
        g = torch.Generator().manual_seed(i)
        A, W = _wide(g, M, K), _wide(g, N, K)
        a, w = om.quantize(A)[0], om.quantize(W)[0]
        Q = tb.mx_quantize(W.to(dev))
        ref, den = om.product(1.0, a, w)
        for x in (A.to(dev), tb.mx_quantize(A.to(dev))):
            assert og.excess(tb.mx_gemm(1.0, x, Q, dtype=F32), ref, den, K) <= 1, (M, N)
        assert og.excess(tb.mx_gemm(1.0, tb.mx_quantize(A.to(dev)), Q), ref, den, K) <= 1, (M, N)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", list(GROUPS))
def test_mx_grouped_gemm(dev, shape, dtype):
    rows, sizes, lead = GROUPS[shape]
    off = _split(rows, sizes, lead)
    for i, (K, N) in enumerate([(40, 33), (512, 128), (1032, 72), (200, 264), (256, 520)]):
        g = torch.Generator().manual_seed(i)
        A = torch.randn(rows, K, generator=g).to(dtype)
        W = torch.randn(len(sizes), N, K, generator=g).to(dtype)
        D = tb.mx_grouped_gemm(1.0, A.to(dev), tb.mx_quantize(W.to(dev)), off.to(dev))
        ref, den = om.product(1.0, om.quantize(A)[0], om.quantize(W)[0], off)
        assert D.dtype == dtype and og.excess(D, ref, den, K) <= 1, (K, N)


@pytest.mark.parametrize("out", DTYPES)
def test_alpha_beta_and_result_type(dev, out):
    rows, sizes, lead = GROUPS["gaps"]
    off = _split(rows, sizes, lead).to(torch.int64)
    g = torch.Generator().manual_seed(2)
    A, W = torch.randn(rows, 200, generator=g), torch.randn(len(sizes), 72, 200, generator=g)
    a, w = om.quantize(A)[0], om.quantize(W)[0]
    E = tb.mx_quantize(W.to(dev))
    for C in (torch.randn(rows, 72, generator=g).to(out), torch.randn(72, generator=g).to(out),
              torch.randn(rows, 145, generator=g).to(out)[:, 1:73]):  # fmt: skip
        D = tb.mx_grouped_gemm(-1.5, A.to(dev), E, off.to(dev), 0.25, C.to(dev), dtype=out)
        assert og.excess(D, *om.product(-1.5, a, w, off, 0.25, C), 200) <= 1
        D = tb.mx_gemm(-1.5, A.to(dev), E[1], 0.25, C.to(dev), dtype=out)
        assert og.excess(D, *om.product(-1.5, a, w[1], None, 0.25, C), 200) <= 1


def test_nan_blocks_reach_their_results_only(dev):
    g = torch.Generator().manual_seed(3)
    A, W = torch.randn(40, 300, generator=g), torch.randn(3, 50, 300, generator=g)
    off = _split(40, [10, 12, 8], 5)
    want = tb.mx_grouped_gemm(1.0, A.to(dev), tb.mx_quantize(W.to(dev)), off.to(dev))
    Ab, Wb = A.clone(), W.clone()
    Ab[2, 7], Ab[9, 299], Wb[1, 4, 0], Wb[1, 49, 200] = (float(x) for x in ("nan", "inf", "nan", "-inf"))
    got = tb.mx_grouped_gemm(1.0, Ab.to(dev), tb.mx_quantize(Wb.to(dev)), off.to(dev))
    bad = torch.zeros(40, 50, dtype=torch.bool)
    bad[9], bad[15:27, 4], bad[15:27, 49] = True, True, True
    assert torch.equal(got.cpu().isnan(), bad) and torch.equal(got.cpu()[~bad], want.cpu()[~bad])


def test_captured_graph_serves_any_routing(dev):
    g = torch.Generator().manual_seed(9)
    A, E = torch.randn(96, 512, generator=g).to(dev), tb.mx_quantize(torch.randn(6, 128, 512, generator=g).to(dev))
    off = _split(96, [16] * 6).to(dev)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        tb.mx_grouped_gemm(1.0, A, E, off)
        tb.mx_gemm(1.0, A, E[0])
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        D, P = tb.mx_grouped_gemm(1.0, A, E, off), tb.mx_gemm(1.0, A, E[0])
    for i, sizes in enumerate(([16] * 6, [0, 0, 96, 0, 0, 0], [1, 2, 3, 4, 5, 6], [40, 0, 40, 0, 1, 0])):
        off.copy_(_split(96, sizes))
        A.mul_(1.0 + i)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(D, tb.mx_grouped_gemm(1.0, A, E, off)) and torch.equal(P, tb.mx_gemm(1.0, A, E[0]))


def test_scales_far_apart(dev):
    # products whose scales go to both ends: below the fp32 range they vanish, above it they are infinite
    X = torch.full((4, 128), 1.5)
    S = torch.full((4, 4), 127, dtype=torch.uint8)
    S[1], S[2], S[3] = 0, 252, 60
    Q = tb.mx_quantize(X)
    M = tb.MXMatrix.from_parts(Q.codes, S, 128).to(dev)
    D = tb.mx_gemm(1.0, M, M, dtype=F32).cpu().double()
    v = M.dequantize().cpu().double()[:, 0]
    want = 128 * v[:, None] * v[None, :]
    for i in range(4):
        for j in range(4):
            if want[i, j] < 2.0**-126:
                assert 0 <= D[i, j] <= 2.0**-126
            else:
                assert D[i, j] == (want[i, j] if want[i, j] < 2.0**128 else float("inf")), (i, j)


MX_REACH = {
    "ring_kernel 256 x 256": [(3, 5200, 520, 2312), (1, 7000, 1160, 2568)],
    "ring_kernel 128 x 128": [(5, 20000, 2056, 1032)],
    "ring_kernel 64 x 128": [(3, 2600, 1032, 1288), (8, 1500, 264, 1032), (8, 900, 520, 264), (3, 700, 1030, 520)],
    "rows_kernel": [(8, 8, 4100, 520), (2, 20, 1030, 136)],
}


@pytest.mark.parametrize("kernel", list(MX_REACH))
def test_each_kernel(dev, kernel):
    for i, (G, R, K, N) in enumerate(MX_REACH[kernel]):
        assert plan(2, BF16, 1, G, R, 0, N, K) == kernel
        g = torch.Generator(device=dev).manual_seed(i)
        off = uneven(G, R, i)
        A = torch.randn(R, K, generator=g, device=dev) * torch.exp2(torch.arange(R, device=dev) % 7)[:, None]
        E = tb.mx_quantize(torch.randn(G, N, K, generator=g, device=dev))
        a, w = tb.mx_quantize(A).dequantize().double(), E.dequantize().double()
        ref, den = torch.zeros(2, R, N, dtype=torch.float64, device=dev)
        for j, p, q in og.rows_of(off, R):
            W = w[j].T.contiguous()
            ref[p:q], den[p:q] = a[p:q] @ W, a[p:q].abs() @ W.abs()
        for out in (F32, F16 if kernel != "rows_kernel" else BF16):
            for x in (A, tb.mx_quantize(A)):
                D = tb.mx_grouped_gemm(1.0, x, E, off.to(dev), dtype=out)
                assert og.excess(D.cpu(), ref.cpu(), den.cpu(), K) <= 1, (G, R, K, N, out)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K", [(1, 8192), (1, 8191), (3, 10900), (4, 8192), (16, 2048), (16, 2050), (15, 33)])
def test_few_rows_quantised_in_place(dev, dtype, M, K):
    g = torch.Generator().manual_seed(M)
    A, W = _wide(g, M, K + 2, dtype=dtype)[:, 1:-1], torch.randn(200, K, generator=g)
    A[0, K // 2] = 0.0
    ref, den = om.product(1.0, om.quantize(A)[0], om.quantize(W)[0])
    Q = tb.mx_quantize(W.to(dev))
    for x in (A.to(dev), A.contiguous().to(dev)):
        assert og.excess(tb.mx_gemm(1.0, x, Q, dtype=F32), ref, den, K) <= 1
    A = A.clone()
    A[M - 1, K - 1] = float("inf")
    D = tb.mx_gemm(1.0, A.to(dev), Q, dtype=F32)
    assert D[M - 1].isnan().all() and D[: M - 1].isfinite().all()


def test_tangents_are_refused(dev):
    from torch.autograd import forward_ad as fwd

    A, W = torch.ones(4, 64, device=dev), tb.mx_quantize(torch.ones(3, 64, device=dev))
    with fwd.dual_level():
        with pytest.raises(NotImplementedError, match="no gradient"):
            tb.mx_gemm(1.0, fwd.make_dual(A, A), W)
        assert torch.equal(tb.mx_gemm(1.0, A, W), torch.full((4, 3), 64.0, device=dev))


@pytest.mark.parametrize("M,K", [(1, 40), (17, 33), (130, 520)])
def test_negated_views(dev, M, K):
    # the imaginary part of a conjugate is a view whose values stand in memory with the other sign
    g = torch.Generator().manual_seed(M)
    x, c = torch.randn(M, K, 2, generator=g), torch.randn(M, 24, 2, generator=g)
    conj = lambda t: torch.view_as_complex(t.to(dev)).conj().imag
    A, C = conj(x), conj(c)
    assert A.is_neg() and C.is_neg()
    _same(tb.mx_quantize(A), -x[..., 1])
    _same(tb.mx_quantize(A.mT, trans=True), -x[..., 1])
    _same(tb.mx_quantize(A[None]), -x[None, ..., 1])
    W = torch.randn(24, K, generator=g)
    Q = tb.mx_quantize(W.to(dev))
    a, w = om.quantize(-x[..., 1])[0], om.quantize(W)[0]
    assert og.excess(tb.mx_gemm(1.0, A, Q), *om.product(1.0, a, w), K) <= 1
    assert og.excess(tb.mx_gemm(1.0, A, Q, 0.5, C), *om.product(1.0, a, w, None, 0.5, -c[..., 1]), K) <= 1


# (groups, rows, N, K) by what rows_kernel does with them: (blocks of 16 rows, waves along K, A of values quantised inside).
# Columns end inside a tile, and where waves split the columns some of them lie past N as a whole.
ROWS = {
    (2, 8, 0): [(1, 20, 72, 2056), (2, 30, 200, 1030)],
    (2, 4, 0): [(13, 801, 520, 64), (5, 200, 2056, 64)],
    (2, 2, 0): [(57, 1140, 520, 64)],
    (2, 1, 0): [(64, 3968, 1032, 64)],
    (1, 8, 0): [(16, 60, 200, 2050), (64, 320, 72, 2056)],
    (1, 8, 1): [(16, 60, 200, 2048), (2, 9, 520, 1030)],
    (1, 4, 1): [(41, 287, 520, 520), (5, 5, 4104, 520)],
    (1, 2, 1): [(9, 18, 4104, 64), (64, 448, 520, 64)],
    (1, 1, 1): [(57, 399, 1032, 64), (23, 23, 4104, 520), (57, 399, 4104, 1030)],
}


@pytest.mark.parametrize("how", list(ROWS))
@pytest.mark.parametrize("dtype", DTYPES)
def test_each_form_of_the_few_rows_kernel(dev, dtype, how):
    for G, R, N, K in ROWS[how]:
        assert rows_plan(2, dtype, 1, G, R, N, K) == how
        g = torch.Generator(device=dev).manual_seed(R)
        # one group fills a block of 16 rows where there are several groups, the others share what is left unevenly
        sizes = torch.bincount(torch.arange(R - min(R, 16 * (G > 1))) % max(G - 1, 1) + (G > 1), minlength=G)
        sizes[0] = R if G == 1 else min(R, 16)
        off = _split(R, sizes.tolist())
        A = torch.randn(R, K + 6, generator=g, device=dev) * torch.exp2(torch.arange(R, device=dev) % 7)[:, None]
        A = A.to(dtype)[:, 3:-3]
        E = tb.mx_quantize(torch.randn(G, N, K, generator=g, device=dev))
        q = tb.mx_quantize(A)
        ref, den = torch.zeros(2, R, N, dtype=torch.float64, device=dev)
        for j, a, b in og.rows_of(off, R):
            x, W = q.dequantize().double()[a:b], E[j].dequantize().double().T.contiguous()
            ref[a:b], den[a:b] = x @ W, x.abs() @ W.abs()
        ref, den = ref.cpu(), den.cpu()
        for x in (A, A.contiguous(), q):
            D = tb.mx_grouped_gemm(1.0, x, E, off.to(dev), dtype=F32)
            assert og.excess(D.cpu(), ref, den, K) <= 1, (G, R, N, K)
        if G == 1:
            assert og.excess(tb.mx_gemm(1.0, A, E[0], dtype=F32).cpu(), ref, den, K) <= 1
