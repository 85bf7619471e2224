"""grouped_gemm / grouped_rank_k on the GPU against 64-bit products, at sizes, layouts and group shapes where they can go
wrong. The bound is `oracle.grouped.excess`'s."""

import pytest
import torch

import trnblas_amd as tb
from oracle import grouped as og
from oracle.grouped import GROUPS
from oracle.grouped import plan as _plan
from oracle.grouped import rows_plan
from oracle.grouped import split as _split
from oracle.grouped import uneven as _uneven

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
DTYPES = [F32, BF16, F16]


def _randn(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g).to(dtype)


# (K, N): below and across the tiles of 16, 32, 64, 128 and 256, multiples of 16 bytes and not
SIZES = [(1, 1), (7, 5), (33, 70), (64, 128), (100, 61), (136, 264), (264, 136), (512, 520), (515, 257), (1032, 384)]


@pytest.mark.parametrize("shape", list(GROUPS))
@pytest.mark.parametrize("dtype", DTYPES)
def test_grouped_gemm(dev, shape, dtype):
    rows, sizes, lead = GROUPS[shape]
    off = _split(rows, sizes, lead)
    for i, (K, N) in enumerate(SIZES):
        for transB in (False, True):
            g = torch.Generator().manual_seed(100 * i + transB)
            A = _randn(g, rows, K, dtype=dtype)
            B = _randn(g, len(sizes), *((N, K) if transB else (K, N)), dtype=dtype)
            D = tb.grouped_gemm(1.0, A.to(dev), B.to(dev), off.to(dev), transB=transB)
            ref, den = og.grouped_gemm(1.0, A, B, off, transB=transB)
            assert D.dtype == dtype and og.excess(D, ref, den, K) <= 1, (K, N, transB)


@pytest.mark.parametrize("shape", ["one", "token", "gaps", "small", "uneven", "single"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_grouped_rank_k(dev, shape, dtype):
    rows, sizes, lead = GROUPS[shape]
    off = _split(rows, sizes, lead)
    for i, (M, N) in enumerate([(1, 1), (5, 7), (70, 33), (128, 64), (136, 264), (264, 512), (257, 515)]):
        g = torch.Generator().manual_seed(i)
        A, B = _randn(g, rows, M, dtype=dtype), _randn(g, rows, N, dtype=dtype)
        for out in {dtype, F32}:
            D = tb.grouped_rank_k(1.0, A.to(dev), B.to(dev), off.to(dev), dtype=out)
            ref, den = og.grouped_rank_k(1.0, A, B, off)
            assert D.dtype == out and og.excess(D, ref, den, rows) <= 1, (M, N, out)


@pytest.mark.parametrize("dtype", DTYPES)
def test_fp32_products_keep_the_fp32_gate(dev, dtype):
    # same-sign operands: the worst case of a running sum; fp32 is held to 1e-6 |A||B| as `gemm` is
    g = torch.Generator().manual_seed(5)
    A, B = torch.rand(300, 4100, generator=g).to(dtype), torch.rand(2, 4100, 260, generator=g).to(dtype)
    off = _split(300, [130, 170])
    D = tb.grouped_gemm(1.0, A.to(dev), B.to(dev), off.to(dev), dtype=F32)
    ref, den = og.grouped_gemm(1.0, A, B, off)
    assert float(((D.double().cpu() - ref).abs() / den).max()) <= (1e-6 if dtype == F32 else 4100 * 2.0**-23)
    A, B = torch.rand(4100, 136, generator=g).to(dtype), torch.rand(4100, 260, generator=g).to(dtype)
    off = _split(4100, [4000, 100])
    D = tb.grouped_rank_k(1.0, A.to(dev), B.to(dev), off.to(dev), dtype=F32)
    ref, den = og.grouped_rank_k(1.0, A, B, off)
    assert float(((D.double().cpu() - ref).abs() / den).max()) <= (1e-6 if dtype == F32 else 4000 * 2.0**-23)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K,N", [(64, 128), (100, 61), (264, 256)])
def test_alpha_beta_and_result_type(dev, dtype, K, N):
    rows, sizes, lead = GROUPS["gaps"]
    off = _split(rows, sizes, lead).to(torch.int64)
    g = torch.Generator().manual_seed(2)
    A, B = _randn(g, rows, K, dtype=dtype), _randn(g, len(sizes), K, N, dtype=dtype)
    for out in {dtype, F32}:
        for C in (_randn(g, rows, N, dtype=out), _randn(g, N, dtype=out), _randn(g, rows, 2 * N + 1, dtype=out)[:, 1 : N + 1]):
            D = tb.grouped_gemm(-1.5, A.to(dev), B.to(dev), off.to(dev), 0.25, C.to(dev), dtype=out)
            ref, den = og.grouped_gemm(-1.5, A, B, off, 0.25, C)
            assert og.excess(D, ref, den, K) <= 1
        W = _randn(g, rows, N, dtype=dtype)
        C = _randn(g, len(sizes), K, N, dtype=out)
        D = tb.grouped_rank_k(-1.5, A.to(dev), W.to(dev), off.to(dev), 1.0, C.to(dev), dtype=out)
        ref, den = og.grouped_rank_k(-1.5, A, W, off, 1.0, C)
        assert og.excess(D, ref, den, rows) <= 1


def test_nan_in_c_is_not_read_without_beta(dev):
    A, B, off = torch.ones(40, 64, device=dev), torch.ones(2, 64, 32, device=dev), _split(40, [10, 20]).to(dev)
    C = torch.full((40, 32), float("nan"), device=dev)
    D = tb.grouped_gemm(1.0, A, B, off, 0.0, C)
    assert torch.equal(D[:30], torch.full((30, 32), 64.0, device=dev)) and not D[30:].any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_values_of_other_groups_stay_out(dev, dtype):
    # infinities and NaN in rows of no group, in rows of other groups and in their matrices, and past the ends of padded
    # rows: none of them reaches a result
    for K, N in ((40, 72), (61, 33), (256, 256)):
        g = torch.Generator().manual_seed(3)
        off = _split(60, [9, 21, 0, 5], 10)
        Ap, Bp = _randn(g, 60, K + 8, dtype=dtype), _randn(g, 4, K, N + 8, dtype=dtype)
        W = _randn(g, 60, N, dtype=dtype)
        bad = Ap.clone(), Bp.clone(), W.clone()
        bad[0][:10], bad[0][19:40], bad[0][45:], bad[0][:, K:] = (float(x) for x in ("inf", "nan", "nan", "inf"))
        bad[1][1:3], bad[1][:, :, N:] = float("nan"), float("inf")
        bad[2][:10], bad[2][19:40], bad[2][45:] = float("nan"), float("inf"), float("nan")
        A, B, W = Ap.to(dev), Bp.to(dev), W.to(dev)
        Ab, Bb, Wb = (x.to(dev) for x in bad)
        want = tb.grouped_gemm(1.0, A[:, :K], B[:, :, :N], off.to(dev))
        got = tb.grouped_gemm(1.0, Ab[:, :K], Bb[:, :, :N], off.to(dev))
        for a, b in ((10, 19), (40, 45)):
            assert torch.equal(got[a:b], want[a:b]) and want[a:b].isfinite().all()
        assert not got[:10].any() and not got[45:].any()
        want = tb.grouped_rank_k(1.0, A[:, :K], W, off.to(dev))
        got = tb.grouped_rank_k(1.0, Ab[:, :K], Wb, off.to(dev))
        for i in (0, 2, 3):
            assert torch.equal(got[i], want[i]) and want[i].isfinite().all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K,N", [(64, 128), (100, 61), (520, 264)])
def test_layouts(dev, dtype, K, N):
    rows, sizes = 150, [17, 33, 1, 64, 35]
    off = _split(rows, sizes)
    g = torch.Generator().manual_seed(4)
    A, B = _randn(g, rows, K, dtype=dtype), _randn(g, 5, K, N, dtype=dtype)
    ref, den = og.grouped_gemm(1.0, A, B, off)
    Ad, Bd, od = A.to(dev), B.to(dev), off.to(dev)

    def inside(X, before, after):  # X inside a larger buffer: another leading dimension and another alignment
        P = torch.full((*X.shape[:-1], X.shape[-1] + before + after), float("nan"), dtype=dtype, device=dev)
        P[..., before : before + X.shape[-1]] = X
        return P[..., before : before + X.shape[-1]]

    views = {
        "wide": (inside(Ad, 0, 8), inside(Bd, 0, 16)),
        "shifted": (inside(Ad, 1, 2), inside(Bd, 3, 0)),
        "aligned_shift": (inside(Ad, 8, 8), inside(Bd, 16, 8)),
        "transposed_a": (Ad.mT.contiguous().mT, Bd),
        "transposed_b": (Ad, Bd.mT.contiguous().mT),
        "groups_apart": (Ad, torch.stack([Bd, Bd * 0 + float("nan")], 1)[:, 0]),
        "rows_apart": (torch.stack([Ad, Ad * 0 + float("nan")], 1)[:, 0], Bd),
    }
    for name, (a, b) in views.items():
        D = tb.grouped_gemm(1.0, a, b, od)
        assert og.excess(D, ref, den, K) <= 1, name
    one = B[2].to(dev).expand(5, K, N)
    D = tb.grouped_gemm(1.0, Ad, one, od)
    assert og.excess(D, *og.grouped_gemm(1.0, A, B[2].expand(5, K, N), off), K) <= 1
    W = _randn(g, rows, N, dtype=dtype)
    ref, den = og.grouped_rank_k(1.0, A, W, off)
    for a, w in ((inside(Ad, 1, 2), inside(W.to(dev), 0, 3)), (inside(Ad, 8, 8), inside(W.to(dev), 8, 0))):
        assert og.excess(tb.grouped_rank_k(1.0, a, w, od), ref, den, rows) <= 1


def test_offsets_outside_the_rows_are_clamped(dev):
    g = torch.Generator().manual_seed(6)
    A, B = _randn(g, 50, 32), _randn(g, 3, 32, 16)
    want = tb.grouped_gemm(1.0, A.to(dev), B.to(dev), torch.tensor([0, 20, 20, 50], device=dev))
    for dt, big in ((torch.int32, 2**31 - 1), (torch.int64, 2**40)):
        off = torch.tensor([-big, 20, 20, big], dtype=dt, device=dev)
        assert torch.equal(tb.grouped_gemm(1.0, A.to(dev), B.to(dev), off), want)
    # decreasing offsets: any values, but nothing outside the operands is touched
    off = torch.tensor([40, 10, 60, 0], dtype=torch.int32, device=dev)
    assert tb.grouped_gemm(1.0, A.to(dev), B.to(dev), off).shape == (50, 16)
    assert tb.grouped_rank_k(1.0, A.to(dev), A.to(dev), off).shape == (3, 32, 32)


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradients(dev, dtype):
    rows, sizes, lead = GROUPS["gaps"]
    off = _split(rows, sizes, lead)
    g = torch.Generator().manual_seed(7)
    for transB in (False, True):
        K, N = 72, 136
        A = _randn(g, rows, K, dtype=dtype)
        B = _randn(g, len(sizes), *((N, K) if transB else (K, N)), dtype=dtype)
        dD = _randn(g, rows, N, dtype=dtype)
        a, b = A.to(dev).requires_grad_(), B.to(dev).requires_grad_()
        D = tb.grouped_gemm(1.0, a, b, off.to(dev), transB=transB)
        dA, dB = torch.autograd.grad(D, (a, b), dD.to(dev))
        assert og.excess(D, *og.grouped_gemm(1.0, A, B, off, transB=transB), K) <= 1
        assert og.excess(dA, *og.grouped_gemm(1.0, dD, B, off, transB=not transB), N) <= 1
        want = og.grouped_rank_k(1.0, dD, A, off) if transB else og.grouped_rank_k(1.0, A, dD, off)
        assert og.excess(dB, *want, rows) <= 1 and dB.shape == B.shape


def test_other_stream(dev):
    g = torch.Generator().manual_seed(8)
    A, B, off = _randn(g, 90, 64).to(dev), _randn(g, 3, 64, 48).to(dev), _split(90, [30, 1, 59]).to(dev)
    want = tb.grouped_gemm(1.0, A, B, off)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        big = torch.randn(2048, 2048, device=dev)
        for _ in range(4):
            big = big @ big * 1e-3  # keeps the stream busy: a launch elsewhere would read A too early
        A2 = A + 0 * big[0, 0].nan_to_num(0.0, 0.0, 0.0)
        got = tb.grouped_gemm(1.0, A2, B, off)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype,K,N", [(BF16, 128, 256), (F16, 61, 33), (F32, 64, 48)])
def test_captured_graph_serves_any_routing(dev, dtype, K, N):
    g = torch.Generator().manual_seed(9)
    A, B, W = (_randn(g, *s, dtype=dtype).to(dev) for s in ((96, K), (6, K, N), (96, N)))
    off = _split(96, [16] * 6).to(dev)

    def both():
        return tb.grouped_gemm(1.0, A, B, off), tb.grouped_rank_k(1.0, A, W, off)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        both()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        D, P = both()
    for sizes in ([16] * 6, [0, 0, 96, 0, 0, 0], [1, 2, 3, 4, 5, 6], [40, 0, 40, 0, 1, 0]):
        off.copy_(_split(96, sizes))
        graph.replay()
        torch.cuda.synchronize()
        want = both()
        torch.cuda.synchronize()
        assert torch.equal(D, want[0]) and torch.equal(P, want[1])


def test_long_rows_pass_32_bit_offsets(dev):
    # rows whose byte offsets pass 2^32, and a B whose groups lie 2^32 bytes apart
    ld = 1 << 20
    A = torch.empty(2200, ld, dtype=BF16, device=dev)[:, :64]
    B = torch.empty(3, ld, 1024, dtype=BF16, device=dev)[:, :64, :72]
    g = torch.Generator().manual_seed(10)
    Ah, Bh = _randn(g, 2200, 64, dtype=BF16), _randn(g, 3, 64, 72, dtype=BF16)
    A.copy_(Ah)
    B.copy_(Bh)
    off = _split(2200, [2100, 0, 100])
    D = tb.grouped_gemm(1.0, A, B, off.to(dev))
    assert og.excess(D, *og.grouped_gemm(1.0, Ah, Bh, off), 64) <= 1
    W = _randn(g, 2200, 40, dtype=BF16)
    P = tb.grouped_rank_k(1.0, A, W.to(dev), off.to(dev))
    assert og.excess(P, *og.grouped_rank_k(1.0, Ah, W, off), 2100) <= 1


# Sizes that reach each kernel: (groups, rows, K, N). 256 x 256 tiles with whole rounds and a last one in quarters, with
# ragged ends of rows, columns and K, K of fewer values than a k-tile, and an odd number of k-tiles.
REACH = {
    "ring_kernel 256 x 256": [(3, 5200, 520, 2312), (1, 7000, 1160, 2568)],
    "ring_kernel 128 x 128": [(5, 20000, 2056, 1032), (3, 2600, 1032, 1288), (5, 9000, 40, 2304)],
    "ring_kernel 64 x 128": [(8, 1500, 264, 1032), (8, 900, 520, 264), (3, 500, 72, 1032)],
    "rows_kernel": [(8, 8, 1032, 520), (5, 60, 264, 136)],
}


def _excess_gpu(D, ref, den, k):
    return og.excess(D.cpu(), ref.cpu(), den.cpu(), k)


@pytest.mark.parametrize("kernel", list(REACH))
@pytest.mark.parametrize("transB", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_each_kernel_of_grouped_gemm(dev, dtype, transB, kernel):
    for i, (G, R, K, N) in enumerate(REACH[kernel]):
        if dtype != F32:
            assert _plan(0, dtype, transB, G, R, 0, N, K) == kernel
        g = torch.Generator(device=dev).manual_seed(i)
        off = _uneven(G, R, i)
        A = torch.randn(R, K, generator=g, device=dev).to(dtype)
        B = torch.randn(G, *((N, K) if transB else (K, N)), generator=g, device=dev).to(dtype)
        C = torch.randn(R, N, generator=g, device=dev).to(dtype)
        for beta in (0.0, 0.5):
            D = tb.grouped_gemm(1.0, A, B, off.to(dev), beta, C, transB=transB)
            ref = beta * C.double()
            den = ref.abs()
            for j, a, b in og.rows_of(off, R):
                W = (B[j].T if transB else B[j]).double().contiguous()
                ref[a:b] += A[a:b].double() @ W
                den[a:b] += A[a:b].double().abs() @ W.abs()
            assert _excess_gpu(D, ref, den, K) <= 1, (G, R, K, N, beta)


RANK_K = {  # (groups, rows, M, N)
    "ring_kernel 256 x 256": [(3, 9000, 2056, 2312)],
    "ring_kernel 128 x 128": [(8, 4100, 2056, 1032), (3, 2600, 1032, 1288)],
    "ring_kernel 64 x 128": [(8, 900, 264, 1032)],
}


@pytest.mark.parametrize("kernel", list(RANK_K))
@pytest.mark.parametrize("dtype", DTYPES)
def test_each_kernel_of_grouped_rank_k(dev, dtype, kernel):
    for i, (G, R, M, N) in enumerate(RANK_K[kernel]):
        if dtype != F32:
            assert _plan(1, dtype, 0, G, R, M, N, 0) == kernel
        g = torch.Generator(device=dev).manual_seed(i)
        off = _uneven(G, R, i)
        A = torch.randn(R, M, generator=g, device=dev).to(dtype)
        B = torch.randn(R, N, generator=g, device=dev).to(dtype)
        C = torch.randn(G, M, N, generator=g, device=dev)
        ref, den = torch.zeros(2, G, M, N, dtype=torch.float64, device=dev)
        for j, a, b in og.rows_of(off, R):
            left = A[a:b].double().T.contiguous()
            ref[j], den[j] = left @ B[a:b].double(), left.abs() @ B[a:b].double().abs()
        assert _excess_gpu(tb.grouped_rank_k(1.0, A, B, off.to(dev)), ref, den, R) <= 1, (G, R, M, N)
        D = tb.grouped_rank_k(1.0, A, B, off.to(dev), 1.0, C, dtype=F32)
        assert _excess_gpu(D, ref + C.double(), den + C.double().abs(), R) <= 1, (G, R, M, N)


@pytest.mark.parametrize("dtype", DTYPES)
def test_packed_operands(dev, dtype):
    # large operands that start or end anywhere are copied first; the results are those of aligned ones
    G, R, K, N = 3, 4099, 1021, 2043
    for transB in (False, True):
        g = torch.Generator(device=dev).manual_seed(1)
        off = _uneven(G, R, 1)
        A = torch.randn(R, K + 3, generator=g, device=dev).to(dtype)[:, 1:-2]
        B = torch.randn(G, *((N, K) if transB else (K, N)), generator=g, device=dev).to(dtype)
        D = tb.grouped_gemm(1.0, A, B, off.to(dev), transB=transB)
        dB = tb.grouped_rank_k(1.0, A, D, off.to(dev))
        ref, den = torch.zeros(2, R, N, dtype=torch.float64, device=dev)
        for j, a, b in og.rows_of(off, R):
            W = (B[j].T if transB else B[j]).double().contiguous()
            ref[a:b], den[a:b] = A[a:b].double() @ W, A[a:b].double().abs() @ W.abs()
        assert _excess_gpu(D, ref, den, K) <= 1
        ref, den = torch.zeros(2, G, K, N, dtype=torch.float64, device=dev)
        for j, a, b in og.rows_of(off, R):
            left = A[a:b].double().T.contiguous()
            ref[j], den[j] = left @ D[a:b].double(), left.abs() @ D[a:b].double().abs()
        assert _excess_gpu(dB, ref, den, R) <= 1


def _amid_nans(x, left):
    """x as a view of a larger buffer of NaNs, its rows starting anywhere."""
    buf = torch.full((*x.shape[:-2], x.shape[-2] + 2, x.shape[-1] + left + 3), float("nan"), dtype=x.dtype, device=x.device)
    view = buf[..., 1:-1, left : left + x.shape[-1]]
    return view.copy_(x)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K,N", [(1, 3), (3, 4), (4, 7), (5, 8), (7, 9), (8, 65), (9, 1), (31, 66), (33, 5), (64, 129), (65, 71)])
def test_extents_near_16_bytes_amid_nans(dev, dtype, K, N):
    # rows shorter than, equal to and just past 16 bytes; nothing from outside an operand reaches a sum
    G, R = 2, 213
    g = torch.Generator(device=dev).manual_seed(K)
    off = torch.tensor([1, 70, 211])
    A = torch.randn(R, K, generator=g, device=dev).to(dtype)
    dD = torch.randn(R, N, generator=g, device=dev).to(dtype)
    for transB in (False, True):
        B = torch.randn(G, *((N, K) if transB else (K, N)), generator=g, device=dev).to(dtype)
        D = tb.grouped_gemm(1.0, _amid_nans(A, 1), _amid_nans(B, 3), off.to(dev), transB=transB)
        assert og.excess(D.cpu(), *og.grouped_gemm(1.0, A.cpu(), (B.mT if transB else B).cpu(), off), K) <= 1
    P = tb.grouped_rank_k(1.0, _amid_nans(A, 1), _amid_nans(dD, 3), off.to(dev))
    assert og.excess(P.cpu(), *og.grouped_rank_k(1.0, A.cpu(), dD.cpu(), off), R) <= 1


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("G", [4, 8, 16])  # 4, 2 and 1 waves of a workgroup along K
def test_few_rows_of_large_matrices(dev, dtype, G):
    K, N = 2056, 4104
    R = G + 3
    assert _plan(0, dtype, 1, G, R, 0, N, K) == "rows_kernel"
    g = torch.Generator(device=dev).manual_seed(G)
    off = torch.arange(G + 1) + 1
    off[2:] += 1
    A = torch.randn(R, K, generator=g, device=dev).to(dtype)
    B = torch.randn(G, N, K, generator=g, device=dev).to(dtype)
    D = tb.grouped_gemm(1.0, A, B, off.to(dev), transB=True)
    ref, den = torch.zeros(2, R, N, dtype=torch.float64, device=dev)
    for j, a, b in og.rows_of(off, R):
        W = B[j].double().T.contiguous()
        ref[a:b], den[a:b] = A[a:b].double() @ W, A[a:b].double().abs() @ W.abs()
    assert _excess_gpu(D, ref, den, K) <= 1


@pytest.mark.parametrize("dtype", DTYPES)
def test_forward_mode_tangents(dev, dtype):
    from torch.autograd import forward_ad as fwd

    rows, sizes, lead = GROUPS["gaps"]
    off = _split(rows, sizes, lead)
    g = torch.Generator().manual_seed(11)
    A, B, W = (_randn(g, *s, dtype=dtype) for s in ((rows, 72), (len(sizes), 72, 40), (rows, 40)))
    tA, tB, tW = (_randn(g, *x.shape, dtype=dtype) for x in (A, B, W))
    with fwd.dual_level():
        dual = lambda x, t: fwd.make_dual(x.to(dev), t.to(dev))
        D = fwd.unpack_dual(tb.grouped_gemm(1.0, dual(A, tA), dual(B, tB), off.to(dev)))
        P = fwd.unpack_dual(tb.grouped_rank_k(1.0, dual(A, tA), dual(W, tW), off.to(dev)))
        one = fwd.unpack_dual(tb.grouped_gemm(1.0, A.to(dev), dual(B, tB), off.to(dev)))
        M = fwd.unpack_dual(tb.gemm(1.0, dual(A, tA), dual(B, tB).select(0, 1)))
    a, b = og.grouped_gemm(1.0, tA, B, off), og.grouped_gemm(1.0, A, tB, off)
    assert og.excess(D.primal, *og.grouped_gemm(1.0, A, B, off), 72) <= 1
    assert og.excess(D.tangent, a[0] + b[0], a[1] + b[1], 2 * 72) <= 1
    assert og.excess(one.tangent, *b, 72) <= 1
    a, b = og.grouped_rank_k(1.0, tA, W, off), og.grouped_rank_k(1.0, A, tW, off)
    assert og.excess(P.tangent, a[0] + b[0], a[1] + b[1], 2 * rows) <= 1
    assert M.tangent is not None


def test_negated_views(dev):
    # the imaginary part of a conjugate is a view whose values stand in memory with the other sign
    for R, K, N in ((150, 64, 128), (150, 1, 1), (150, 33, 1), (4099, 1021, 2043)):  # the last is packed
        off = _split(R, [17, 33, 1, 64, R - 115])
        g = torch.Generator(device=dev).manual_seed(K)
        z = lambda *s: torch.randn(*s, 2, generator=g, device=dev)
        conj = lambda x: torch.view_as_complex(x).conj().imag
        a, b, w, c = z(R, K), z(5, K, N), z(R, N), z(R, N)
        A, B, W, C = (conj(x) for x in (a, b, w, c))
        assert all(x.is_neg() for x in (A, B, W, C))
        D = tb.grouped_gemm(1.0, A, B, off.to(dev), 0.5, C)
        assert og.excess(D, *og.grouped_gemm(1.0, -a[..., 1].cpu(), -b[..., 1].cpu(), off, 0.5, -c[..., 1].cpu()), K) <= 1
        D = tb.grouped_gemm(1.0, -a[..., 1], B, off.to(dev))
        assert og.excess(D, *og.grouped_gemm(1.0, -a[..., 1].cpu(), -b[..., 1].cpu(), off), K) <= 1
        D = tb.grouped_rank_k(1.0, A, W, off.to(dev))
        assert og.excess(D, *og.grouped_rank_k(1.0, -a[..., 1].cpu(), -w[..., 1].cpu(), off), R) <= 1
        D = tb.grouped_rank_k(1.0, A, -w[..., 1], off.to(dev))
        assert og.excess(D, *og.grouped_rank_k(1.0, -a[..., 1].cpu(), -w[..., 1].cpu(), off), R) <= 1


# fp32 results of 16-bit operands: sums in chains of at most 4096 values, of which the largest error on same-sign values was
# measured as 1.43e-6 |A||B| (a single chain: 2.2e-6 after 8192, 3.9e-6 after 32768); several chains average their errors.
CHAIN_GATE = 2e-6
LONG = {  # (op, groups, rows, M, N, K)
    "ring_kernel 256 x 256": [(1, 3, 36000, 2056, 2312, 0), (0, 3, 5200, 0, 2312, 16392)],
    "ring_kernel 128 x 128": [(1, 2, 36000, 1032, 1288, 0), (0, 3, 2600, 0, 1288, 16392)],
    "ring_kernel 64 x 128": [(1, 2, 36000, 264, 520, 0), (0, 1, 600, 0, 520, 33000)],
    "rows_kernel": [(0, 1, 9, 0, 520, 66000)],
    "ring_kernel 64 x 128, rows_kernel": [(0, 8, 9, 0, 4104, 33000)],  # by transB
    "grouped_any_kernel": [(1, 2, 36000, 129, 260, 0), (0, 2, 70, 0, 260, 33001)],
}


def _gemm_ref(A, B, off, transB):
    """(A B, |A| |B|) in float64 on A's device."""
    ref, den = torch.zeros(2, A.shape[0], B.shape[1 if transB else 2], dtype=torch.float64, device=A.device)
    for j, a, b in og.rows_of(off, A.shape[0]):
        W = (B[j].T if transB else B[j]).double().contiguous()
        ref[a:b], den[a:b] = A[a:b].double() @ W, A[a:b].double().abs() @ W.abs()
    return ref, den


def _rank_k_ref(A, B, off):
    ref, den = torch.zeros(2, off.shape[0] - 1, A.shape[1], B.shape[1], dtype=torch.float64, device=A.device)
    for j, a, b in og.rows_of(off, A.shape[0]):
        left = A[a:b].double().T.contiguous()
        ref[j], den[j] = left @ B[a:b].double(), left.abs() @ B[a:b].double().abs()
    return ref, den


def _relative(D, ref, den):
    return float(((D.double() - ref).abs() / den.clamp_min(2.0**-100)).max())


@pytest.mark.parametrize("kernel", list(LONG))
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_fp32_results_of_16_bit_operands_over_long_k(dev, dtype, kernel):
    for i, (op, G, R, M, N, K) in enumerate(LONG[kernel]):
        g = torch.Generator(device=dev).manual_seed(i)
        rand = lambda *s: torch.rand(*s, generator=g, device=dev).to(dtype)
        off = _uneven(G, R, i)
        for transB in (False, True) if op == 0 else (False,):
            assert _plan(op, dtype, transB, G, R, M, N, K) == kernel.split(", ")[-1 if transB else 0]
            if op == 0:
                A, B = rand(R, K), rand(G, *((N, K) if transB else (K, N)))
                ref, den = _gemm_ref(A, B, off, transB)
                call = lambda *c: tb.grouped_gemm(1.0, A, B, off.to(dev), *c, transB=transB, dtype=F32)
            else:
                A, B = rand(R, M), rand(R, N)
                ref, den = _rank_k_ref(A, B, off)
                call = lambda *c: tb.grouped_rank_k(1.0, A, B, off.to(dev), *c, dtype=F32)
            assert _relative(call(), ref, den) <= CHAIN_GATE, (op, G, R, transB)
            C = 100.0 * torch.rand(ref.shape, generator=g, device=dev)
            assert _relative(call(0.5, C), ref + 0.5 * C.double(), den + 0.5 * C.double()) <= CHAIN_GATE, (op, G, R, transB)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_gradient_of_an_fp32_result_is_not_rounded(dev, dtype):
    # its values pass the range of fp16 and fall below it, and have more bits than a 16-bit type holds
    rows, sizes, K, N = 60, [9, 21, 0, 25], 24, 40
    off = _split(rows, sizes)
    g = torch.Generator().manual_seed(12)
    A, B = (torch.randn(rows, K, generator=g) * 1e-3).to(dtype), (torch.randn(4, K, N, generator=g) * 2e-3).to(dtype)
    dD = torch.randn(rows, N, generator=g) * torch.tensor([1e5, 1e-5]).repeat_interleave(rows // 2)[:, None]
    for transB in (False, True):
        b0 = B.mT.contiguous() if transB else B
        a, b = A.to(dev).requires_grad_(), b0.to(dev).requires_grad_()
        D = tb.grouped_gemm(2.0, a, b, off.to(dev), transB=transB, dtype=torch.float32)
        dA, dB = torch.autograd.grad(D, (a, b), dD.to(dev))
        assert dA.dtype == dB.dtype == dtype
        assert og.excess(dA, *og.grouped_gemm(2.0, dD, b0, off, transB=not transB), N) <= 1
        assert og.excess(dB, *og.grouped_rank_k(2.0, *((dD, A) if transB else (A, dD)), off), rows) <= 1
    W, dP = (torch.randn(rows, N, generator=g) * 1e-3).to(dtype), torch.randn(4, K, N, generator=g) * 1e5
    a, w = A.to(dev).requires_grad_(), W.to(dev).requires_grad_()
    dA, dW = torch.autograd.grad(tb.grouped_rank_k(1.0, a, w, off.to(dev), dtype=torch.float32), (a, w), dP.to(dev))
    assert og.excess(dA, *og.grouped_gemm(1.0, W, dP.mT, off), N) <= 1
    assert og.excess(dW, *og.grouped_gemm(1.0, A, dP, off), K) <= 1


# fp32 sums restart every 64 values of k (up to 1024 in long ones), so same-sign products keep `gemm`'s gate on each kernel:
# (groups, rows, N, K)
FP32 = {
    "ring_kernel 64 x 128": [(3, 5200, 2312, 4100), (3, 2600, 1288, 1032)],
    "rows_kernel": [(8, 8, 520, 4100), (5, 60, 136, 264)],
    "grouped_any_kernel": [(2, 900, 520, 4104), (16, 32, 2056, 1032)],
}


@pytest.mark.parametrize("kernel", list(FP32))
@pytest.mark.parametrize("transB", [False, True])
def test_each_fp32_kernel_keeps_the_fp32_gate(dev, transB, kernel):
    for i, (G, R, N, K) in enumerate(FP32[kernel]):
        assert _plan(0, F32, transB, G, R, 0, N, K) == kernel
        g = torch.Generator(device=dev).manual_seed(i)
        off = _uneven(G, R, i) if R > 4 * G else torch.arange(G + 1) * (R // G)
        A = torch.rand(R, K, generator=g, device=dev)
        B = torch.rand(G, *((N, K) if transB else (K, N)), generator=g, device=dev)
        C = torch.rand(R, N, generator=g, device=dev)
        ref, den = _gemm_ref(A, B, off, transB)
        D = tb.grouped_gemm(1.0, A, B, off.to(dev), transB=transB)
        assert _relative(D, ref, den) <= 1e-6, (G, R, N, K)
        D = tb.grouped_gemm(1.0, A, B, off.to(dev), 0.5, C, transB=transB)
        assert _relative(D, ref + 0.5 * C.double(), den + 0.5 * C.double()) <= 1e-6, (G, R, N, K)


@pytest.mark.parametrize("dtype,waves,G,R,N,K", [
    (F32, 8, 8, 24, 520, 4104), (F32, 4, 23, 184, 752, 1412), (F32, 1, 33, 165, 18400, 132),
    (BF16, 8, 8, 64, 296, 1832), (BF16, 4, 39, 234, 480, 1504), (F16, 2, 38, 152, 1328, 560), (BF16, 1, 33, 132, 5304, 144),
])  # fmt: skip
def test_each_form_of_the_few_rows_kernel(dev, dtype, waves, G, R, N, K):
    # K-contiguous matrices, one block of 16 rows; one group fills it where it can
    assert rows_plan(0, dtype, 1, G, R, N, K) == (1, waves, 0)
    g = torch.Generator(device=dev).manual_seed(R)
    sizes = torch.bincount(torch.arange(R - min(R, 16)) % (G - 1) + 1, minlength=G)
    sizes[0] = min(R, 16)
    off = _split(R, sizes.tolist())
    A = torch.randn(R, K, generator=g, device=dev).to(dtype)
    B = torch.randn(G, N, K, generator=g, device=dev).to(dtype)
    ref, den = _gemm_ref(A, B, off, True)
    D = tb.grouped_gemm(1.0, A, B, off.to(dev), transB=True)
    assert _excess_gpu(D, ref, den, K) <= 1


@pytest.mark.parametrize("G,R,N,K", [(3, 5200, 2313, 16392), (3, 2600, 1290, 16392), (1, 600, 519, 33000), (1, 300, 37, 8200)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_chains_into_rows_that_start_anywhere(dev, dtype, G, R, N, K):
    # results whose rows are no multiple of 16 bytes go out through LDS, and each further chain takes them up from there
    g = torch.Generator(device=dev).manual_seed(N)
    off = _uneven(G, R, 1)
    A, B = torch.rand(R, K, generator=g, device=dev).to(dtype), torch.rand(G, N, K, generator=g, device=dev).to(dtype)
    C = 100.0 * torch.rand(R, N, generator=g, device=dev)
    ref, den = _gemm_ref(A, B, off, True)
    D = tb.grouped_gemm(1.0, A, B, off.to(dev), transB=True, dtype=F32)
    assert _relative(D, ref, den) <= CHAIN_GATE and not D[int(off[-1]) :].any()
    D = tb.grouped_gemm(-2.0, A, B, off.to(dev), 0.5, C, transB=True, dtype=F32)
    assert _relative(D, -2.0 * ref + 0.5 * C.double(), 2.0 * den + 0.5 * C.double()) <= CHAIN_GATE


@pytest.mark.parametrize("blocks,waves,transB,G,R,N,K", [
    (1, 8, 0, 2, 9, 72, 33000), (2, 8, 0, 1, 20, 72, 33000), (1, 8, 1, 2, 9, 72, 33000), (2, 8, 1, 1, 20, 72, 33000),
    (1, 4, 1, 8, 16, 2056, 16400), (1, 2, 1, 64, 128, 480, 8200), (1, 1, 1, 16, 32, 4104, 4104),
])  # fmt: skip
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_chains_of_the_few_rows_kernel(dev, dtype, blocks, waves, transB, G, R, N, K):
    # a wave's share of k is longer than a chain
    assert rows_plan(0, dtype, transB, G, R, N, K) == (blocks, waves, 0)
    g = torch.Generator(device=dev).manual_seed(K)
    off = torch.arange(G + 1) * (R // G)
    A = torch.rand(R, K, generator=g, device=dev).to(dtype)
    B = torch.rand(G, *((N, K) if transB else (K, N)), generator=g, device=dev).to(dtype)
    ref, den = _gemm_ref(A, B, off, transB)
    assert _relative(tb.grouped_gemm(1.0, A, B, off.to(dev), transB=bool(transB), dtype=F32), ref, den) <= CHAIN_GATE


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_chains_of_rows_shorter_than_16_bytes(dev, dtype):
    g = torch.Generator(device=dev).manual_seed(13)
    rand = lambda *s: torch.rand(*s, generator=g, device=dev).to(dtype)
    off = _split(36000, [20000, 0, 15990], 4)
    for M, N in ((5, 260), (260, 3), (1, 1)):
        A, B = rand(36000, M), rand(36000, N)
        assert _relative(tb.grouped_rank_k(1.0, A, B, off.to(dev), dtype=F32), *_rank_k_ref(A, B, off)) <= CHAIN_GATE, (M, N)
    off = _split(70, [33, 30], 4)
    for N in (1, 5):
        A, B = rand(70, 33001), rand(2, 33001, N)
        assert _relative(tb.grouped_gemm(1.0, A, B, off.to(dev), dtype=F32), *_gemm_ref(A, B, off, False)) <= CHAIN_GATE, N
