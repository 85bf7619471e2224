"""gated_gemm / grouped_gated_gemm on the GPU against 64-bit formulas, at sizes, layouts and group shapes where they can go
wrong. Bounds: `oracle.gated`'s, from the roundings that the arithmetic makes."""

import pytest
import torch

import trnblas_amd as tb
from oracle import gated as og
from oracle import grouped as gg
from oracle.grouped import GROUPS
from oracle.grouped import split as _split
from oracle.grouped import uneven as _uneven

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
DTYPES = [F32, BF16, F16]


def _operands(seed, dtype, rows, K, N, groups, transB, device="cpu"):
    g = torch.Generator(device=device).manual_seed(seed)
    A = torch.randn(rows, K, generator=g, device=device).to(dtype)
    B = torch.randn(groups, *((2 * N, K) if transB else (K, 2 * N)), generator=g, device=device) * max(K, 1) ** -0.5
    return A, B.to(dtype)


def _holds(H, A, B, off, transB, act):
    P, den = og.products(A, B, off, transB)
    return og.ratio(H, *og.forward(act, P, den, A.shape[1], H.dtype)) <= 1


def _plan(dtype, transB, groups, rows, N, K):
    from trnblas_amd.hip import _lib

    return _lib.load().trnblas_hip_gated_plan(_lib.DTYPE_CODES[dtype], transB, groups, rows, N, K).decode()


# (dtype, transB, groups, rows, N, K) that each kernel serves: results that end inside a tile
REACH = {
    "gated_ring_kernel 256 x 128": [(BF16, 0, 8, 2600, 2056, 264), (F16, 1, 8, 2600, 2056, 520), (BF16, 1, 8, 5200, 1032, 264)],
    "gated_ring_kernel 128 x 64": [(F16, 0, 40, 9000, 264, 72), (BF16, 1, 1, 900, 4104, 136)],
    "gated_ring_kernel 64 x 64": [(BF16, 0, 3, 300, 520, 264), (F16, 1, 3, 300, 520, 1032), (F32, 0, 3, 300, 520, 260), (F32, 1, 1, 900, 260, 516)],
    "rows_kernel 16 1": [(BF16, 1, 64, 64, 2056, 72), (F16, 1, 40, 40, 4104, 72), (F32, 1, 64, 64, 1032, 68)],
    "rows_kernel 16 2": [(BF16, 1, 8, 8, 4104, 1032), (F16, 1, 64, 64, 520, 1040)],
    "rows_kernel 16 4": [(BF16, 1, 8, 8, 2056, 1032), (F16, 1, 64, 64, 264, 1040)],
    "rows_kernel 16 8": [(BF16, 0, 1, 3, 72, 264), (F16, 1, 3, 3, 72, 1032), (F32, 0, 3, 3, 72, 260), (F32, 1, 1, 1, 72, 4100)],
    "rows_kernel 32 8": [(BF16, 0, 1, 20, 72, 264), (F16, 1, 3, 27, 72, 520)],
}


@pytest.mark.parametrize("kernel", list(REACH))
def test_each_kernel(dev, kernel):
    for i, (dtype, transB, G, R, N, K) in enumerate(REACH[kernel]):
        assert _plan(dtype, transB, G, R, N, K) == kernel, (dtype, transB, G, R, N, K)
        A, B = _operands(i, dtype, R, K, N, G, transB, dev)
        off = _uneven(G, R, i) if R > 4 * G else torch.arange(G + 1) * (R // G)
        act = og.ACTS[i % 5]
        H = tb.grouped_gated_gemm(A, B, off.to(dev), act, transB=bool(transB))
        assert _holds(H, A, B, off, transB, act), (dtype, transB, G, R, N, K)
        # with what a backward pass needs of it beside it: the same values, and both sums
        P, den = og.products(A, B, off, transB)
        from trnblas_amd.hip import gated_kernels

        H2, S = gated_kernels.gated_gemm(A, B.mT if transB else B, off.to(dev), act, dtype, True)
        assert torch.equal(H2, H)
        e = (K + 2) * 2.0**-23 * den
        assert og.ratio(S, P, e + og.EPS[dtype] * (P.abs() + e) + og.TINY[dtype]) <= 1
        if K % 8 == 0 and transB:  # columns that are no multiple of four: results go out value by value
            b = B[:, : 2 * (N - 3)].contiguous()
            H = tb.grouped_gated_gemm(A, b, off.to(dev), act, transB=True)
            assert _holds(H, A, b, off, True, act)
            H2, S = gated_kernels.gated_gemm(A, b.mT, off.to(dev), act, dtype, True)
            P, den = og.products(A, b, off, True)
            e = (K + 2) * 2.0**-23 * den
            assert torch.equal(H2, H) and og.ratio(S, P, e + og.EPS[dtype] * (P.abs() + e) + og.TINY[dtype]) <= 1


def test_packed_operands(dev):
    # large ones that LDS DMA cannot read in place
    for dtype, R, K, N, transB in ((BF16, 1100, 1021, 515, False), (F16, 1100, 1021, 515, True), (BF16, 1100, 1024, 515, False), (F32, 1100, 1021, 515, False)):
        A, B = _operands(R, dtype, R, K, N, 1, transB, dev)
        off = torch.tensor([0, R])
        for a in (A, torch.nn.functional.pad(A, (1, 2))[:, 1 : K + 1]):
            assert _holds(tb.gated_gemm(a, B[0], transB=transB), A, B, off, transB, "silu"), (dtype, K, transB)
        a, b = A.requires_grad_(), B[0].requires_grad_()
        dH = torch.randn(R, N, generator=torch.Generator(device=dev).manual_seed(1), device=dev).to(dtype)
        grads = torch.autograd.grad(tb.gated_gemm(a, b, transB=transB), (a, b), dH)
        assert _gradients_hold([grads[0], grads[1][None]], A.detach(), B.detach(), off, transB, "silu", dH, dtype)


# (K, N): below and across the tiles of 16, 32, 64 and 128 columns, multiples of 16 bytes and not
SIZES = [(1, 1), (7, 5), (33, 70), (64, 128), (100, 61), (136, 264), (264, 136), (512, 520), (515, 257), (1032, 384)]


@pytest.mark.parametrize("shape", list(GROUPS))
@pytest.mark.parametrize("dtype", DTYPES)
def test_grouped(dev, shape, dtype):
    rows, sizes, lead = GROUPS[shape]
    off = _split(rows, sizes, lead)
    for i, (K, N) in enumerate(SIZES):
        for transB in (False, True):
            A, B = _operands(100 * i + transB, dtype, rows, K, N, len(sizes), transB)
            act = og.ACTS[i % 3]
            H = tb.grouped_gated_gemm(A.to(dev), B.to(dev), off.to(dev), act, transB=transB)
            assert H.dtype == dtype and _holds(H, A, B, off, transB, act), (K, N, transB)


@pytest.mark.parametrize("act", og.ACTS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_dense(dev, dtype, act):
    for i, (R, K, N) in enumerate([(1, 64, 128), (3, 515, 257), (16, 4104, 72), (17, 256, 64), (70, 33, 61), (129, 136, 264),
                                   (300, 520, 136), (513, 64, 1032)]):  # fmt: skip
        for transB in (False, True):
            A, B = _operands(i, dtype, R, K, N, 1, transB)
            off = torch.tensor([0, R])
            for out in {dtype, F32}:
                H = tb.gated_gemm(A.to(dev), B[0].to(dev), act, transB=transB, dtype=out)
                assert H.dtype == out and _holds(H, A, B, off, transB, act), (R, K, N, transB, out)


def _gradients_hold(grads, A, B, off, transB, act, dH, out):
    """dA and dB against the formula: dP is off by its bound (rounded to `out`), the products by fp32 sums and one rounding."""
    dtype, K = A.dtype, A.shape[1]
    P, den = og.products(A, B, off, transB)
    dP, e = og.backward(act, P, dH), og.gradient_bounds(act, P, den, dH, K, out)
    Bk = B.mT if transB else B
    want, bound = torch.zeros(A.shape, dtype=torch.float64, device=A.device), og.TINY[dtype] * torch.ones_like(A, dtype=torch.float64)
    dB, eB = torch.zeros(Bk.shape, dtype=torch.float64, device=A.device), torch.full(Bk.shape, og.TINY[dtype], dtype=torch.float64, device=A.device)
    for j, a, b in gg.rows_of(off, A.shape[0]):
        W = Bk[j].double().T.contiguous()
        X = A[a:b].double().T.contiguous()
        want[a:b] = dP[a:b] @ W
        bound[a:b] += e[a:b] @ W.abs() + (Bk.shape[2] + 2) * 2.0**-23 * ((dP[a:b].abs() + e[a:b]) @ W.abs())
        dB[j] = X @ dP[a:b]
        eB[j] += X.abs() @ e[a:b] + (b - a + 2) * 2.0**-23 * (X.abs() @ (dP[a:b].abs() + e[a:b]))
    bound, eB = bound + og.EPS[dtype] * (want.abs() + bound), eB + og.EPS[dtype] * (dB.abs() + eB)
    if transB:
        dB, eB = dB.mT, eB.mT
    return og.ratio(grads[0], want, bound) <= 1 and og.ratio(grads[1], dB, eB) <= 1


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "sigmoid"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_gradients(dev, dtype, act):
    for i, (shape, K, N) in enumerate([("one", 40, 8), ("token", 33, 17), ("gaps", 136, 72), ("small", 64, 128),
                                       ("uneven", 264, 136), ("uneven", 100, 61), ("single", 520, 257)]):  # fmt: skip
        rows, sizes, lead = GROUPS[shape]
        off = _split(rows, sizes, lead)
        for transB in (False, True):
            A, B = _operands(i, dtype, rows, K, N, len(sizes), transB)
            dH = torch.randn(rows, N, generator=torch.Generator().manual_seed(i))
            for out in {dtype, F32}:
                a, b = A.to(dev).requires_grad_(), B.to(dev).requires_grad_()
                H = tb.grouped_gated_gemm(a, b, off.to(dev), act, transB=transB, dtype=out)
                assert _holds(H, A, B, off, transB, act)
                grads = torch.autograd.grad(H, (a, b), dH.to(dev, out))
                assert _gradients_hold([x.cpu() for x in grads], A, B, off, transB, act, dH.to(out), out), (shape, K, N, transB, out)


@pytest.mark.parametrize("dtype", DTYPES)
def test_dense_gradients(dev, dtype):
    for R, K, N in ((1, 24, 8), (130, 264, 72), (257, 61, 33)):
        off = torch.tensor([0, R])
        for transB in (False, True):
            A, B = _operands(R, dtype, R, K, N, 1, transB)
            dH = torch.randn(R, N, generator=torch.Generator().manual_seed(1)).to(dtype)
            a, b = A.to(dev).requires_grad_(), B[0].to(dev).requires_grad_()
            grads = torch.autograd.grad(tb.gated_gemm(a, b, "gelu", transB=transB), (a, b), dH.to(dev))
            assert _gradients_hold([grads[0].cpu(), grads[1].cpu()[None]], A, B, off, transB, "gelu", dH, dtype), (R, transB)
            # each alone, and a gradient that is one value for all
            one = torch.ones((), dtype=dtype, device=dev).expand(R, N)
            x = torch.autograd.grad(tb.gated_gemm(a, b.detach(), "gelu", transB=transB), a, one)[0]
            y = torch.autograd.grad(tb.gated_gemm(a.detach(), b, "gelu", transB=transB), b, one)[0]
            assert _gradients_hold([x.cpu(), y.cpu()[None]], A, B, off, transB, "gelu", torch.ones(R, N), dtype), (R, transB)


def test_gradients_against_differences(dev):
    g = torch.Generator().manual_seed(3)
    A, B = torch.randn(9, 12, generator=g).to(dev), torch.randn(2, 12, 16, generator=g).to(dev)
    tA, tB = torch.randn(9, 12, generator=g).to(dev), torch.randn(2, 12, 16, generator=g).to(dev)
    off = torch.tensor([1, 4, 8], device=dev)
    dH = torch.randn(9, 8, generator=g).to(dev)
    for act in ("silu", "gelu", "gelu_tanh", "sigmoid"):
        f = lambda h: (tb.grouped_gated_gemm(A + h * tA, B + h * tB, off, act) * dH).double().sum()
        a, b = A.clone().requires_grad_(), B.clone().requires_grad_()
        dA, dB = torch.autograd.grad(tb.grouped_gated_gemm(a, b, off, act), (a, b), dH)
        want = float((dA * tA).double().sum() + (dB * tB).double().sum())
        # a central difference of step 2^-6: its own error falls with the square of the step, fp32's grows with its inverse
        d = [float((f(h) - f(-h)) / (2 * h)) for h in (2.0**-6, 2.0**-5)]
        assert abs((4 * d[0] - d[1]) / 3 - want) <= 2e-3 * abs(want) + 2e-3


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(dev, dtype):
    # operands inside larger buffers, at any column and leading dimension, with NaN around them; results and gradients alike
    rows, K, N = 45, 72, 40
    off = _split(rows, [20, 0, 19], 3)
    for transB in (False, True):
        A, B = _operands(4, dtype, rows, K, N, 3, transB)
        want = tb.grouped_gated_gemm(A.to(dev), B.to(dev), off.to(dev), transB=transB)
        for left in (0, 1, 8):
            X = torch.full((rows, K + 24), float("nan"), dtype=dtype, device=dev)
            Y = torch.full((3, B.shape[1] + 3, B.shape[2] + 24), float("nan"), dtype=dtype, device=dev)
            X[:, left : left + K], Y[:, 2:-1, left : left + B.shape[2]] = A.to(dev), B.to(dev)
            x, y = X[:, left : left + K], Y[:, 2:-1, left : left + B.shape[2]]
            assert _holds(tb.grouped_gated_gemm(x, y, off.to(dev), transB=transB), A, B, off, transB, "silu")
            a, b = x.detach().requires_grad_(), y.detach().requires_grad_()
            dH = torch.ones_like(want)
            grads = torch.autograd.grad(tb.grouped_gated_gemm(a, b, off.to(dev), transB=transB), (a, b), dH)
            assert _gradients_hold([t.cpu() for t in grads], A, B, off, transB, "silu", dH.cpu(), dtype)
        # one matrix for all groups, and rows taken in steps
        one = B[:1].to(dev).expand(3, *B.shape[1:])
        H = tb.grouped_gated_gemm(A.to(dev), one, off.to(dev), transB=transB)
        assert _holds(H, A, B[:1].expand(3, *B.shape[1:]), off, transB, "silu")
        wide = torch.randn(rows, 2 * K, generator=torch.Generator().manual_seed(5)).to(dtype)
        assert _holds(tb.grouped_gated_gemm(wide.to(dev)[:, ::2], B.to(dev), off.to(dev), transB=transB), wide[:, ::2], B, off, transB, "silu")


@pytest.mark.parametrize("dtype", DTYPES)
def test_values_of_other_groups_stay_out(dev, dtype):
    for K, N in ((40, 72), (61, 33), (256, 256)):
        off = _split(60, [9, 21, 0, 5], 10)
        A, B = _operands(3, dtype, 60, K, N, 4, False)
        bad = A.clone(), B.clone()
        bad[0][:10], bad[0][19:40], bad[0][45:] = (float(x) for x in ("inf", "nan", "nan"))
        bad[1][1:3] = float("nan")
        want = tb.grouped_gated_gemm(A.to(dev), B.to(dev), off.to(dev))
        a, b = (x.to(dev).requires_grad_() for x in bad)
        got = tb.grouped_gated_gemm(a, b, off.to(dev))
        for i, j in ((10, 19), (40, 45)):
            assert torch.equal(got[i:j], want[i:j]) and want[i:j].isfinite().all()
        assert not got[:10].any() and not got[45:].any()
        # what stands in the gradient of rows of no group reaches no other gradient
        dH = torch.ones(60, N, dtype=dtype)
        dH[:10], dH[45:] = float("inf"), float("nan")
        dA, dB = torch.autograd.grad(got, (a, b), dH.to(dev))
        assert not dA[:10].any() and not dA[45:].any() and dA[10:19].isfinite().all() and dA[40:45].isfinite().all()
        assert dB[0].isfinite().all() and dB[3].isfinite().all() and not dB[2].any()


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_fp32_results_over_long_k(dev, dtype):
    # same-sign values: a 16-bit product's sums restart every 4096 values of k, which keeps them within 2e-6 of |A||B|
    K = 16400
    for R, N, transB in ((3, 40, True), (40, 72, False), (300, 136, True)):
        g = torch.Generator(device=dev).manual_seed(R)
        A = torch.rand(R, K, generator=g, device=dev).to(dtype)
        B = (torch.rand(*((2 * N, K) if transB else (K, 2 * N)), generator=g, device=dev) / K).to(dtype)
        H = tb.gated_gemm(A, B, "relu", transB=transB, dtype=F32)
        W = (B.T if transB else B).double().contiguous()
        P = A.double() @ W
        ref = P[:, :N] * P[:, N:]
        assert float(((H.double() - ref).abs() / ref).max()) <= 2 * 2e-6 + 2.0**-22, (R, N)


def test_activations_far_from_zero(dev):
    x = torch.tensor([-3e38, -1e20, -700.0, -90.0, -20.0, -3.0, 0.0, 3.0, 20.0, 90.0, 700.0, 1e20, 3e38])
    A = torch.stack([x, torch.ones_like(x)], 1)
    for act in og.ACTS:
        a = A.to(dev).requires_grad_()
        H = tb.gated_gemm(a, torch.eye(2, device=dev), act)
        y, slope = og.gate(act, x.double().clamp(-1e4, 1e4))
        y = og.gate(act, x.double())[0]
        assert torch.allclose(H.detach()[:, 0].double().cpu(), y, rtol=1e-5, atol=1e-30), act
        (dA,) = torch.autograd.grad(H, a, torch.ones_like(H))
        assert torch.allclose(dA[:, 0].double().cpu(), slope, rtol=1e-5, atol=1e-6), act
        nan = tb.gated_gemm(torch.full((1, 2), float("nan"), device=dev), torch.eye(2, device=dev), act)
        assert nan.isnan().all()


def test_second_derivatives_and_tangents(dev):
    from torch.autograd import forward_ad as fwd

    g = torch.Generator().manual_seed(8)
    A, B, tA = (torch.randn(s, generator=g) for s in ((20, 16), (16, 24), (20, 16)))
    f = lambda a, b: tb.gated_gemm(a, b, "gelu_tanh")

    def second(device, dtype):
        a, b = A.to(device, dtype).requires_grad_(), B.to(device, dtype).requires_grad_()
        dA, dB = torch.autograd.grad(f(a, b).square().sum(), (a, b), create_graph=True)
        return torch.autograd.grad(dA.square().sum() + dB.square().sum(), (a, b))

    for got, want in zip(second(dev, F32), second("cpu", torch.float64)):
        assert torch.allclose(got.double().cpu(), want, rtol=1e-4, atol=1e-4 * float(want.abs().max()))
    with fwd.dual_level():
        got = fwd.unpack_dual(f(fwd.make_dual(A.to(dev), tA.to(dev)), B.to(dev))).tangent
        want = fwd.unpack_dual(f(fwd.make_dual(A.double(), tA.double()), B.double())).tangent
    assert torch.allclose(got.double().cpu(), want, rtol=1e-5, atol=1e-5 * float(want.abs().max()))


def test_negated_views(dev):
    g = torch.Generator().manual_seed(9)
    z = lambda *s: torch.randn(*s, 2, generator=g)
    conj = lambda x: torch.view_as_complex(x.to(dev)).conj().imag
    for K, N in ((64, 40), (33, 7)):
        a, b = z(50, K), z(2, K, 2 * N)
        off = torch.tensor([0, 20, 50])
        A, B = conj(a), conj(b)
        assert A.is_neg() and B.is_neg()
        H = tb.grouped_gated_gemm(A, B, off.to(dev))
        assert _holds(H, -a[..., 1], -b[..., 1], off, False, "silu")
        x = (-a[..., 1]).to(dev).requires_grad_()
        dH = z(50, N)
        (dA,) = torch.autograd.grad(tb.grouped_gated_gemm(x, B, off.to(dev)), x, conj(dH))
        (want,) = torch.autograd.grad(tb.grouped_gated_gemm(x, -b[..., 1].to(dev), off.to(dev)), x, -dH[..., 1].to(dev))
        assert torch.allclose(dA, want, rtol=1e-5, atol=1e-5)


def test_sizes_of_zero(dev):
    off = torch.tensor([0, 0, 0], device=dev)
    z = lambda *s: torch.zeros(*s, device=dev)
    assert tb.grouped_gated_gemm(z(0, 4), z(2, 4, 6), off).shape == (0, 3)
    H = tb.grouped_gated_gemm(torch.ones(5, 0, device=dev), z(2, 0, 6), torch.tensor([0, 2, 5], device=dev))
    assert H.shape == (5, 3) and not H.any()
    H = tb.grouped_gated_gemm(torch.ones(3, 4, device=dev), z(0, 4, 6), torch.tensor([0], device=dev))
    assert H.shape == (3, 3) and not H.any()
    assert tb.gated_gemm(z(3, 4), z(4, 0)).shape == (3, 0) and tb.gated_gemm(z(0, 4), z(4, 2)).shape == (0, 1)
    a, b = z(0, 4).requires_grad_(), z(4, 2).requires_grad_()
    dA, dB = torch.autograd.grad(tb.gated_gemm(a, b), (a, b), z(0, 1))
    assert dA.shape == (0, 4) and dB.shape == (4, 2) and not dB.any()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_captured_graph_serves_any_routing(dev, dtype):
    A, B = _operands(9, dtype, 96, 136, 72, 6, True)
    A, B, W = A.to(dev), B.to(dev), B[0].to(dev)
    off = _split(96, [16] * 6).to(dev)
    calls = lambda: (tb.grouped_gated_gemm(A, B, off, transB=True), tb.gated_gemm(A, W, "gelu", transB=True), tb.gated_gemm(A[:3], W, transB=True))
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


def test_captured_training_step(dev):
    # forward and backward in one graph, replayed on other values
    A, B = _operands(10, BF16, 64, 136, 72, 2, False)
    a, b, off = A.to(dev).requires_grad_(), B.to(dev).requires_grad_(), torch.tensor([0, 30, 64], device=dev)
    dH = torch.randn(64, 72, generator=torch.Generator().manual_seed(2)).to(dev, BF16)

    def step():
        H = tb.grouped_gated_gemm(a, b, off)
        return (H.detach(), *torch.autograd.grad(H, (a, b), dH))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        with torch.no_grad():
            a.mul_(1.0 + i)
        off.copy_(torch.tensor([i, 20 + 10 * i, 64 - i]))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, step()))


def test_two_streams_at_once(dev):
    A, B = _operands(11, BF16, 700, 264, 136, 3, True, dev)
    off = _uneven(3, 700, 0).to(dev)
    want = tb.grouped_gated_gemm(A, B, off, transB=True)
    streams = [torch.cuda.Stream() for _ in range(2)]
    out = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            out += [tb.grouped_gated_gemm(A, B, off, transB=True) for _ in range(5)]
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(x, want) for x in out)


def test_training_block_against_64_bits(dev):
    # the whole feed-forward block as a training step runs it: gated projections, then the product back to the model's width
    g = torch.Generator().manual_seed(4)
    x, W, V = (torch.randn(s, generator=g) * f for s, f in (((40, 64), 1.0), ((64, 96), 0.125), ((1, 48, 64), 0.15)))

    def run(gated, product, *args):
        args = [t.detach().clone().requires_grad_() for t in args]
        y = product(gated(args[0], args[1]), args[2])
        return [y.detach(), *torch.autograd.grad(y.square().sum(), args)]

    off = torch.tensor([0, 40], device=dev)
    got = run(lambda a, b: tb.gated_gemm(a, b), lambda h, v: tb.grouped_gemm(1.0, h, v, off), *(t.to(dev) for t in (x, W, V)))

    def plain(a, b):
        G, U = (a @ b).chunk(2, -1)
        return G / (1 + torch.exp(-G)) * U

    want = run(plain, lambda h, v: h @ v[0], *(t.double() for t in (x, W, V)))
    for a, b in zip(got, want):
        assert torch.allclose(a.double().cpu(), b, rtol=1e-4, atol=1e-5 * float(b.abs().max()))
