"""Gated projections and 4-bit weights where offsets pass 32 bits, rows lie far apart, and parts of K are summed in workspaces:
the calls that the ordinary sizes of `test_gated_gpu.py` and `test_int4_gpu.py` do not make. Bounds: theirs."""

import pytest
import torch

import trnblas_amd as tb
from oracle import gated as oa
from oracle import grouped as og
from oracle import int4 as oi
from trnblas_amd.hip import _lib
from trnblas_amd.int4 import Int4Matrix

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _blocks(Q, a, b):
    """Blocks a .. b - 1 of sixteen rows of a matrix."""
    cut = lambda t: None if t is None else t[a:b]
    return Int4Matrix(cut(Q.codes), cut(Q.scales), cut(Q.zeros), (16 * (b - a), Q.shape[1]), Q.group)


def _many_blocks(blocks, K, group, dev):
    """A matrix of random codes, its scales near one; zero points too."""
    g = torch.Generator(device=dev).manual_seed(0)
    codes = torch.empty(blocks, K // 128, 1024, dtype=torch.uint8, device=dev)
    codes.view(torch.int64).random_(generator=g)
    of = (blocks, K // 128, 16, 128 // group)
    scales = (torch.rand(of, generator=g, device=dev) + 0.5).to(F16)
    zeros = torch.randint(0, 16, of, generator=g, device=dev, dtype=torch.uint8)
    return Int4Matrix(codes, scales, zeros, (16 * blocks, K), group)


@pytest.mark.parametrize("rows", [1, 20, 260])
def test_int4_past_32_bits(dev, rows):
    # 4.3 GB of codes; results of 2.2e9 values
    K, blocks = 1024, (1 << 19) + 5
    Q = _many_blocks(blocks, K, 64, dev)
    A = torch.randn(rows, K, generator=torch.Generator().manual_seed(rows)).to(dev, F16) / 64
    D = tb.int4_gemm(1.0, A, Q)
    H = tb.gated_gemm(A, Q, "silu")
    assert D.shape == (rows, 16 * blocks) and H.shape == (rows, 8 * blocks)
    for a in (0, (blocks // 2) - 8, blocks - 16):
        W = _blocks(Q, a, a + 16).dequantize().double()
        ref, den = A.double() @ W.T, A.double().abs() @ W.abs().T
        assert og.excess(D[:, 16 * a : 16 * a + 256].cpu(), ref.cpu(), den.cpu(), K) <= 1, a
    half = 8 * blocks  # an odd number of blocks: ups start inside one
    for n in (0, half - 128):
        a, b = n // 16, (half + n) // 16
        rows_of = lambda first, lo: _blocks(Q, lo, min(blocks, lo + 10)).dequantize().double()[first - 16 * lo :][:128]
        W = torch.cat([rows_of(n, a), rows_of(half + n, b)])[None]
        P, d = oa.products(A, W, torch.tensor([0, rows]), True)
        assert oa.ratio(H[:, n : n + 128], *oa.forward("silu", P, d, K, F16)) <= 1, n
    del D, H


def test_int4_quantize_past_32_bits(dev):
    K, blocks = 1024, (1 << 18) + 3
    X = torch.randn(16 * blocks, K, dtype=BF16, device=dev)
    Q = tb.int4_quantize(X, 32, zeros=True)
    D = tb.int4_dequantize(Q, BF16)
    for a in (0, blocks // 2, blocks - 2):
        x = X[16 * a : 16 * a + 32].clone()
        R = tb.int4_quantize(x, 32, zeros=True)
        S = _blocks(Q, a, a + 2)
        assert torch.equal(S.codes, R.codes) and torch.equal(S.scales, R.scales) and torch.equal(S.zeros, R.zeros)
        assert torch.equal(D[16 * a : 16 * a + 32], tb.int4_dequantize(R, BF16))


@pytest.mark.parametrize("K", [1 << 22, (1 << 22) - 1])
def test_int4_longest_rows(dev, K):
    # read in place, and laid out first
    g = torch.Generator(device=dev).manual_seed(1)
    A = torch.randn(130, K, generator=g, device=dev, dtype=F16)
    Q = tb.int4_quantize(torch.randn(24, K, generator=g, device=dev, dtype=F16), 128)
    W = Q.dequantize().double()
    for R in (1, 64, 130):
        a = A[:R].double()
        ref, den = a @ W.T, a.abs() @ W.abs().T
        assert og.excess(tb.int4_gemm(1.0, A[:R], Q, dtype=F32).cpu(), ref.cpu(), den.cpu(), K) <= 1, R


def test_int4_rows_far_apart(dev):
    # on both sides of the distance up to which rows are read in place
    g = torch.Generator().manual_seed(2)
    Q, W = oi.random_matrix(g, 40, 256, group=64, zeros=True, scale_dtype=BF16)
    Q = Q.to(dev)
    for R in (3, 130):
        for step in (1 << 22, (1 << 22) + 8):
            A = torch.randn(R, 256, generator=g).to(BF16)
            X = torch.empty(R * step, dtype=BF16, device=dev).as_strided((R, 256), (step, 1))
            X.copy_(A)
            assert og.excess(tb.int4_gemm(1.0, X, Q), *oi.product(1.0, A, W), 256) <= 1, (R, step)


def test_gated_past_32_bits(dev):
    # weights past 2^31 values either way round, and the products that a gradient needs; small whole numbers over 16: every order
    # of summation gives the same products
    K, N = 512, (1 << 21) + 8
    B = torch.empty(2 * N, K, dtype=BF16, device=dev).random_(-2, 3, generator=torch.Generator(device=dev).manual_seed(3)).mul_(1 / 16)
    for R in (2, 40, 600):
        A = torch.randint(-1, 2, (R, K), generator=torch.Generator().manual_seed(R)).to(dev, BF16)
        a = A.clone().requires_grad_(R == 600)
        H = tb.gated_gemm(a, B, "gelu", transB=True)
        for n in (0, N // 2, N - 64):
            W = torch.cat([B[n : n + 64], B[N + n : N + n + 64]])
            P, d = oa.products(A, W[None], torch.tensor([0, R]), True)
            assert oa.ratio(H[:, n : n + 64].detach(), *oa.forward("gelu", P, d, K, BF16)) <= 1, (R, n)
        if R == 600:  # the gradient of a few columns alone: the others' products are zeros
            dH = torch.zeros_like(H)
            dH[:, N - 64 :] = 1.0
            (dA,) = torch.autograd.grad(H, a, dH)
            W = torch.cat([B[N - 64 : N], B[2 * N - 64 :]]).contiguous()
            b = A.clone().requires_grad_()
            (want,) = torch.autograd.grad(tb.gated_gemm(b, W, "gelu", transB=True), b, torch.ones(R, 64, dtype=BF16, device=dev))
            # the same terms in another order: sums of 128 terms below 2 (128^2 * 2^-24 * 2 = 2^-9 apart at most), then one rounding each
            assert ((dA.double() - want.double()).abs() <= 2.0**-7 * want.double().abs() + 2.0**-9).all()
        del H
    B = B.view(K, 2 * N)
    A = torch.randn(40, K, generator=torch.Generator().manual_seed(9)).to(dev, BF16)
    H = tb.gated_gemm(A, B, "relu")
    for n in (0, N - 64):
        W = torch.cat([B[:, n : n + 64], B[:, N + n : N + n + 64]], 1)
        P, d = oa.products(A, W[None], torch.tensor([0, 40]), False)
        assert oa.ratio(H[:, n : n + 64], *oa.forward("relu", P, d, K, BF16)) <= 1, n


def _splits(R, N, K):
    import ctypes

    plan = (ctypes.c_int32 * 5)()
    _lib.call("trnblas_hip_int4_plan", _lib.DTYPE_CODES[BF16], 0, 1, R, N, K, 128, plan)
    return plan[1]


def test_parts_of_k_in_two_graphs_and_streams(dev):
    # each call's sums are its own: two graphs replayed in turns and at once, eager calls between
    R, N, K = 200, 4096, 4096
    assert _splits(R, N, K) > 1
    g = torch.Generator().manual_seed(4)
    Q = tb.int4_quantize(torch.randn(N, K, generator=g).to(dev), 128)
    A = [torch.randn(R, K, generator=g).to(dev, BF16) for _ in range(2)]
    graphs, out = [], []
    for a in A:
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            tb.int4_gemm(1.0, a, Q)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out.append(tb.int4_gemm(1.0, a, Q))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in A]
    for i in range(4):
        for a in A:
            a.mul_(1.0 + 0.5 * i)
        for s, graph in zip(streams, graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                graph.replay()
        eager = [tb.int4_gemm(1.0, a, Q) for a in A]
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, eager)), i


def test_gradients_of_broadcast_and_strided_results(dev):
    # a sum's gradient is one value everywhere; a transposed result's comes in columns
    g = torch.Generator().manual_seed(5)
    for dtype in (F32, BF16):
        A, B = torch.randn(33, 40, generator=g).to(dev, dtype), (torch.randn(40, 48, generator=g) / 6).to(dev, dtype)
        for of in (lambda H: H.sum(), lambda H: (H.mT * 1.0).sum(), lambda H: H[:1].sum(), lambda H: H[:, :1].sum()):
            a, b = A.clone().requires_grad_(), B.clone().requires_grad_()
            H = tb.gated_gemm(a, b)
            (dH,) = torch.autograd.grad(of(H), H, retain_graph=True)
            got = torch.autograd.grad(of(H), (a, b))
            want = torch.autograd.grad(tb.gated_gemm(a, b), (a, b), dH.contiguous())
            assert all(torch.equal(x, y) for x, y in zip(got, want))
