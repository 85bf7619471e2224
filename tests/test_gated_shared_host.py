"""Gradients of gated projections whose operands depend on each other, against the same formulas in plain operations: a path
through the other operand counts once, with and without create_graph."""

import pytest
import torch

import trnblas_amd as tb

_SILU = torch.nn.functional.silu


def _plain(a, b):
    G, U = (a @ b).chunk(2, -1)
    return _SILU(G) * U


def _plain_grouped(a, E, sizes):
    return torch.cat([_plain(x, E[g]) for g, x in enumerate(a.split(sizes))])


def _random(*shape, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)


SIZES = [3, 0, 4]
OFF = torch.tensor([0, 3, 3, 7])
X, E, W = _random(7, 6, seed=0), _random(3, 6, 12, seed=1), _random(6, 8, seed=2)
# name: (leaves, the framework's result, plain operations')
CASES = {
    "two layers that share weights": (
        (X, E),
        lambda x, e: tb.grouped_gated_gemm(tb.grouped_gated_gemm(x, e, OFF), e, OFF),
        lambda x, e: _plain_grouped(_plain_grouped(x, e, SIZES), e, SIZES),
    ),
    "two layers that share transposed weights": (
        (X, E),
        lambda x, e: tb.grouped_gated_gemm(tb.grouped_gated_gemm(x, e.mT, OFF, transB=True), e.mT, OFF, transB=True),
        lambda x, e: _plain_grouped(_plain_grouped(x, e, SIZES), e, SIZES),
    ),
    "weights computed from the rows": (
        (X, W),
        lambda x, w: tb.gated_gemm(x, x.mT @ x @ w),
        lambda x, w: _plain(x, x.mT @ x @ w),
    ),
    "rows computed from the weights": (
        (X, W),
        lambda x, w: tb.gated_gemm(x @ w @ w.mT, w),
        lambda x, w: _plain(x @ w @ w.mT, w),
    ),
    "one tensor twice": (
        (X[:6],),
        lambda x: tb.gated_gemm(x, x),
        lambda x: _plain(x, x),
    ),
    "one tensor twice, transposed": (
        (X[:6],),
        lambda x: tb.gated_gemm(x, x, transB=True),
        lambda x: _plain(x, x.mT),
    ),
}


@pytest.mark.parametrize("create_graph", [False, True])
@pytest.mark.parametrize("name", list(CASES))
def test_gradients(name, create_graph):
    leaves, own, plain = CASES[name]
    leaves = [t.clone().requires_grad_() for t in leaves]
    grads = [torch.autograd.grad(f(*leaves).square().sum(), leaves, create_graph=create_graph) for f in (own, plain)]
    for got, want in zip(*grads):
        # 64 bits, some hundred operations
        assert torch.allclose(got, want, rtol=1e-11, atol=1e-11 * float(want.detach().abs().max()))


@pytest.mark.parametrize("name", list(CASES))
def test_second_derivatives(name):
    leaves, own, plain = CASES[name]
    leaves = [t.clone().requires_grad_() for t in leaves]

    def second(f):
        first = torch.autograd.grad(f(*leaves).square().sum(), leaves, create_graph=True)
        return torch.autograd.grad(sum(g.square().sum() for g in first), leaves)

    for got, want in zip(second(own), second(plain)):
        assert torch.allclose(got, want, rtol=1e-10, atol=1e-10 * float(want.abs().max()))


def test_gradient_penalty_of_one_operand():
    # the other is a constant, or depends on the one that counts
    x, w = X.clone().requires_grad_(), W.clone().requires_grad_()
    for own, plain in ((tb.gated_gemm(x, w.detach()), _plain(x, w.detach())), (tb.gated_gemm(x.detach(), w), _plain(x.detach(), w))):
        of = [t for t in (x, w) if torch.autograd.grad(plain.sum(), t, retain_graph=True, allow_unused=True)[0] is not None]
        got, want = (torch.autograd.grad(torch.autograd.grad(h.square().sum(), of, create_graph=True)[0].square().sum(), of) for h in (own, plain))
        assert torch.allclose(got[0], want[0], rtol=1e-10, atol=1e-10)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "relu", "sigmoid"])
def test_tangent_of_the_result_s_gradient(act):
    # without create_graph: the gradients are linear in it, and so are their tangents
    from torch.autograd import forward_ad as fwd

    dH, t = _random(7, 6, seed=3), _random(7, 6, seed=4)
    x, e = X.clone().requires_grad_(), E.clone().requires_grad_()
    for a, b in ((x, e), (x, E), (X, e)):
        of = [leaf for leaf in (a, b) if leaf.requires_grad]
        h = tb.grouped_gated_gemm(a, b, OFF, act)
        want = torch.autograd.grad(h, of, dH, retain_graph=True), torch.autograd.grad(h, of, t, retain_graph=True)
        with fwd.dual_level():
            got = [fwd.unpack_dual(g) for g in torch.autograd.grad(h, of, fwd.make_dual(dH, t))]
        for g, value, tangent in zip(got, *want):
            assert torch.equal(g.primal, value) and torch.equal(g.tangent, tangent)
