"""Gated projections, the first half of a feed-forward block: `gated_gemm`, `grouped_gated_gemm`.

    H = act(A G) * (A U)       op(B) = [G | U], 2 N columns

Both projections are one product; the activation and the product of the two halves are
taken from its fp32 sums, and H is rounded once. No counterpart in the reference;
operands as in `gemm` and `grouped_gemm`. Activations: "silu", "gelu" (by erf),
"gelu_tanh", "relu" and "sigmoid".

    H = gated_gemm(x, W, "silu", transB=True)           # x (R, K), W (2 N, K): gate rows, then up rows
    H = grouped_gated_gemm(x, E, offsets)               # rows sorted by expert, E (G, K, 2 N)
    H = gated_gemm(x, int4_quantize(W))                 # served from 4-bit weights

Differentiable: where a gradient is asked for, the forward pass keeps P = [A G | A U], the backward pass forms

    dP = [dH * U * act'(G) | dH * act(G)]     dA = dP op(B)^T     dB = A^T dP

with dP in the result's type (the operand type of its products; an fp32 result's is
fp32, and its products are). P is kept in fp32: in fp16 a gate below -65504 would be infinite and its gradients NaN, and in
bf16 the gradients would be 0.0030 of their norm from the 64-bit ones. 16-bit ones come out 0.0023 (bf16) and 0.00029 (fp16)
from them, by dP's rounding and their own, which alone leaves 0.0017 and 0.00021 (dP as two pieces would double the work of both
products); a dP past 65504 is infinite in fp16. Where that matters, `dtype=torch.float32` has dP in fp32. Second derivatives and
forward-mode tangents go through a product in fp32 and elementary operations.
"""

from __future__ import annotations

import torch
from torch.autograd import forward_ad as _fwd

from ._flags import trans_flag
from .grouped import _check_offsets, _check_operands, _check_result, _fast_call, _gemm, _GroupedGemm, _narrowed, _rank_k, _widened
from .hip import dispatch as _d
from .int4 import Int4Matrix
from .int4 import _product as _int4_product

__all__ = ["gated_gemm", "grouped_gated_gemm"]


_kernels = None


def _gk():
    global _kernels
    if _kernels is None:
        from .hip import gated_kernels

        _kernels = gated_kernels
    return _kernels


_ACTS = {
    "silu": torch.nn.functional.silu,
    "gelu": torch.nn.functional.gelu,
    "gelu_tanh": lambda x: torch.nn.functional.gelu(x, approximate="tanh"),
    "relu": torch.relu,
    "sigmoid": torch.sigmoid,
}


def _check_activation(what: str, activation) -> str:
    if not isinstance(activation, str) or activation not in _ACTS:
        raise ValueError(f"{what}: activation must be one of {sorted(_ACTS)}, got {activation!r}")
    return activation


def _gate_torch(P, act):
    G, U = P.chunk(2, -1)
    return _ACTS[act](G) * U


def _composed(A, b, offsets, act, out):
    """H by operations that are differentiable any number of times, in either mode."""
    wide = torch.promote_types(A.dtype, torch.float32)
    return _gate_torch(_GroupedGemm.apply(1.0, A, b, offsets, 0.0, None, wide), act).to(out)


def _forward(A, b, offsets, act, out, save):
    """(H, P in fp32 at least where `save` says so)."""
    if _d._grouped_on_hip("gated_gemm", A, b):
        try:
            if save:
                kc = b.stride(2) != 1 and b.stride(1) == 1
                HP = _gk().gated_gemm_fast(A, b.mT if kc else b, offsets, act, kc, out, True)
                if HP is not None:
                    return HP
            return _gk().gated_gemm(A, b, offsets, act, out, save)
        except Exception as exc:  # noqa: BLE001
            _d._kernel_failed(exc)
    wide = torch.promote_types(A.dtype, torch.float32)
    P = _d.grouped_gemm(1.0, A, b, offsets, 0.0, None, wide)
    return _gate_torch(P, act).to(out), P if save else None


def _backward(P, dH, act):
    """dP in dH's type."""
    if _d._grouped_on_hip("gated_gemm", dH, P):
        try:
            return _gk().gate_backward(P, dH, act)
        except Exception as exc:  # noqa: BLE001
            _d._kernel_failed(exc)
    with torch.enable_grad():
        p = P.detach().requires_grad_()
        (dP,) = torch.autograd.grad(_gate_torch(p, act), p, dH.to(p.dtype))
    return dP.to(dH.dtype)


class _GatedGemm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, A, b, offsets, act, out):
        H, P = _forward(A, b, offsets, act, out, True)
        ctx.save_for_backward(A, b, offsets, P)
        ctx.act, ctx.out = act, out
        return H

    @staticmethod
    def backward(ctx, dH):
        if torch.is_grad_enabled():  # a derivative of this one may be asked for
            # by views of their own: where one operand depends on the other, the gradient to it ends at
            # the operand, and what leads on from there is counted by whoever asked
            A, b, offsets, _ = ctx.saved_tensors
            A, b = A.view_as(A), b.view_as(b)
            H = _composed(A, b, offsets, ctx.act, ctx.out)
            wanted = [x for x, need in zip((A, b), ctx.needs_input_grad) if need]
            grads = iter(torch.autograd.grad(H, wanted, dH, create_graph=True))
            return *(next(grads) if need else None for need in ctx.needs_input_grad[:2]), None, None, None
        if _d._has_tangent(dH):  # the gradients are linear in it
            dH, t = _fwd.unpack_dual(dH)
            both = zip(_GatedGemm._gradients(ctx, dH), _GatedGemm._gradients(ctx, t))
            dA, dB = (None if g is None else _fwd.make_dual(g, tangent) for g, tangent in both)
        else:
            dA, dB = _GatedGemm._gradients(ctx, dH)
        return dA, dB, None, None, None

    @staticmethod
    def _gradients(ctx, dH):
        """(dA, dB), None what no gradient is asked for."""
        A, b, offsets, P = ctx.saved_tensors
        dP, dt = _backward(P, dH, ctx.act), A.dtype
        if dP.dtype != dt:
            dP, A, b = _widened(dP, A, b)
        dA = dB = None
        if ctx.needs_input_grad[0]:
            dA = _gemm(1.0, dP, b.mT, offsets, 0.0, None, A.dtype)
        if ctx.needs_input_grad[1]:
            if b.stride(1) == 1 and b.stride(2) > 1:  # op(B) is a transposed view: so is its gradient
                dB = _rank_k(1.0, dP, A, offsets, 0.0, None, A.dtype).mT
            else:
                dB = _rank_k(1.0, A, dP, offsets, 0.0, None, A.dtype)
        if A.dtype != dt:
            dA, dB = _narrowed(dt, dA, dB)
        return dA, dB


def _fast(A, B, offsets, activation, transB, dtype):
    """The short way; None: something is out of the ordinary."""
    if type(activation) is str and type(transB) is bool and _fast_call(A, B, offsets, True) and B.dim() == (2 if offsets is None else 3):
        try:
            return _gk().gated_gemm_fast(A, B, offsets, activation, transB, dtype)
        except _d.HipKernelError as exc:
            _d._kernel_failed(exc)
    return None


def _gated(what, A, b, offsets, activation, dtype):
    """b: op(B) (G, K, 2 N)."""
    act = _check_activation(what, activation)
    if A.shape[1] != b.shape[1]:
        raise ValueError(f"{what}: inner dimensions differ: A {tuple(A.shape)}, op(B) {tuple(b.shape)}")
    if b.shape[2] % 2:
        raise ValueError(f"{what}: op(B) must have the gates' columns and as many again, got {b.shape[2]}")
    out = _check_result(what, (A.shape[0], b.shape[2] // 2), dtype, 0.0, None, A)
    if _d._has_tangent(A, b):
        return _composed(A, b, offsets, act, out)
    if _d._wants_grad(A, b):
        return _GatedGemm.apply(A, b, offsets, act, out)
    return _forward(A, b, offsets, act, out, False)[0]


def _int4_gated(what, A, B, offsets, activation, transB, dtype, grouped):
    act = _check_activation(what, activation)
    trans_flag(transB, "transB")
    return _int4_product(what, 1.0, A, B, offsets, 0.0, None, dtype, (act, lambda P: _gate_torch(P, act)), grouped)


def gated_gemm(
    A: torch.Tensor,
    B: torch.Tensor | Int4Matrix,
    activation: str = "silu",
    transB: bool = False,
    dtype: torch.dtype | None = None,
) -> torch.Tensor:
    """act(A @ G) * (A @ U) for op(B) = [G | U].

    A (R, K), B (K, 2 N), or (2 N, K) with transB: gate rows first. The result (R, N)
    has the operands' dtype, or `dtype` float32. B may be an Int4Matrix (2 N, K) (`transB` then says nothing
    new): rows of any float type, results in any, no gradient.
    """
    if isinstance(B, Int4Matrix):
        return _int4_gated("gated_gemm", A, B, None, activation, transB, dtype, False)
    H = _fast(A, B, None, activation, transB, dtype)
    if H is not None:
        return H
    _check_operands("gated_gemm", A, B, (2, 2))
    b = B.mT if trans_flag(transB, "transB") else B
    return _gated("gated_gemm", A, b[None], None, activation, dtype)


def grouped_gated_gemm(
    A: torch.Tensor,
    B: torch.Tensor | Int4Matrix,
    offsets: torch.Tensor,
    activation: str = "silu",
    transB: bool = False,
    dtype: torch.dtype | None = None,
) -> torch.Tensor:
    """H[r] = act(A[r] @ G[g]) * (A[r] @ U[g]) for the rows r of group g, op(B[g]) = [G[g] | U[g]]:
    `grouped_gemm` with `gated_gemm`'s products, B (groups, K, 2 N), or (groups, 2 N, K) with transB.
    Rows of no group come out as zeros. B may be an Int4Matrix (groups, 2 N, K) as in `gated_gemm`."""
    if isinstance(B, Int4Matrix):
        return _int4_gated("grouped_gated_gemm", A, B, offsets, activation, transB, dtype, True)
    if isinstance(offsets, torch.Tensor):
        H = _fast(A, B, offsets, activation, transB, dtype)
        if H is not None:
            return H
    _check_operands("grouped_gated_gemm", A, B, (2, 3))
    b = B.mT if trans_flag(transB, "transB") else B
    _check_offsets("grouped_gated_gemm", offsets, A, b.shape[0])
    return _gated("grouped_gated_gemm", A, b, offsets, activation, dtype)
