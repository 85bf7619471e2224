"""Products over ragged groups of rows: `grouped_gemm` and `grouped_rank_k`.

Rows sorted by expert, each expert with its own matrix, as many rows per
expert as a router gave it. No counterpart in the reference; signatures and
result semantics follow `gemm` (a fresh result, C never written, alpha / beta
fused). Both are differentiable, and each other's gradients:

    D = grouped_gemm(A, B)     dA = grouped_gemm(dD, B^T)   dB = grouped_rank_k(A, dD)
    D = grouped_rank_k(A, B)   dA = grouped_gemm(B, dD^T)   dB = grouped_gemm(A, dD)

The gradient of an fp32 result of 16-bit operands meets them in fp32 (those
products run at the fp32 rate) and is rounded to their type once, at the end. In
forward mode, with tangents tA, tB and tC: tD = alpha (tA B + A tB) + beta tC.

`offsets` (int32 or int64, groups + 1 entries, nondecreasing) gives group g the
rows offsets[g] .. offsets[g + 1] - 1; groups may be empty, and rows before
the first or after the last group belong to none. On a ROCm GPU the offsets are
read by the kernel: no call waits for them, so a captured graph serves any
routing. Entries outside [0, R] are clamped; decreasing ones give unspecified
rows (never an access outside the operands).
"""

from __future__ import annotations

import torch
from torch.autograd import forward_ad as _fwd

from ._flags import trans_flag
from .hip import dispatch as _d

__all__ = ["grouped_gemm", "grouped_rank_k"]


_kernels = None


def _gk():
    global _kernels
    if _kernels is None:
        from .hip import grouped_kernels

        _kernels = grouped_kernels
    return _kernels


def _fast_call(A, B, offsets) -> bool:
    """Tensors on the GPU, no gradient, and the kernels serve: the call may take the short way."""
    return (
        type(A) in _PLAIN
        and type(B) in _PLAIN
        and type(offsets) is torch.Tensor
        and A.is_cuda
        and not ((A.requires_grad or B.requires_grad) and torch.is_grad_enabled())
        and _fwd._current_level < 0
        and _d._use_hip()
    )


_PLAIN = (torch.Tensor, torch.nn.Parameter)


def _check_offsets(what: str, offsets, like: torch.Tensor, groups: int | None = None) -> int:
    if not isinstance(offsets, torch.Tensor) or offsets.dim() != 1 or offsets.shape[0] < 1:
        raise ValueError(f"{what}: offsets must be a 1-D tensor of groups + 1 row numbers")
    if offsets.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{what}: offsets must be int32 or int64, got {offsets.dtype}")
    if offsets.device != like.device:
        raise ValueError(f"{what}: offsets on {offsets.device}, operands on {like.device}")
    if groups is not None and offsets.shape[0] != groups + 1:
        raise ValueError(f"{what}: {groups} groups need {groups + 1} offsets, got {offsets.shape[0]}")
    return offsets.shape[0] - 1


def _check_result(what: str, shape, dtype, beta, C, operand: torch.Tensor, types=None) -> torch.dtype:
    """The result's dtype; C's shape, dtype and device checked against it."""
    out = operand.dtype if dtype is None else dtype
    if out not in (types or (operand.dtype, torch.float32)):
        raise TypeError(f"{what}: result dtype {out} for {operand.dtype} operands (theirs or float32)")
    if beta != 0.0:
        if C is None:
            raise ValueError(f"{what}: beta != 0 needs C")
        if C.dtype != out:
            raise TypeError(f"{what}: C is {C.dtype}, the result {out}")
        if C.device != operand.device:
            raise ValueError(f"{what}: C on {C.device}, operands on {operand.device}")
        if C.dim() > len(shape) or any(c not in (1, s) for c, s in zip(C.shape[::-1], shape[::-1])):
            raise ValueError(f"{what}: C {tuple(C.shape)} does not broadcast to {tuple(shape)}")
    return out


def _check_operands(what: str, A, B, dims) -> None:
    for name, X, dim in (("A", A, dims[0]), ("B", B, dims[1])):
        if not isinstance(X, torch.Tensor) or X.dim() != dim:
            raise ValueError(f"{what}: {name} must be a {dim}-D tensor")
        if not X.is_floating_point():
            raise TypeError(f"{what}: {name} must be a real floating tensor, got {X.dtype}")
    if A.dtype != B.dtype:
        raise TypeError(f"{what}: mixed dtypes {A.dtype}, {B.dtype}")
    if A.device != B.device:
        raise ValueError(f"{what}: operands on different devices: {A.device} and {B.device}")


def _gemm(alpha, A, B, offsets, beta, C, out_dtype):
    """The product for the autograd functions, B as in _d.grouped_gemm: the short way where it serves."""
    if beta == 0.0 and A.is_cuda and _d._use_hip():
        kc = B.stride(2) != 1 and B.stride(1) == 1
        try:
            D = _gk().grouped_gemm_fast(alpha, A, B.mT if kc else B, offsets, kc, out_dtype)
            if D is not None:
                return D
        except _d.HipKernelError as exc:
            _d._kernel_failed(exc)
    return _d.grouped_gemm(alpha, A, B, offsets, beta, C, out_dtype)


def _rank_k(alpha, A, B, offsets, beta, C, out_dtype):
    if beta == 0.0 and A.is_cuda and _d._use_hip():
        try:
            D = _gk().grouped_rank_k_fast(alpha, A, B, offsets, out_dtype)
            if D is not None:
                return D
        except _d.HipKernelError as exc:
            _d._kernel_failed(exc)
    return _d.grouped_rank_k(alpha, A, B, offsets, beta, C, out_dtype)


def _differentiable(function, product, *args):
    """A product of a backward pass, itself differentiable only where that is asked for."""
    return function.apply(*args) if torch.is_grad_enabled() or _fwd._current_level >= 0 else product(*args)


def _widened(dD, A, B):
    """The operands of a backward product in one type: an fp32 gradient is not rounded to 16-bit operands' type, whose
    range (fp16: 65504) it may pass."""
    wide = torch.promote_types(dD.dtype, A.dtype)
    return dD.to(wide), A.to(wide), B.to(wide)


def _narrowed(dtype, *grads):
    return (None if g is None else g.to(dtype) for g in grads)


def _tangent(ctx, product, tA, tB, tC):
    """The tangent of a product, summed in fp32 at least and rounded once."""
    A, B, offsets = ctx.saved_for_forward
    wide = torch.promote_types(ctx.out_dtype, torch.float32)
    t = None if tC is None else ctx.beta * tC.to(wide)
    for a, b in ((tA, B), (A, tB)):
        if a is not None and b is not None:
            t = product(ctx.alpha, a, b, offsets, 0.0 if t is None else 1.0, t, wide)
    return t.to(ctx.out_dtype)


def _save(ctx, alpha, A, B, offsets, beta, out_dtype):
    ctx.save_for_backward(A, B, offsets)
    if _fwd._current_level >= 0:
        ctx.save_for_forward(A, B, offsets)
    ctx.alpha, ctx.beta, ctx.out_dtype = alpha, beta, out_dtype


class _GroupedGemm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, alpha, A, B, offsets, beta, C, out_dtype):
        _save(ctx, alpha, A, B, offsets, beta, out_dtype)
        return _gemm(alpha, A, B, offsets, beta, C, out_dtype)

    @staticmethod
    def jvp(ctx, _alpha, tA, tB, _offsets, _beta, tC, _out_dtype):
        return _tangent(ctx, _gemm, tA, tB, tC)

    @staticmethod
    def backward(ctx, dD):
        A, B, offsets = ctx.saved_tensors
        dA = dB = dC = None
        if ctx.needs_input_grad[5]:
            dC = ctx.beta * dD
        dt = A.dtype
        if dD.dtype != dt:
            dD, A, B = _widened(dD, A, B)
        if ctx.needs_input_grad[1]:
            dA = _differentiable(_GroupedGemm, _gemm, ctx.alpha, dD, B.mT, offsets, 0.0, None, A.dtype)
        if ctx.needs_input_grad[2]:
            if B.stride(1) == 1 and B.stride(2) > 1:  # B is a transposed view: so is its gradient
                dB = _differentiable(_GroupedRankK, _rank_k, ctx.alpha, dD, A, offsets, 0.0, None, B.dtype).mT
            else:
                dB = _differentiable(_GroupedRankK, _rank_k, ctx.alpha, A, dD, offsets, 0.0, None, B.dtype)
        if A.dtype != dt:
            dA, dB = _narrowed(dt, dA, dB)
        return None, dA, dB, None, None, dC, None


class _GroupedRankK(torch.autograd.Function):
    @staticmethod
    def forward(ctx, alpha, A, B, offsets, beta, C, out_dtype):
        _save(ctx, alpha, A, B, offsets, beta, out_dtype)
        return _rank_k(alpha, A, B, offsets, beta, C, out_dtype)

    @staticmethod
    def jvp(ctx, _alpha, tA, tB, _offsets, _beta, tC, _out_dtype):
        return _tangent(ctx, _rank_k, tA, tB, tC)

    @staticmethod
    def backward(ctx, dD):
        A, B, offsets = ctx.saved_tensors
        dA = dB = dC = None
        if ctx.needs_input_grad[5]:
            dC = ctx.beta * dD
        dt = A.dtype
        if dD.dtype != dt:
            dD, A, B = _widened(dD, A, B)
        if ctx.needs_input_grad[1]:
            dA = _differentiable(_GroupedGemm, _gemm, ctx.alpha, B, dD.mT, offsets, 0.0, None, A.dtype)
        if ctx.needs_input_grad[2]:
            dB = _differentiable(_GroupedGemm, _gemm, ctx.alpha, A, dD, offsets, 0.0, None, B.dtype)
        if A.dtype != dt:
            dA, dB = _narrowed(dt, dA, dB)
        return None, dA, dB, None, None, dC, None


def grouped_gemm(
    alpha: float,
    A: torch.Tensor,
    B: torch.Tensor,
    offsets: torch.Tensor,
    beta: float = 0.0,
    C: torch.Tensor | None = None,
    transB: bool = False,
    dtype: torch.dtype | None = None,
) -> torch.Tensor:
    """D[r] = alpha * A[r] @ op(B[g]) + beta * C[r] for the rows r of group g.

    A (R, K), B (G, K, N), or (G, N, K) with transB; D (R, N) in the operands'
    dtype, or `dtype` float32 (16-bit operands are summed in fp32 either way).
    Rows of no group come out as beta * C[r]. A C that broadcasts to (R, N) is
    taken as in `gemm`. One launch on the GPU, whatever the group sizes.
    """
    if beta == 0.0 and _fast_call(A, B, offsets) and type(transB) is bool:
        try:
            D = _gk().grouped_gemm_fast(alpha, A, B, offsets, transB, dtype)
            if D is not None:
                return D
        except _d.HipKernelError as exc:
            _d._kernel_failed(exc)
    _check_operands("grouped_gemm", A, B, (2, 3))
    b = B.mT if trans_flag(transB, "transB") else B
    _check_offsets("grouped_gemm", offsets, A, b.shape[0])
    if A.shape[1] != b.shape[1]:
        raise ValueError(f"grouped_gemm: inner dimensions differ: A {tuple(A.shape)}, op(B) {tuple(b.shape)}")
    shape = (A.shape[0], b.shape[2])
    out = _check_result("grouped_gemm", shape, dtype, beta, C, A)
    c = C.expand(shape) if beta != 0.0 else None
    if _d._wants_grad(A, B, *(() if c is None else (c,))):
        return _GroupedGemm.apply(alpha, A, b, offsets, beta, c, out)
    return _d.grouped_gemm(alpha, A, b, offsets, beta, c, out)


def grouped_rank_k(
    alpha: float,
    A: torch.Tensor,
    B: torch.Tensor,
    offsets: torch.Tensor,
    beta: float = 0.0,
    C: torch.Tensor | None = None,
    dtype: torch.dtype | None = None,
) -> torch.Tensor:
    """D[g] = alpha * A_g^T @ B_g + beta * C[g], A_g and B_g the rows of group g.

    A (R, M), B (R, N); D (G, M, N) in the operands' dtype, or `dtype` float32
    (with beta = 1 the gradient of earlier calls is added to in fp32). A group
    without rows gives beta * C[g].
    """
    if beta == 0.0 and _fast_call(A, B, offsets):
        try:
            D = _gk().grouped_rank_k_fast(alpha, A, B, offsets, dtype)
            if D is not None:
                return D
        except _d.HipKernelError as exc:
            _d._kernel_failed(exc)
    _check_operands("grouped_rank_k", A, B, (2, 2))
    groups = _check_offsets("grouped_rank_k", offsets, A)
    if A.shape[0] != B.shape[0]:
        raise ValueError(f"grouped_rank_k: A has {A.shape[0]} rows, B {B.shape[0]}")
    shape = (groups, A.shape[1], B.shape[1])
    out = _check_result("grouped_rank_k", shape, dtype, beta, C, A)
    c = C.expand(shape) if beta != 0.0 else None
    if _d._wants_grad(A, B, *(() if c is None else (c,))):
        return _GroupedRankK.apply(alpha, A, B, offsets, beta, c, out)
    return _d.grouped_rank_k(alpha, A, B, offsets, beta, c, out)
