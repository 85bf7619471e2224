"""Tensor-level wrappers of the gated projections' C ABI, in the manner of
`grouped_kernels.py`.
"""

from __future__ import annotations

import torch

from . import _lib
from ._lib import ptr, stream_of
from .grouped_kernels import _ready, _up, grouped_gemm, offsets_of, row_major
from .kernels import _batched_layout, _pack_k, _probed_call, _require_device

ACTS = {"silu": 0, "gelu": 1, "gelu_tanh": 2, "relu": 3, "sigmoid": 4}  # TRNBLAS_ACT_*


def gate(P: torch.Tensor, act: str, out_dtype: torch.dtype, save: bool):
    """(H, S): act(P[:, :N]) * P[:, N:] in out_dtype, and where `save` says so P in that type."""
    R, N = P.shape[0], P.shape[1] // 2
    H = torch.empty((R, N), dtype=out_dtype, device=P.device)
    S = torch.empty((R, 2 * N), dtype=out_dtype, device=P.device) if save and out_dtype != P.dtype else None
    _probed_call(
        "gate", "trnblas_hip_gate", ACTS[act], _lib.DTYPE_CODES[P.dtype], _lib.DTYPE_CODES[out_dtype], R, N, ptr(P),
        max(2 * N, 1), ptr(H), max(N, 1), ptr(S), max(2 * N, 1), stream_of(P.device),
    )  # fmt: skip
    return H, (P if S is None else S) if save else None


def gate_backward(P: torch.Tensor, dH: torch.Tensor, act: str) -> torch.Tensor:
    """dP of H = act(P[:, :N]) * P[:, N:] for the gradient dH of H (P's type)."""
    R, N = dH.shape
    dH, ldg = row_major(dH.resolve_neg())
    D = torch.empty_like(P)
    _probed_call(
        "gate_backward", "trnblas_hip_gate_backward", ACTS[act], _lib.DTYPE_CODES[P.dtype], R, N, ptr(P), max(2 * N, 1),
        ptr(dH), max(ldg, N), ptr(D), max(2 * N, 1), stream_of(P.device),
    )  # fmt: skip
    return D


# An fp32 result of 16-bit operands goes through the fp32 product, as it stands, and a launch of the gate.
# Operands that the fused kernels cannot read in place are copied first, rows padded with zeros, from so many
# multiply-adds on; below it the product goes to fp32 by `grouped_gemm`'s kernels, and the gate is a launch of its own.
_PACK_MACS = 1 << 30


def gated_gemm(A: torch.Tensor, B: torch.Tensor, offsets, act: str, out_dtype: torch.dtype, save: bool):
    """(H, P) for A (R, K) and B (G, K, 2 N): H = act(G) * U of P = [G | U] = A[r] @ B[g]; P (in
    out_dtype) only where `save` says so, else None. Rows of no group are zeros."""
    A, B = A.resolve_neg(), B.resolve_neg()
    dev = _require_device(A, B, offsets)
    R, K = A.shape
    G, N = B.shape[0], B.shape[2] // 2
    es = A.element_size()
    ev, padded = 16 // es, False
    a, lda = row_major(A)
    b, tb, ldb, sb = _batched_layout(B)
    su = N * ldb if tb else N
    a_ok = _ready(a.data_ptr(), lda, 0, K, ev)
    b_ok = _ready(b.data_ptr(), ldb, sb, K if tb else N, ev) and su % ev == 0
    if out_dtype != A.dtype or (not (a_ok and b_ok) and 2 * R * K * N < _PACK_MACS):
        return gate(grouped_gemm(A, B, offsets, out_dtype=torch.float32), act, out_dtype, save)
    if not a_ok:
        a, lda, padded = _pack_k(A, _up(K, ev)), _up(K, ev), True
    if not b_ok:
        if tb:
            b = _pack_k(B.mT, _up(K, ev))
            ldb, sb, su = b.stride(1), b.stride(0), N * b.stride(1)
        else:  # gate and up columns of a row one after the other, each padded
            b = _pack_k(B.reshape(G, 2 * K, N), _up(N, ev))
            ldb, sb, su = 2 * b.stride(1), b.stride(0), b.stride(1)
        padded = True
    o, o64 = offsets_of(offsets)
    H = torch.empty((R, N), dtype=out_dtype, device=dev)
    P = torch.empty((R, 2 * N), dtype=out_dtype, device=dev) if save else None
    _probed_call(
        "gated_gemm", "trnblas_hip_gated_gemm", ACTS[act], _lib.DTYPE_CODES[A.dtype], int(tb), G, R, N, K, ptr(a), lda, ptr(b), ldb, sb, su, ptr(o), o64, ptr(H), max(N, 1), ptr(P), max(2 * N, 1),
        int(padded), stream_of(dev),
    )  # fmt: skip
    return H, P
