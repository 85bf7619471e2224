"""Tensor-level wrappers of the gated projections' C ABI, in the manner of
`grouped_kernels.py`.
"""

from __future__ import annotations

import torch

from . import _lib
from ._lib import ptr, stream_of
from .grouped_kernels import grouped_gemm, row_major
from .kernels import _probed_call

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


def gated_gemm(A: torch.Tensor, B: torch.Tensor, offsets, act: str, out_dtype: torch.dtype, save: bool):
    """(H, P) for A (R, K) and B (G, K, 2 N): H = act(G) * U of P = [G | U] = A[r] @ B[g]; P (in
    out_dtype) only where `save` says so, else None. Rows of no group are zeros."""
    return gate(grouped_gemm(A, B, offsets, out_dtype=torch.float32), act, out_dtype, save)
