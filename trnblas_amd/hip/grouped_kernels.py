"""Tensor-level wrappers of the grouped and the microscaled 4-bit products' C ABI, in the manner of
`kernels.py`: device tensors in, a fresh output on their device, launched on
torch's current stream. The group offsets stay on the device: no call waits
for the GPU.
"""

from __future__ import annotations

import torch

from . import _lib
from ._lib import ptr, stream_of
from .kernels import _batched_layout, _probed_call, _require_device


def row_major(X: torch.Tensor) -> tuple[torch.Tensor, int]:
    """(tensor, ld) of a 2-D view whose rows are contiguous, else of a copy."""
    r, c = X.shape
    if (X.stride(1) == 1 or c <= 1) and (X.stride(0) >= c or r <= 1):
        return X, max(X.stride(0), c, 1)
    X = X.contiguous()
    return X, max(c, 1)


def offsets_of(offsets: torch.Tensor) -> tuple[torch.Tensor, int]:
    return offsets.contiguous(), int(offsets.dtype == torch.int64)


def _output_like(C: torch.Tensor | None, beta: float, shape, dtype, dev):
    """(D, c) for an output of `shape`: c is None when beta or C leave it out."""
    D = torch.empty(shape, dtype=dtype, device=dev)
    if beta == 0.0 or C is None:
        return D, None
    c = C.expand(shape)
    n = shape[-1]
    return D, c if (c.stride(-1) == 1 or n <= 1) and (c.stride(-2) >= n or shape[-2] <= 1) else c.contiguous()


def grouped_gemm(
    A: torch.Tensor,
    B: torch.Tensor,
    offsets: torch.Tensor,
    alpha: float = 1.0,
    beta: float = 0.0,
    C: torch.Tensor | None = None,
    out_dtype: torch.dtype | None = None,
) -> torch.Tensor:
    """alpha * A[r] @ B[g] + beta * C[r] for the rows r of each group g: A
    (R, K), B (G, K, N) (transposed views are read in place), offsets (G + 1)."""
    dev = _require_device(A, B, offsets, *(() if C is None else (C,)))
    R, K = A.shape
    G, _, N = B.shape
    a, lda = row_major(A)
    b, tb, ldb, sb = _batched_layout(B)
    o, o64 = offsets_of(offsets)
    D, c = _output_like(C, beta, (R, N), out_dtype or A.dtype, dev)
    _probed_call(
        "grouped_gemm", "trnblas_hip_grouped_gemm", _lib.DTYPE_CODES[A.dtype], int(D.dtype == torch.float32), int(tb),
        G, R, N, K, float(alpha), ptr(a), lda, ptr(b), ldb, sb, ptr(o), o64, float(beta) if c is not None else 0.0,
        ptr(c), max(c.stride(0), N) if c is not None else N, ptr(D), max(N, 1), stream_of(dev),
    )  # fmt: skip
    return D


def grouped_rank_k(
    A: torch.Tensor,
    B: torch.Tensor,
    offsets: torch.Tensor,
    alpha: float = 1.0,
    beta: float = 0.0,
    C: torch.Tensor | None = None,
    out_dtype: torch.dtype | None = None,
) -> torch.Tensor:
    """alpha * A_g^T @ B_g + beta * C[g] for each group g of the rows of A
    (R, M) and B (R, N): (G, M, N)."""
    dev = _require_device(A, B, offsets, *(() if C is None else (C,)))
    R, M = A.shape
    N = B.shape[1]
    G = offsets.shape[0] - 1
    a, lda = row_major(A)
    b, ldb = row_major(B)
    o, o64 = offsets_of(offsets)
    D, c = _output_like(C, beta, (G, M, N), out_dtype or A.dtype, dev)
    _probed_call(
        "grouped_rank_k", "trnblas_hip_grouped_rank_k", _lib.DTYPE_CODES[A.dtype], int(D.dtype == torch.float32),
        G, R, M, N, float(alpha), ptr(a), lda, ptr(b), ldb, ptr(o), o64, float(beta) if c is not None else 0.0,
        ptr(c), max(c.stride(1), N) if c is not None else N, c.stride(0) if c is not None and G > 1 else 0,
        ptr(D), max(N, 1), M * N, stream_of(dev),
    )  # fmt: skip
    return D


def mx_buffers(shape, dev) -> tuple[torch.Tensor, torch.Tensor]:
    """Fresh (codes, scales) buffers of a matrix (..., R, K); see
    include/trnblas_hip.h for their layout."""
    *lead, R, K = shape
    codes = torch.empty((*lead, R, -(-K // 32) * 16), dtype=torch.uint8, device=dev)
    return codes, torch.empty((*lead, -(-R // 16), -(-K // 512), 256), dtype=torch.uint8, device=dev)


def mx_quantize(X: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of X (R, K) or (batch, R, K), any strides."""
    dev = _require_device(X)
    codes, scales = mx_buffers(X.shape, dev)
    if any(s < 0 for s in X.stride()):
        X = X.contiguous()
    batch, sx = (X.shape[0], X.stride(0)) if X.dim() == 3 else (1, 0)
    R, K = X.shape[-2:]
    _probed_call(
        "mx_quantize", "trnblas_hip_mx_quantize", _lib.DTYPE_CODES[X.dtype], R, K, ptr(X), X.stride(-2), X.stride(-1),
        sx, ptr(codes), ptr(scales), batch, stream_of(dev),
    )  # fmt: skip
    return codes, scales


def mx_dequantize(codes: torch.Tensor, scales: torch.Tensor, K: int, dtype: torch.dtype) -> torch.Tensor:
    dev = _require_device(codes, scales)
    *lead, R, _ = codes.shape
    D = torch.empty((*lead, R, K), dtype=dtype, device=dev)
    _probed_call(
        "mx_dequantize", "trnblas_hip_mx_dequantize", _lib.DTYPE_CODES[dtype], R, K, ptr(codes), ptr(scales), ptr(D),
        max(K, 1), R * K, lead[0] if lead else 1, stream_of(dev),
    )  # fmt: skip
    return D


def mx_gemm(
    a: tuple[torch.Tensor, torch.Tensor],
    b: tuple[torch.Tensor, torch.Tensor],
    K: int,
    out_dtype: torch.dtype,
    offsets: torch.Tensor | None = None,
    alpha: float = 1.0,
    beta: float = 0.0,
    C: torch.Tensor | None = None,
) -> torch.Tensor:
    """alpha * A[r] @ B[g]^T + beta * C[r] of (codes, scales) pairs: A (R, K),
    B (N, K), or (G, N, K) with offsets (G + 1)."""
    dev = _require_device(*a, *b, *(() if C is None else (C,)), *(() if offsets is None else (offsets,)))
    R, N = a[0].shape[0], b[0].shape[-2]
    o, o64 = (None, 0) if offsets is None else offsets_of(offsets)
    D, c = _output_like(C, beta, (R, N), out_dtype, dev)
    _probed_call(
        "mx_gemm", "trnblas_hip_mx_gemm", _lib.DTYPE_CODES[out_dtype], 1 if offsets is None else b[0].shape[0], R, N, K,
        float(alpha), ptr(a[0]), ptr(a[1]), ptr(b[0]), ptr(b[1]), ptr(o), o64, float(beta) if c is not None else 0.0,
        ptr(c), max(c.stride(0), N) if c is not None else N, ptr(D), max(N, 1), stream_of(dev),
    )  # fmt: skip
    return D
