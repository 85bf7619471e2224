"""Tensor-level wrappers of the 4-bit integer weights' C ABI, in the manner of
`grouped_kernels.py`. `q` stands for an Int4Matrix's (codes, scales, zeros) and `group`.
"""

from __future__ import annotations

import torch

from . import _lib
from ._lib import ptr, stream_of
from .gated_kernels import ACTS
from .grouped_kernels import _output_like, offsets_of
from .kernels import _probed_call, _require_device


def buffers(shape, group: int, scale_dtype: torch.dtype, zeros: bool, dev):
    """Fresh (codes, scales, zeros) of matrices (..., R, K); see include/trnblas_hip.h for their layout."""
    *lead, R, K = shape
    blocks, chunks = -(-R // 16), -(-K // 128)
    codes = torch.empty((*lead, blocks, chunks, 1024), dtype=torch.uint8, device=dev)
    of_groups = (*lead, blocks, chunks * (128 // group), 16)
    scales = torch.empty(of_groups, dtype=scale_dtype, device=dev)
    return codes, scales, torch.empty(of_groups, dtype=torch.uint8, device=dev) if zeros else None


def quantize(X: torch.Tensor, group: int, zeros: bool, scale_dtype: torch.dtype):
    """(codes, scales, zeros) of X (R, K) or (batch, R, K), any strides."""
    X = X.resolve_neg()
    dev = _require_device(X)
    if any(s < 0 for s in X.stride()):
        X = X.contiguous()
    codes, scales, z = buffers(X.shape, group, scale_dtype, zeros, dev)
    batch, sx = (X.shape[0], X.stride(0)) if X.dim() == 3 else (1, 0)
    R, K = X.shape[-2:]
    _probed_call(
        "int4_quantize", "trnblas_hip_int4_quantize", _lib.DTYPE_CODES[X.dtype], _lib.DTYPE_CODES[scale_dtype], R, K, group,
        ptr(X), X.stride(-2), X.stride(-1), sx, ptr(codes), ptr(scales), ptr(z), batch, stream_of(dev),
    )  # fmt: skip
    return codes, scales, z


def dequantize(q, shape, group: int, dtype: torch.dtype) -> torch.Tensor:
    codes, scales, zeros = q
    *lead, R, K = shape
    D = torch.empty(tuple(shape), dtype=dtype, device=codes.device)
    _probed_call(
        "int4_dequantize", "trnblas_hip_int4_dequantize", _lib.DTYPE_CODES[dtype], _lib.DTYPE_CODES[scales.dtype], R, K, group,
        ptr(codes), ptr(scales), ptr(zeros), ptr(D), max(K, 1), R * K, lead[0] if lead else 1, stream_of(codes.device),
    )  # fmt: skip
    return D


def _workspace(A: torch.Tensor) -> int:
    """trnblas_hip_int4_gemm_workspace (the same formula; a library call costs more), 0 where the rows are read in place."""
    R, K = A.shape
    es = A.element_size()
    if es == 2 and A.stride(1) == 1 and K % 8 == 0 and A.data_ptr() % 16 == 0 and (A.stride(0) % 8 == 0 or R <= 1):
        return 0
    return R * (-(-K // 128) * 128) * 2 * (3 if es == 4 else 1)


def int4_gemm(
    A: torch.Tensor,
    q,
    N: int,
    group: int,
    out_dtype: torch.dtype,
    offsets: torch.Tensor | None = None,
    alpha: float = 1.0,
    beta: float = 0.0,
    C: torch.Tensor | None = None,
    act: str | None = None,
) -> torch.Tensor:
    """alpha * A[r] @ W[g]^T + beta * C[r] for A (R, K) and matrices of N rows; with an activation act(A[r] @ G^T) * (A[r] @ U^T)
    of 2 N rows."""
    codes, scales, zeros = q
    A = A.resolve_neg()
    dev = _require_device(A, codes, scales, zeros, C, offsets)
    if any(s < 0 for s in A.stride()):
        A = A.contiguous()
    R, K = A.shape
    o, o64 = offsets_of(offsets)
    D, c = _output_like(C, beta, (R, N), out_dtype, dev)
    ws = torch.empty(_workspace(A), dtype=torch.uint8, device=dev)
    _probed_call(
        "int4_gemm", "trnblas_hip_int4_gemm", _lib.DTYPE_CODES[A.dtype], _lib.DTYPE_CODES[out_dtype], int(act is not None),
        ACTS.get(act, 0), 1 if offsets is None else codes.shape[0], R, N, K, group, float(alpha), ptr(A), A.stride(0),
        A.stride(1), ptr(codes), ptr(scales), ptr(zeros), _lib.DTYPE_CODES[scales.dtype], ptr(o), o64,
        float(beta) if c is not None else 0.0, ptr(c), max(c.stride(0), N) if c is not None else N, ptr(D), max(N, 1), ptr(ws),
        ws.numel(), stream_of(dev),
    )  # fmt: skip
    return D
