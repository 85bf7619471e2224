"""Tensor-level wrappers of the 4-bit integer weights' C ABI, in the manner of
`grouped_kernels.py`. `q` stands for an Int4Matrix's (codes, scales, zeros) and `group`.
"""

from __future__ import annotations

import functools

import torch

from . import _lib
from ._lib import ptr, stream_of
from . import grouped_kernels as _grouped
from . import kernels as _kernels
from .gated_kernels import ACTS
from .grouped_kernels import _checked, _fn, _output_like, offsets_of
from .kernels import _probed_call, _require_device


def buffers(shape, group: int, scale_dtype: torch.dtype, zeros: bool, dev):
    """Fresh (codes, scales, zeros) of matrices (..., R, K); see include/trnblas_hip.h for their layout."""
    *lead, R, K = shape
    blocks, chunks = -(-R // 16), -(-K // 128)
    codes = torch.empty((*lead, blocks, chunks, 1024), dtype=torch.uint8, device=dev)
    of_groups = (*lead, blocks, chunks, 16, 128 // group)
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


FAR = 1 << 22  # elements between rows that are read in place (int4.hip)


@functools.lru_cache(maxsize=4096)
def _partial_bytes(dev: int, code: int, gated: int, groups: int, R: int, N: int, K: int, group: int) -> int:
    """Bytes of the parts' sums: trnblas_hip_int4_gemm_workspace without the rows'. dev: the current device, by whose compute
    units the plan goes."""
    total = _fn("trnblas_hip_int4_gemm_workspace")(code, gated, groups, R, N, K, group)
    return total - _rows_bytes(code, R, K) if total else 0


def _rows_bytes(code: int, R: int, K: int) -> int:
    return R * (-(-K // 128) * 128) * 2 * (3 if code == 0 else 1)


def _in_place(A: torch.Tensor) -> bool:
    """Whether the kernels read these rows as they are."""
    R, K = A.shape
    return (
        A.element_size() == 2 and A.stride(1) == 1 and K % 8 == 0 and A.data_ptr() % 16 == 0
        and (R <= 1 or (A.stride(0) % 8 == 0 and A.stride(0) <= FAR))
    )  # fmt: skip


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
    code, G, gated = _lib.DTYPE_CODES[A.dtype], 1 if offsets is None else codes.shape[0], int(act is not None)
    with torch.cuda.device(dev):
        n = _partial_bytes(dev.index, code, gated, G, R, N, K, group)
    ws = torch.empty(n + (0 if _in_place(A) else _rows_bytes(code, R, K)), dtype=torch.uint8, device=dev)
    _probed_call(
        "int4_gemm", "trnblas_hip_int4_gemm", code, _lib.DTYPE_CODES[out_dtype], gated, ACTS.get(act, 0), G, R, N, K, group, float(alpha), ptr(A), A.stride(0),
        A.stride(1), ptr(codes), ptr(scales), ptr(zeros), _lib.DTYPE_CODES[scales.dtype], ptr(o), o64,
        float(beta) if c is not None else 0.0, ptr(c), max(c.stride(0), N) if c is not None else N, ptr(D), max(N, 1), ptr(ws),
        ws.numel(), stream_of(dev),
    )  # fmt: skip
    return D


# The common calls without the general path's checks, one by one, as in `grouped_kernels.py` (a general call takes 14 us on
# the host, these 9): None where anything is out of the ordinary.


def int4_gemm_fast(alpha, A, B, offsets, out_dtype, act=None):
    """B: the Int4Matrix. Serves rows that the kernels read in place."""
    code = _lib.DTYPE_CODES.get(A.dtype)
    out = code if out_dtype is None else _lib.DTYPE_CODES.get(out_dtype)
    if not code or out is None or _kernels._launch_probe is not None or A.dim() != 2:
        return None
    codes, scales, zeros = B.codes, B.scales, B.zeros
    R, K = A.shape
    sr, sk = A.stride()
    dev = A.get_device()
    N = B.shape[-2]
    gated = 0
    if act is not None:
        gated, act = 1, ACTS.get(act)
        if act is None or N % 2:
            return None
        N //= 2
    pa = A.data_ptr()
    if (
        K != B.shape[-1] or sk != 1 or sr < K or (K | sr) % 8 or sr > FAR or pa % 16 or N == 0 or dev != _grouped._current_device()
        or codes.get_device() != dev or A.is_neg()
    ):  # fmt: skip
        return None
    G, o, o64 = 1, None, False
    if offsets is not None:
        G = codes.shape[0]
        if (
            offsets.get_device() != dev or offsets.dtype not in _grouped._INTS or offsets.shape != (G + 1,)
            or offsets.stride() != (1,)
        ):  # fmt: skip
            return None
        o, o64 = offsets.data_ptr(), offsets.dtype is torch.int64
    D = A.new_empty((R, N), dtype=out_dtype)
    n = _partial_bytes(dev, code, gated, G, R, N, K, B.group)
    ws = codes.new_empty(n) if n else None
    rc = _fn("trnblas_hip_int4_gemm")(
        code, out, gated, act or 0, G, R, N, K, B.group, alpha, pa, sr, 1, codes.data_ptr(), scales.data_ptr(),
        None if zeros is None else zeros.data_ptr(), _SCALE_CODES[scales.dtype], o, o64, 0.0, None, N, D.data_ptr(), N,
        ws.data_ptr() if n else None, n, _grouped._raw_stream(dev),
    )  # fmt: skip
    _checked("trnblas_hip_int4_gemm", rc)
    return D


_SCALE_CODES = {torch.bfloat16: 1, torch.float16: 2}


def quantize_fast(X, group, zeros, scale_dtype):
    """(codes, scales, zeros) of X (R, K), or None."""
    code = _lib.DTYPE_CODES.get(X.dtype)
    dev = X.get_device()
    if code is None or dev != _grouped._current_device() or X.dim() != 2 or _kernels._launch_probe is not None or X.is_neg():
        return None
    R, K = X.shape
    sr, sk = X.stride()
    if sr < 0 or sk < 0:
        return None
    blocks, chunks = -(-R // 16), -(-K // 128)
    codes = X.new_empty((blocks, chunks, 1024), dtype=torch.uint8)
    of_groups = (blocks, chunks, 16, 128 // group)
    scales = X.new_empty(of_groups, dtype=scale_dtype)
    z = X.new_empty(of_groups, dtype=torch.uint8) if zeros else None
    rc = _fn("trnblas_hip_int4_quantize")(
        code, _SCALE_CODES[scale_dtype], R, K, group, X.data_ptr(), sr, sk, 0, codes.data_ptr(), scales.data_ptr(),
        None if z is None else z.data_ptr(), 1, _grouped._raw_stream(dev),
    )  # fmt: skip
    _checked("trnblas_hip_int4_quantize", rc)
    return codes, scales, z


def dequantize_fast(q, shape, group, dtype):
    """The values of one matrix, or None."""
    codes, scales, zeros = q
    dev = codes.get_device()
    if dev != _grouped._current_device() or len(shape) != 2 or _kernels._launch_probe is not None:
        return None
    R, K = shape
    D = codes.new_empty((R, K), dtype=dtype)
    rc = _fn("trnblas_hip_int4_dequantize")(
        _lib.DTYPE_CODES[dtype], _SCALE_CODES[scales.dtype], R, K, group, codes.data_ptr(), scales.data_ptr(),
        None if zeros is None else zeros.data_ptr(), D.data_ptr(), K or 1, R * K, 1, _grouped._raw_stream(dev),
    )  # fmt: skip
    _checked("trnblas_hip_int4_dequantize", rc)
    return D
