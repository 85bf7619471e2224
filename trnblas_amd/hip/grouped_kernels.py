"""Tensor-level wrappers of the grouped and the microscaled 4-bit products' C ABI, in the manner of
`kernels.py`: device tensors in, a fresh output on their device, launched on
torch's current stream. The group offsets stay on the device: no call waits
for the GPU.
"""

from __future__ import annotations

import torch

from . import _lib
from ._lib import ptr, stream_of
from . import kernels as _kernels
from .kernels import _batched_layout, _pack_k, _probed_call, _require_device


def row_major(X: torch.Tensor) -> tuple[torch.Tensor, int]:
    """(tensor, ld) of a 2-D view whose rows are contiguous, else of a copy."""
    r, c = X.shape
    if (X.stride(1) == 1 or c <= 1) and (X.stride(0) >= c or r <= 1):
        return X, max(X.stride(0), c, 1)
    X = X.contiguous()
    return X, max(c, 1)


def offsets_of(offsets: torch.Tensor | None) -> tuple[torch.Tensor | None, int]:
    """None: all rows are one group."""
    return (None, 0) if offsets is None else (offsets.contiguous(), int(offsets.dtype == torch.int64))


def _output_like(C: torch.Tensor | None, beta: float, shape, dtype, dev):
    """(D, c) for an output of `shape`: c is None when beta or C leave it out."""
    D = torch.empty(shape, dtype=dtype, device=dev)
    if beta == 0.0 or C is None:
        return D, None
    c = C.resolve_neg().expand(shape)
    n = shape[-1]
    return D, c if (c.stride(-1) == 1 or n <= 1) and (c.stride(-2) >= n or shape[-2] <= 1) else c.contiguous()


# Operands that LDS DMA cannot read in place (base, leading dimension or extent no
# multiple of 16 bytes) are copied first, their rows padded with zeros, where the
# copies cost less than grouped_any_kernel's loads: both read and write at about 4 TB/s
# and start in 4 us each; the kernel makes 400 TFLOP/s (rank_k 310; fp32 90) of such operands,
# the ring kernels 800 (fp32 115) of copied ones. bf16 16383 rows in 8 groups, 2047 x
# 4095: 678 us in place, 450 packed; 4093 rows, 1023 x 2047: 61 and 64. Products of few flops per byte stay in place.
_PACK_SAVES = {  # us per multiply-add
    ("gemm", 2): 2 * (1 / 400e6 - 1 / 800e6), ("rank_k", 2): 2 * (1 / 310e6 - 1 / 800e6),
    ("gemm", 4): 2 * (1 / 90e6 - 1 / 115e6), ("rank_k", 4): 2 * (1 / 90e6 - 1 / 115e6),
}  # fmt: skip


def _ready(p: int, ld: int, stride: int, ext: int, ev: int) -> bool:
    return p % 16 == 0 and ld % ev == 0 and stride % ev == 0 and ext % ev == 0


def _pack_pays(op: str, es: int, macs: int, copied: int) -> bool:
    """copied: elements of the operands that are not ready."""
    return macs * _PACK_SAVES[op, es] > 8 + 2 * copied * es / 4e6


def _up(n: int, ev: int) -> int:
    return -(-n // ev) * ev


def grouped_gemm(
    A: torch.Tensor,
    B: torch.Tensor,
    offsets: torch.Tensor | None,
    alpha: float = 1.0,
    beta: float = 0.0,
    C: torch.Tensor | None = None,
    out_dtype: torch.dtype | None = None,
) -> torch.Tensor:
    """alpha * A[r] @ B[g] + beta * C[r] for the rows r of each group g: A
    (R, K), B (G, K, N) (transposed views are read in place), offsets (G + 1), or
    None for one group of all rows."""
    A, B = A.resolve_neg(), B.resolve_neg()
    dev = _require_device(A, B, offsets, *(() if C is None else (C,)))
    R, K = A.shape
    G, _, N = B.shape
    a, lda = row_major(A)
    b, tb, ldb, sb = _batched_layout(B)
    ev, padded = 16 // A.element_size(), False
    a_ok = _ready(a.data_ptr(), lda, 0, K, ev)
    b_ok = _ready(b.data_ptr(), ldb, sb, K if tb else N, ev)
    if not (a_ok and b_ok):
        padded = _pack_pays("gemm", A.element_size(), R * K * N, (not a_ok) * R * K + (not b_ok) * G * K * N)
    if padded and not a_ok:
        a, lda = _pack_k(A, _up(K, ev)), _up(K, ev)
    if padded and not b_ok:
        b = _pack_k(B.mT if tb else B, _up(K if tb else N, ev))
        ldb, sb = b.stride(1), b.stride(0)
    o, o64 = offsets_of(offsets)
    D, c = _output_like(C, beta, (R, N), out_dtype or A.dtype, dev)
    _probed_call(
        "grouped_gemm", "trnblas_hip_grouped_gemm", _lib.DTYPE_CODES[A.dtype], int(D.dtype == torch.float32), int(tb),
        G, R, N, K, float(alpha), ptr(a), lda, ptr(b), ldb, sb, ptr(o), o64, float(beta) if c is not None else 0.0,
        ptr(c), max(c.stride(0), N) if c is not None else N, ptr(D), max(N, 1), int(padded), stream_of(dev),
    )  # fmt: skip
    return D


def grouped_rank_k(
    A: torch.Tensor,
    B: torch.Tensor,
    offsets: torch.Tensor | None,
    alpha: float = 1.0,
    beta: float = 0.0,
    C: torch.Tensor | None = None,
    out_dtype: torch.dtype | None = None,
) -> torch.Tensor:
    """alpha * A_g^T @ B_g + beta * C[g] for each group g of the rows of A
    (R, M) and B (R, N): (G, M, N)."""
    A, B = A.resolve_neg(), B.resolve_neg()
    dev = _require_device(A, B, offsets, *(() if C is None else (C,)))
    R, M = A.shape
    N = B.shape[1]
    G = 1 if offsets is None else offsets.shape[0] - 1
    a, lda = row_major(A)
    b, ldb = row_major(B)
    ev, padded = 16 // A.element_size(), False
    a_ok, b_ok = _ready(a.data_ptr(), lda, 0, M, ev), _ready(b.data_ptr(), ldb, 0, N, ev)
    if not (a_ok and b_ok):
        padded = _pack_pays("rank_k", A.element_size(), R * M * N, (not a_ok) * R * M + (not b_ok) * R * N)
    if padded and not a_ok:
        a, lda = _pack_k(A, _up(M, ev)), _up(M, ev)
    if padded and not b_ok:
        b, ldb = _pack_k(B, _up(N, ev)), _up(N, ev)
    o, o64 = offsets_of(offsets)
    D, c = _output_like(C, beta, (G, M, N), out_dtype or A.dtype, dev)
    _probed_call(
        "grouped_rank_k", "trnblas_hip_grouped_rank_k", _lib.DTYPE_CODES[A.dtype], int(D.dtype == torch.float32),
        G, R, M, N, float(alpha), ptr(a), lda, ptr(b), ldb, ptr(o), o64, float(beta) if c is not None else 0.0,
        ptr(c), max(c.stride(1), N) if c is not None else N, c.stride(0) if c is not None and G > 1 else 0,
        ptr(D), max(N, 1), M * N, int(padded), stream_of(dev),
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
    X = X.resolve_neg()
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
    *lead, R, _ = codes.shape
    D = codes.new_empty((*lead, R, K), dtype=dtype)
    _probed_call(
        "mx_dequantize", "trnblas_hip_mx_dequantize", _lib.DTYPE_CODES[dtype], R, K, ptr(codes), ptr(scales), ptr(D),
        max(K, 1), R * K, lead[0] if lead else 1, stream_of(codes.device),
    )  # fmt: skip
    return D


def mx_gemm_from(
    A: torch.Tensor,
    b: tuple[torch.Tensor, torch.Tensor],
    out_dtype: torch.dtype,
    offsets: torch.Tensor | None = None,
    alpha: float = 1.0,
    beta: float = 0.0,
    C: torch.Tensor | None = None,
) -> torch.Tensor:
    """`mx_gemm` of a float A (R, K), quantised on the way (in the same call)."""
    A = A.resolve_neg()
    dev = _require_device(A, *b, *(() if C is None else (C,)), *(() if offsets is None else (offsets,)))
    if any(s < 0 for s in A.stride()):
        A = A.contiguous()
    R, K = A.shape
    N = b[0].shape[-2]
    o, o64 = offsets_of(offsets)
    D, c = _output_like(C, beta, (R, N), out_dtype, dev)
    ws = torch.empty(_from_workspace(R, K), dtype=torch.uint8, device=dev)
    _probed_call(
        "mx_gemm", "trnblas_hip_mx_gemm_from", _lib.DTYPE_CODES[A.dtype], _lib.DTYPE_CODES[out_dtype],
        1 if offsets is None else b[0].shape[0], R, N, K, float(alpha), ptr(A), A.stride(0), A.stride(1), ptr(b[0]), ptr(b[1]),
        ptr(o), o64, float(beta) if c is not None else 0.0, ptr(c), max(c.stride(0), N) if c is not None else N, ptr(D),
        max(N, 1), ptr(ws), ws.numel(), stream_of(dev),
    )  # fmt: skip
    return D


def _from_workspace(R: int, K: int) -> int:
    """trnblas_hip_mx_gemm_from_workspace (the same formula; a library call costs more)."""
    return -(-R * -(-K // 32) * 16 // 256) * 256 + -(-R // 16) * -(-K // 512) * 256


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
    o, o64 = offsets_of(offsets)
    D, c = _output_like(C, beta, (R, N), out_dtype, dev)
    _probed_call(
        "mx_gemm", "trnblas_hip_mx_gemm", _lib.DTYPE_CODES[out_dtype], 1 if offsets is None else b[0].shape[0], R, N, K,
        float(alpha), ptr(a[0]), ptr(a[1]), ptr(b[0]), ptr(b[1]), ptr(o), o64, float(beta) if c is not None else 0.0,
        ptr(c), max(c.stride(0), N) if c is not None else N, ptr(D), max(N, 1), stream_of(dev),
    )  # fmt: skip
    return D


# ── the common calls without the general path's checks, one by one ────────────
#
# A call with few rows takes as long on the host as on the GPU (the general path
# 12 us, these 8). Each returns None where anything is out of the ordinary: the
# general path then reports it or deals with it.

_PACK_LOOK = 1 << 30  # multiply-adds below which no packing pays
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice
_fns: dict = {}
_INTS = (torch.int32, torch.int64)


def _fn(name: str):
    f = _fns.get(name)
    if f is None:
        f = _fns[name] = getattr(_lib.load(), name)
    return f


def _checked(name: str, rc: int) -> None:
    if rc < 0:
        msg = _lib.load().trnblas_hip_last_error()
        raise _lib.HipKernelError(name, rc, msg.decode() if msg else "")


def grouped_gemm_fast(alpha, A, B, offsets, transB, out_dtype):
    code = _lib.DTYPE_CODES.get(A.dtype)
    if code is None or B.dtype is not A.dtype or _kernels._launch_probe is not None or A.dim() != 2 or B.dim() != 3:
        return None
    R, K = A.shape
    lda, s1 = A.stride()
    G, b0, b1 = B.shape
    sb, t0, t1 = B.stride()
    k, N = (b1, b0) if transB else (b0, b1)
    dev = A.get_device()
    if (
        k != K or s1 != 1 or lda < K or t1 != 1 or t0 < b1 or sb < 0 or N == 0 or dev != _current_device()
        or B.get_device() != dev or A.is_neg() or B.is_neg()
    ):  # fmt: skip
        return None
    o, o64 = None, False
    if offsets is not None:
        if (
            offsets.get_device() != dev or offsets.dtype not in _INTS or offsets.shape != (G + 1,) or offsets.stride() != (1,)
        ):  # fmt: skip
            return None
        o, o64 = offsets.data_ptr(), offsets.dtype is torch.int64
    if out_dtype is not None and out_dtype is not A.dtype and out_dtype is not torch.float32:
        return None
    pa, pb = A.data_ptr(), B.data_ptr()
    ev = 4 if code == 0 else 8
    if (pa | pb) % 16 or (lda | t0 | sb | K | b1) % ev:
        if R * K * N > _PACK_LOOK:
            return None  # the general path may pack
    D = A.new_empty((R, N), dtype=out_dtype)
    rc = _fn("trnblas_hip_grouped_gemm")(
        code, D.dtype is torch.float32, transB, G, R, N, K, alpha, pa, lda, pb, t0, sb, o, o64, 0.0, None, N,
        D.data_ptr(), N, 0, _raw_stream(dev),
    )  # fmt: skip
    _checked("trnblas_hip_grouped_gemm", rc)
    return D


def mx_gemm_fast(alpha, A, b, offsets, out_dtype):
    """b: (codes, scales) of the quantised operand."""
    code = _lib.DTYPE_CODES.get(A.dtype)
    out = code if out_dtype is None else _lib.DTYPE_CODES.get(out_dtype)
    if code is None or out is None or _kernels._launch_probe is not None or A.dim() != 2:
        return None
    codes, scales = b
    R, K = A.shape
    sr, sk = A.stride()
    dev = A.get_device()
    N = codes.shape[-2]
    if dev != _current_device() or codes.get_device() != dev or sr < 0 or sk < 0 or N == 0 or A.is_neg():
        return None
    G, o, o64 = 1, None, False
    if offsets is not None:
        G = codes.shape[0]
        if (
            offsets.get_device() != dev or offsets.dtype not in _INTS or offsets.shape != (G + 1,) or offsets.stride() != (1,)
        ):  # fmt: skip
            return None
        o, o64 = offsets.data_ptr(), offsets.dtype is torch.int64
    D = A.new_empty((R, N), dtype=out_dtype)
    n = _from_workspace(R, K)
    ws = codes.new_empty(n)
    rc = _fn("trnblas_hip_mx_gemm_from")(
        code, out, G, R, N, K, alpha, A.data_ptr(), sr, sk, codes.data_ptr(), scales.data_ptr(), o, o64, 0.0, None, N,
        D.data_ptr(), N, ws.data_ptr(), n, _raw_stream(dev),
    )  # fmt: skip
    _checked("trnblas_hip_mx_gemm_from", rc)
    return D


def grouped_rank_k_fast(alpha, A, B, offsets, out_dtype):
    code = _lib.DTYPE_CODES.get(A.dtype)
    if code is None or B.dtype is not A.dtype or _kernels._launch_probe is not None or A.dim() != 2 or B.dim() != 2:
        return None
    R, M = A.shape
    R2, N = B.shape
    lda, s1 = A.stride()
    ldb, t1 = B.stride()
    dev = A.get_device()
    if (
        R2 != R or s1 != 1 or lda < M or t1 != 1 or ldb < N or M == 0 or N == 0 or dev != _current_device() or B.get_device() != dev
        or A.is_neg() or B.is_neg()
    ):  # fmt: skip
        return None
    G, o, o64 = 1, None, False
    if offsets is not None:
        if offsets.get_device() != dev or offsets.dtype not in _INTS or offsets.dim() != 1 or offsets.stride() != (1,):
            return None
        G, o, o64 = offsets.shape[0] - 1, offsets.data_ptr(), offsets.dtype is torch.int64
    if out_dtype is not None and out_dtype is not A.dtype and out_dtype is not torch.float32:
        return None
    ev = 4 if code == 0 else 8
    if (A.data_ptr() | B.data_ptr()) % 16 or (lda | ldb | M | N) % ev:
        if R * M * N > _PACK_LOOK:
            return None
    D = A.new_empty((G, M, N), dtype=out_dtype)
    rc = _fn("trnblas_hip_grouped_rank_k")(
        code, D.dtype is torch.float32, G, R, M, N, alpha, A.data_ptr(), lda, B.data_ptr(), ldb, o, o64, 0.0, None, N, 0,
        D.data_ptr(), N, M * N, 0, _raw_stream(dev),
    )  # fmt: skip
    _checked("trnblas_hip_grouped_rank_k", rc)
    return D


def mx_quantize_fast(X):
    """(codes, scales) of X (R, K), or None."""
    code = _lib.DTYPE_CODES.get(X.dtype)
    dev = X.get_device()
    if code is None or dev != _current_device() or X.dim() != 2 or _kernels._launch_probe is not None:
        return None
    R, K = X.shape
    sr, sk = X.stride()
    if sr < 0 or sk < 0 or X.is_neg():
        return None
    codes = X.new_empty((R, -(-K // 32) * 16), dtype=torch.uint8)
    scales = X.new_empty((-(-R // 16), -(-K // 512), 256), dtype=torch.uint8)
    rc = _fn("trnblas_hip_mx_quantize")(
        code, R, K, X.data_ptr(), sr, sk, 0, codes.data_ptr(), scales.data_ptr(), 1, _raw_stream(dev)
    )
    _checked("trnblas_hip_mx_quantize", rc)
    return codes, scales


def mx_dequantize_fast(codes, scales, K, dtype):
    """The values of one matrix, or None."""
    dev = codes.get_device()
    if dev != _current_device() or codes.dim() != 2 or _kernels._launch_probe is not None:
        return None
    R = codes.shape[0]
    D = codes.new_empty((R, K), dtype=dtype)
    rc = _fn("trnblas_hip_mx_dequantize")(
        _lib.DTYPE_CODES[dtype], R, K, codes.data_ptr(), scales.data_ptr(), D.data_ptr(), K or 1, R * K, 1, _raw_stream(dev)
    )
    _checked("trnblas_hip_mx_dequantize", rc)
    return D
