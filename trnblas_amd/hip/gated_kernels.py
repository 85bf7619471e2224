"""Tensor-level wrappers of the gated projections' C ABI, in the manner of
`grouped_kernels.py`.
"""

from __future__ import annotations

import torch

from . import _lib
from ._lib import ptr, stream_of
from . import grouped_kernels as _grouped
from . import kernels as _kernels
from .grouped_kernels import _checked, _fn, _ready, _up, grouped_gemm, offsets_of, row_major
from .kernels import _batched_layout, _pack_k, _probed_call, _require_device

ACTS = {"silu": 0, "gelu": 1, "gelu_tanh": 2, "relu": 3, "sigmoid": 4}  # TRNBLAS_ACT_*


def _call(kernel: str, dev: int, *args) -> None:
    """The C entry of `kernel` on `dev`'s current stream: the short way where `dev` is the current device and nothing is probed."""
    name = "trnblas_hip_" + kernel
    if dev == _grouped._current_device() and _kernels._launch_probe is None:
        _checked(name, _fn(name)(*args, _grouped._raw_stream(dev)))
    else:
        _probed_call(kernel, name, *args, stream_of(torch.device("cuda", dev)))


def gate(P: torch.Tensor, act: str, out_dtype: torch.dtype, save: bool):
    """(H, S): act(P[:, :N]) * P[:, N:] in out_dtype, and where `save` says so P (contiguous) in that type."""
    R, N = P.shape[0], P.shape[1] // 2
    H = P.new_empty((R, N), dtype=out_dtype)
    S = P.new_empty((R, 2 * N), dtype=out_dtype) if save and out_dtype != P.dtype else None
    _call(
        "gate", P.get_device(), ACTS[act], _lib.DTYPE_CODES[P.dtype], _lib.DTYPE_CODES[out_dtype], R, N, P.data_ptr(),
        max(2 * N, 1), H.data_ptr(), max(N, 1), ptr(S), max(2 * N, 1),
    )  # fmt: skip
    return H, (P if S is None else S) if save else None


def gate_backward(P: torch.Tensor, dH: torch.Tensor, act: str) -> torch.Tensor:
    """dP, in dH's type, of H = act(P[:, :N]) * P[:, N:] for the gradient dH of H; P fp32."""
    R, N = dH.shape
    ldg = N
    if dH.stride() != (N, 1) or dH.is_neg():
        dH, ldg = row_major(dH.resolve_neg())
    D = P.new_empty((R, 2 * N), dtype=dH.dtype)
    _call(
        "gate_backward", P.get_device(), ACTS[act], _lib.DTYPE_CODES[dH.dtype], R, N, P.data_ptr(), max(2 * N, 1), dH.data_ptr(),
        max(ldg, N), D.data_ptr(), max(2 * N, 1),
    )  # fmt: skip
    return D


# An fp32 result of 16-bit operands goes through the fp32 product, as it stands, and a launch of the gate.
# Operands that the fused kernels cannot read in place are copied first, rows padded with zeros, from so many
# multiply-adds on; below it the product goes to fp32 by `grouped_gemm`'s kernels, and the gate is a launch of its own.
_PACK_MACS = 1 << 30
# So do operands whose rows lie too far apart: a tile's rows (128 bytes of k, of a B whose columns are contiguous) have 32-bit
# offsets (dma_ready, csrc/grouped_run.hpp). The last tokens of sequences, x[:, -1] of (batch, tokens, width), are such rows.
_REACH = (1 << 31) - 1025


def _far(lda: int, ldb: int, kc: bool, es: int) -> bool:
    return 256 * lda * es >= _REACH or (256 * es if kc else 128) * ldb >= _REACH


def gated_gemm(A: torch.Tensor, B: torch.Tensor, offsets, act: str, out_dtype: torch.dtype, save: bool):
    """(H, P) for A (R, K) and B (G, K, 2 N): H = act(G) * U of P = [G | U] = A[r] @ B[g]; P (fp32)
    only where `save` says so, else None. Rows of no group are zeros."""
    A, B = A.resolve_neg(), B.resolve_neg()
    dev = _require_device(A, B, offsets)
    R, K = A.shape
    G, N = B.shape[0], B.shape[2] // 2
    es = A.element_size()
    ev, padded = 16 // es, False
    a, lda = row_major(A)
    b, tb, ldb, sb = _batched_layout(B)
    su = N * ldb if tb else N
    if R == 1:
        lda = max(K, 1)
    ka, kb = _up(K, ev), _up(K, ev) if tb else 2 * _up(N, ev)  # leading dimensions of copies
    a_ok = _ready(a.data_ptr(), lda, 0, K, ev) and not _far(lda, 0, tb, es)
    b_ok = _ready(b.data_ptr(), ldb, sb, K if tb else N, ev) and su % ev == 0 and not _far(0, ldb, tb, es)
    beyond = (not a_ok and _far(ka, 0, tb, es)) or (not b_ok and _far(0, kb, tb, es))
    if out_dtype != A.dtype or beyond or (not (a_ok and b_ok) and 2 * R * K * N < _PACK_MACS):
        P = grouped_gemm(A, B, offsets, out_dtype=torch.float32)
        return gate(P, act, out_dtype, False)[0], P if save else None
    if not a_ok:
        a, lda, padded = _pack_k(A, ka), ka, True
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
    P = torch.empty((R, 2 * N), dtype=torch.float32, device=dev) if save else None
    _probed_call(
        "gated_gemm", "trnblas_hip_gated_gemm", ACTS[act], _lib.DTYPE_CODES[A.dtype], int(tb), G, R, N, K, ptr(a), lda, ptr(b), ldb, sb, su, ptr(o), o64, ptr(H), max(N, 1), ptr(P), max(2 * N, 1),
        int(padded), stream_of(dev),
    )  # fmt: skip
    return H, P


def gated_gemm_fast(A, B, offsets, act, transB, out_dtype, save=False):
    """The common calls without the general path's checks, one by one, as in `grouped_kernels.py` (15 us on the host, these 9; two
    launches 29 and 16): B as given (without offsets 2-D or a stack of one). None where anything is out of the ordinary; (H, P)
    where `save` says so, else H."""
    code, a = _lib.DTYPE_CODES.get(A.dtype), ACTS.get(act)
    if code is None or a is None or B.dtype is not A.dtype or _kernels._launch_probe is not None or A.dim() != 2:
        return None
    same = out_dtype is None or out_dtype is A.dtype
    if (not same and out_dtype is not torch.float32) or (B.dim() != 3 and (B.dim() != 2 or offsets is not None)):
        return None
    R, K = A.shape
    lda, s1 = A.stride()
    G, sb, o, o64 = 1, 0, None, False
    dev = A.get_device()
    if offsets is not None:
        G, sb = B.shape[0], B.stride(0)
        if (
            offsets.get_device() != dev or offsets.dtype not in _grouped._INTS or offsets.shape != (G + 1,)
            or offsets.stride() != (1,) or sb < 0
        ):  # fmt: skip
            return None
        o, o64 = offsets.data_ptr(), offsets.dtype is torch.int64
    elif B.dim() == 3 and B.shape[0] != 1:
        return None
    b0, b1 = B.shape[-2:]
    t0, t1 = B.stride()[-2:]
    k, n2 = (b1, b0) if transB else (b0, b1)
    N = n2 // 2
    pa, pb = A.data_ptr(), B.data_ptr()
    su = N * t0 if transB else N
    if R == 1:
        lda = max(K, 1)
    if (
        k != K or n2 % 2 or s1 != 1 or lda < K or t1 != 1 or t0 < b1 or N == 0 or dev != _grouped._current_device()
        or B.get_device() != dev or A.is_neg() or B.is_neg()
    ):  # fmt: skip
        return None
    if not same or (pa | pb) % 16 or (lda | t0 | sb | su | K | b1) % (4 if code == 0 else 8) or _far(lda, t0, transB, 4 if code == 0 else 2):
        if same and R * K * n2 >= _PACK_MACS:
            return None
        P = _grouped.grouped_gemm_fast(1.0, A, B if B.dim() == 3 else B.unsqueeze(0), offsets, transB, torch.float32)
        if P is None:
            return None
        H = gate(P, act, out_dtype or A.dtype, False)[0]
        return (H, P) if save else H
    H = A.new_empty((R, N))
    P = A.new_empty((R, n2), dtype=torch.float32) if save else None
    rc = _fn("trnblas_hip_gated_gemm")(
        a, code, transB, G, R, N, K, pa, lda, pb, t0, sb, su, o, o64, H.data_ptr(), N, P.data_ptr() if save else None, n2, 0,
        _grouped._raw_stream(dev),
    )  # fmt: skip
    _checked("trnblas_hip_gated_gemm", rc)
    return (H, P) if save else H
