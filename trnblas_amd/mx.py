"""Microscaled 4-bit floats: `mx_quantize`, `mx_dequantize`, `mx_gemm`, `mx_grouped_gemm`.

A value is an e2m1 code (0, .5, 1, 1.5, 2, 3, 4, 6 and a sign) times a power of
two shared by 32 values along K: 4.25 bits a value. The products run on the
4-bit matrix instructions, exact per product, with fp32 sums. No counterpart
in the reference; the products' signatures follow `gemm` and `grouped_gemm`.

    W = mx_quantize(weights)                   # (N, K), once
    y = mx_gemm(1.0, x, W)                     # x (M, K): quantised on the way
    E = mx_quantize(experts)                   # (G, N, K)
    y = mx_grouped_gemm(1.0, x, E, offsets)    # rows sorted by expert

Quantisation of a block: e = floor(log2(max |x|)) - 2 (at least -127), codes
x / 2^e rounded to nearest even and saturated at 6. A block that holds an
infinity or a NaN becomes NaN as a whole. There is no gradient through a
quantised operand: the products refuse operands that require one or carry
a forward-mode tangent.
"""

from __future__ import annotations

import torch
from torch.autograd import forward_ad as _fwd

from ._flags import trans_flag
from .grouped import _check_offsets, _check_result, _gk
from .hip import dispatch as _d

__all__ = ["MXMatrix", "mx_quantize", "mx_dequantize", "mx_gemm", "mx_grouped_gemm"]

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)
_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


class MXMatrix:
    """A matrix (R, K), or a stack (G, R, K), of microscaled 4-bit floats.

    codes: uint8 (..., R, ceil(K / 32) * 16), two codes per byte, the even value
    in the low half. scales: uint8 (..., ceil(R / 16), ceil(K / 512), 256) in the
    order the matrix instructions take them (include/trnblas_hip.h);
    `block_scales` and `from_parts` go to and from plain rows of scale bytes.
    """

    __slots__ = ("codes", "scales", "shape")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, shape):
        shape = torch.Size(shape)
        *lead, R, K = shape
        if len(shape) not in (2, 3):
            raise ValueError(f"MXMatrix: shape must be (R, K) or (G, R, K), got {tuple(shape)}")
        for name, t, want in (("codes", codes, (*lead, R, -(-K // 32) * 16)),
                              ("scales", scales, (*lead, -(-R // 16), -(-K // 512), 256))):  # fmt: skip
            if t.dtype != torch.uint8 or tuple(t.shape) != want:
                raise ValueError(f"MXMatrix: {name} must be uint8 {want}, got {t.dtype} {tuple(t.shape)}")
        if codes.device != scales.device:
            raise ValueError(f"MXMatrix: codes on {codes.device}, scales on {scales.device}")
        # the kernels take both as whole 16-byte groups in a row
        codes, scales = (t if t.is_contiguous() and t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)
                         for t in (codes, scales))  # fmt: skip
        self.codes, self.scales, self.shape = codes, scales, shape

    @classmethod
    def _of(cls, codes: torch.Tensor, scales: torch.Tensor, shape) -> MXMatrix:
        """From buffers that this package laid out itself."""
        Q = object.__new__(cls)
        Q.codes, Q.scales, Q.shape = codes, scales, torch.Size(shape)
        return Q

    @classmethod
    def from_parts(cls, codes: torch.Tensor, block_scales: torch.Tensor, K: int) -> MXMatrix:
        """From codes (as above; values past K must be zero codes) and plain
        scale bytes (..., R, ceil(K / 32)), as checkpoints store them."""
        *lead, R, nb = block_scales.shape
        if block_scales.dtype != torch.uint8 or nb != -(-K // 32):
            raise ValueError(f"MXMatrix: block_scales must be uint8 (..., R, {-(-K // 32)}), got "
                             f"{block_scales.dtype} {tuple(block_scales.shape)}")  # fmt: skip
        s = torch.nn.functional.pad(block_scales, (0, -nb % 16, 0, -R % 16))
        s = s.reshape(*lead, -(-R // 16), 16, -(-nb // 16), 4, 4)  # rows, chunks, b / 4, b % 4
        n = len(lead)
        s = s.permute(*range(n), n, n + 2, n + 4, n + 1, n + 3).reshape(*lead, -(-R // 16), -(-nb // 16), 256)
        return cls(codes, s, (*lead, R, K))

    def block_scales(self) -> torch.Tensor:
        """The scale bytes as plain rows: uint8 (..., R, ceil(K / 32))."""
        *lead, R, K = self.shape
        n = len(lead)
        s = self.scales.reshape(*self.scales.shape[:-1], 4, 16, 4)  # b % 4, row, b / 4
        s = s.permute(*range(n), n, n + 3, n + 1, n + 4, n + 2)
        s = s.reshape(*lead, self.scales.shape[n] * 16, self.scales.shape[n + 1] * 16)
        return s[..., :R, : -(-K // 32)]

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        return mx_dequantize(self, dtype)

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()

    def to(self, device) -> MXMatrix:
        return MXMatrix(self.codes.to(device), self.scales.to(device), self.shape)

    def __getitem__(self, g: int) -> MXMatrix:
        """Matrix g of a stack."""
        if len(self.shape) != 3:
            raise ValueError("MXMatrix: only a stack of matrices is indexed")
        return MXMatrix(self.codes[g], self.scales[g], self.shape[1:])

    def __repr__(self) -> str:
        return f"MXMatrix(shape={tuple(self.shape)}, device={self.device})"


def _pow2(e: torch.Tensor) -> torch.Tensor:
    """2^e in fp32 for whole e of -127 .. 127, from its bits."""
    return torch.where(e < -126, 1 << 22, (e + 127) << 23).to(torch.int32).view(torch.float32)


def _quantize_torch(X: torch.Tensor) -> MXMatrix:
    x = torch.nn.functional.pad(X.float(), (0, -X.shape[-1] % 32)).unflatten(-1, (-1, 32))
    bits = x.abs().contiguous().view(torch.int32)
    field = bits.amax(-1) >> 23
    byte = torch.where(field == 255, 255, (field - 2).clamp_min(0))
    y = x * _pow2((127 - byte).clamp_min(-127)).unsqueeze(-1)
    a = torch.where((byte == 255).unsqueeze(-1), 0.0, y.abs())
    c = (a > 0.25).to(torch.uint8)
    for up in (a >= 0.75, a > 1.25, a >= 1.75, a > 2.5, a >= 3.5, a > 5.0):
        c += up
    c += 8 * ((y < 0) & (a == y.abs())).to(torch.uint8)
    c = c.flatten(-2)
    return MXMatrix.from_parts((c[..., ::2] | c[..., 1::2] << 4).contiguous(), byte.to(torch.uint8), X.shape[-1])


def _dequantize_torch(Q: MXMatrix, dtype: torch.dtype) -> torch.Tensor:
    table = torch.tensor(_VALUES + tuple(-v for v in _VALUES), device=Q.device)
    c = torch.stack([Q.codes & 15, Q.codes >> 4], -1).flatten(-2)
    s = Q.block_scales().int()
    scale = torch.where(s == 255, float("nan"), _pow2((s - 127).clamp_max(127)))
    v = table[c.int()].unflatten(-1, (-1, 32)) * scale.unsqueeze(-1)
    return v.flatten(-2)[..., : Q.shape[-1]].to(dtype)


def mx_quantize(X: torch.Tensor, trans: bool = False) -> MXMatrix:
    """X (R, K) or (G, R, K) as microscaled 4-bit floats, blocks along K.

    trans: X is stored the other way round, (K, R) or (G, K, R) (weights kept
    as the right operand of a product); it is read in place, as any strided
    view is. float32, bfloat16 or float16 (others are rounded to float32
    first). The result carries no gradient.
    """
    if not isinstance(X, torch.Tensor) or X.dim() not in (2, 3):
        raise ValueError("mx_quantize: X must be a 2-D or 3-D tensor")
    if not X.is_floating_point():
        raise TypeError(f"mx_quantize: X must be a real floating tensor, got {X.dtype}")
    if X.requires_grad:
        X = X.detach()
    if X.dtype not in _FLOATS:
        X = X.float()
    if trans_flag(trans):
        X = X.mT
    if _d.mx_on_hip(X):
        try:
            parts = _gk().mx_quantize_fast(X)
            if parts is not None:
                return MXMatrix._of(*parts, X.shape)
            return MXMatrix._of(*_gk().mx_quantize(X), X.shape)
        except Exception as exc:  # noqa: BLE001
            _d._kernel_failed(exc)
    return _quantize_torch(X)


def mx_dequantize(Q: MXMatrix, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values of Q, rounded to nearest even in `dtype` (float32 and bfloat16
    hold them exactly, but for bfloat16 values below 2^-133)."""
    if not isinstance(Q, MXMatrix):
        raise TypeError(f"mx_dequantize: an MXMatrix is needed, got {type(Q).__name__}")
    if dtype not in _FLOATS:
        raise TypeError(f"mx_dequantize: dtype {dtype} (float32, bfloat16 or float16)")
    if _d.mx_on_hip(Q.codes):
        try:
            D = _gk().mx_dequantize_fast(Q.codes, Q.scales, Q.shape[-1], dtype)
            return _gk().mx_dequantize(Q.codes, Q.scales, Q.shape[-1], dtype) if D is None else D
        except Exception as exc:  # noqa: BLE001
            _d._kernel_failed(exc)
    return _dequantize_torch(Q, dtype)


def _product(what: str, alpha, A, B, offsets, beta, C, dtype) -> torch.Tensor:
    dims = 2 if offsets is None else 3
    if (
        beta == 0.0 and type(A) is torch.Tensor and A.is_cuda and type(B) is MXMatrix and len(B.shape) == dims
        and A.dim() == 2 and A.shape[1] == B.shape[-1] and (offsets is None or type(offsets) is torch.Tensor)
        and not (A.requires_grad and torch.is_grad_enabled()) and _fwd._current_level < 0 and _d._use_hip()
    ):  # fmt: skip
        try:  # the short way; None: something is out of the ordinary
            D = _gk().mx_gemm_fast(alpha, A, (B.codes, B.scales), offsets, dtype)
            if D is not None:
                return D
        except _d.HipKernelError as exc:
            _d._kernel_failed(exc)
    if not isinstance(B, MXMatrix) or len(B.shape) != dims:
        raise ValueError(f"{what}: B must be an MXMatrix of {dims} dimensions (see mx_quantize)")
    if isinstance(A, torch.Tensor):
        if A.dim() != 2:
            raise ValueError(f"{what}: A must be 2-D, got {tuple(A.shape)}")
        if A.dtype not in _FLOATS:
            raise TypeError(f"{what}: A is {A.dtype} (float32, bfloat16, float16 or an MXMatrix)")
        if _d._wants_grad(A):
            raise NotImplementedError(f"{what}: no gradient through a quantised operand (detach A, or use no_grad)")
        default = A.dtype
    elif isinstance(A, MXMatrix) and len(A.shape) == 2:
        default = torch.bfloat16
    else:
        raise ValueError(f"{what}: A must be a 2-D tensor or MXMatrix")
    if A.shape[1] != B.shape[-1]:
        raise ValueError(f"{what}: inner dimensions differ: A {tuple(A.shape)}, B {tuple(B.shape)}")
    if A.device != B.device:
        raise ValueError(f"{what}: operands on different devices: {A.device} and {B.device}")
    codes = A.codes if isinstance(A, MXMatrix) else A
    if offsets is not None:
        _check_offsets(what, offsets, codes, B.shape[0])
    shape = (A.shape[0], B.shape[-2])
    out = default if dtype is None else dtype
    _check_result(what, shape, out, beta, C, codes, _FLOATS)
    if beta != 0.0 and _d._wants_grad(C):
        raise NotImplementedError(f"{what}: no gradient (detach C, or use no_grad)")
    c = C.expand(shape) if beta != 0.0 else None
    if _d.mx_on_hip(codes, B.codes):
        try:
            b = (B.codes, B.scales)
            if isinstance(A, MXMatrix):
                return _gk().mx_gemm((A.codes, A.scales), b, A.shape[1], out, offsets, alpha, beta, c)
            return _gk().mx_gemm_from(A, b, out, offsets, alpha, beta, c)
        except Exception as exc:  # noqa: BLE001
            _d._kernel_failed(exc)
    a = _dequantize_torch(A if isinstance(A, MXMatrix) else _quantize_torch(A), torch.float32)
    b = _dequantize_torch(B, torch.float32).mT
    P = a.new_zeros(shape)
    if offsets is None:
        P = a @ b
    else:
        for g, i, j in _d._group_rows(offsets, shape[0]):
            P[i:j] = a[i:j] @ b[g]
    return _d._scaled_sum(P, alpha, beta, c, out)


def mx_gemm(
    alpha: float,
    A: torch.Tensor | MXMatrix,
    B: MXMatrix,
    beta: float = 0.0,
    C: torch.Tensor | None = None,
    dtype: torch.dtype | None = None,
) -> torch.Tensor:
    """alpha * A @ B^T + beta * C for A (M, K) and an MXMatrix B (N, K).

    A is an MXMatrix, or a float tensor that is quantised on the way. The
    result (M, N) has `dtype` (float32, bfloat16 or float16), A's by default
    (bfloat16 for an MXMatrix).
    """
    return _product("mx_gemm", alpha, A, B, None, beta, C, dtype)


def mx_grouped_gemm(
    alpha: float,
    A: torch.Tensor | MXMatrix,
    B: MXMatrix,
    offsets: torch.Tensor,
    beta: float = 0.0,
    C: torch.Tensor | None = None,
    dtype: torch.dtype | None = None,
) -> torch.Tensor:
    """D[r] = alpha * A[r] @ B[g]^T + beta * C[r] for the rows r of group g:
    `grouped_gemm` with microscaled operands, A (R, K) as in `mx_gemm`, B
    (G, N, K). Rows of no group come out as beta * C[r]."""
    if offsets is None:
        raise ValueError("mx_grouped_gemm: offsets must be a 1-D tensor of groups + 1 row numbers")
    return _product("mx_grouped_gemm", alpha, A, B, offsets, beta, C, dtype)
