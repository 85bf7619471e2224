"""4-bit integer weights with scales of groups: `int4_quantize`, `int4_dequantize`, `int4_gemm`, `int4_grouped_gemm`.

A weight is (q - z) s: q of 4 bits, a scale s (bfloat16 or float16) and, where a matrix has them, a
zero point z for each group of 32, 64 or 128 values along K (z = 8 otherwise): 4.125 to 4.75 bits a
value. Rows stay in their type: the products are of exact weights, with fp32 sums (float32 rows
enter as three bfloat16 pieces whose sum they are). No counterpart in the reference; signatures as
of `mx_gemm` and `mx_grouped_gemm`, and `gated_gemm` / `grouped_gated_gemm` take such weights too.

    W = int4_quantize(weights)                               # (N, K), once
    W = Int4Matrix.from_parts(codes, scales, K, 128, zeros)  # or what a checkpoint holds
    y = int4_gemm(1.0, x, W)                                 # x (M, K)
    h = gated_gemm(x, W, "silu")                             # gate rows, then up rows
    y = int4_grouped_gemm(1.0, x, E, offsets)                # rows sorted by expert, E (G, N, K)

There is no gradient through these products: they refuse operands that require one or carry a
forward-mode tangent.
"""

from __future__ import annotations

import torch
from torch.autograd import forward_ad as _fwd

from ._flags import trans_flag
from .grouped import _check_offsets, _check_result
from .hip import dispatch as _d

__all__ = ["Int4Matrix", "int4_quantize", "int4_dequantize", "int4_gemm", "int4_grouped_gemm"]

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)
_SCALES = (torch.bfloat16, torch.float16)
_GROUPS = (32, 64, 128)
_NIBBLES = [0, 2, 4, 6, 1, 3, 5, 7]  # which of a dword's eight values each nibble holds

_kernels = None


def _gk():
    global _kernels
    if _kernels is None:
        from .hip import int4_kernels

        _kernels = int4_kernels
    return _kernels


def _check_group(what: str, group) -> int:
    if type(group) is not int or group not in _GROUPS:
        raise ValueError(f"{what}: group must be 32, 64 or 128, got {group!r}")
    return group


class Int4Matrix:
    """A matrix (R, K), or a stack (G, R, K), of 4-bit integer weights.

    codes: uint8 (..., ceil(R / 16), ceil(K / 128), 1024); scales: bfloat16 or float16 (..., ceil(R / 16),
    ceil(K / 128), 16, 128 / group); zeros: uint8 like the scales, or None: in the order the
    matrix instructions take them (include/trnblas_hip.h). `from_parts` and `parts` go from and to plain rows.
    """

    __slots__ = ("codes", "scales", "zeros", "shape", "group")

    def __init__(self, codes, scales, zeros, shape, group: int):
        shape = torch.Size(shape)
        if len(shape) not in (2, 3):
            raise ValueError(f"Int4Matrix: shape must be (R, K) or (G, R, K), got {tuple(shape)}")
        _check_group("Int4Matrix", group)
        *lead, R, K = shape
        blocks, chunks = -(-R // 16), -(-K // 128)
        of_groups = (*lead, blocks, chunks, 16, 128 // group)
        for name, t, want, types in (("codes", codes, (*lead, blocks, chunks, 1024), (torch.uint8,)),
                                     ("scales", scales, of_groups, _SCALES), ("zeros", zeros, of_groups, (torch.uint8,))):  # fmt: skip
            if t is None and name == "zeros":
                continue
            if not isinstance(t, torch.Tensor) or t.dtype not in types or tuple(t.shape) != want:
                got = f"{t.dtype} {tuple(t.shape)}" if isinstance(t, torch.Tensor) else type(t).__name__
                raise ValueError(f"Int4Matrix: {name} must be {' or '.join(map(str, types))} {want}, got {got}")
            if t.device != codes.device:
                raise ValueError(f"Int4Matrix: codes on {codes.device}, {name} on {t.device}")
        # the kernels take them as whole 16-byte groups in a row
        self.codes, self.scales, self.zeros = (
            t if t is None or (t.is_contiguous() and t.data_ptr() % 16 == 0) else t.clone(memory_format=torch.contiguous_format)
            for t in (codes, scales.detach(), zeros)
        )
        self.shape, self.group = shape, group

    @classmethod
    def _of(cls, parts, shape, group) -> Int4Matrix:
        """From buffers that this package laid out itself."""
        Q = object.__new__(cls)
        Q.codes, Q.scales, Q.zeros = parts
        Q.shape, Q.group = torch.Size(shape), group
        return Q

    @classmethod
    def from_parts(cls, codes: torch.Tensor, scales: torch.Tensor, K: int, group: int, zeros: torch.Tensor | None = None) -> Int4Matrix:
        """From plain rows, as checkpoints store them: codes uint8 (..., R, ceil(K / 2)), two values q to a byte, the even one
        low; scales (..., R, ceil(K / group)), finite or NaN; zeros (whole numbers 0 .. 255) like the scales, or None for 8."""
        _check_group("Int4Matrix", group)
        if type(K) is not int or K < 0:
            raise ValueError(f"Int4Matrix: K must be a whole number, got {K!r}")
        if codes.dtype != torch.uint8 or codes.dim() not in (2, 3) or codes.shape[-1] != -(-K // 2):
            raise ValueError(f"Int4Matrix: codes must be uint8 (..., R, {-(-K // 2)}), got {codes.dtype} {tuple(codes.shape)}")
        *lead, R, _ = codes.shape
        want = (*lead, R, -(-K // group))
        if scales.dtype not in _SCALES or tuple(scales.shape) != want:
            raise ValueError(f"Int4Matrix: scales must be bfloat16 or float16 {want}, got {scales.dtype} {tuple(scales.shape)}")
        if zeros is not None and (zeros.dtype != torch.uint8 or tuple(zeros.shape) != want):
            raise ValueError(f"Int4Matrix: zeros must be uint8 {want}, got {zeros.dtype} {tuple(zeros.shape)}")
        q = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)[..., :K]
        return cls(_laid_out(q), _blocked(scales, K, group), None if zeros is None else _blocked(zeros, K, group), (*lead, R, K), group)

    def parts(self):
        """(codes, scales, zeros) as plain rows: what `from_parts` takes."""
        *lead, R, K = self.shape
        q = _values_of(self.codes)[..., :R, :K]
        q = torch.nn.functional.pad(q, (0, K % 2))
        return (q[..., ::2] | q[..., 1::2] << 4).contiguous(), *(None if t is None else self._rows(t) for t in (self.scales, self.zeros))

    def _rows(self, t):
        """Scales or zero points as rows (..., R, ceil(K / group))."""
        return t.transpose(-3, -2).flatten(-2).flatten(-3, -2)[..., : self.shape[-2], : -(-self.shape[-1] // self.group)]

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        return int4_dequantize(self, dtype)

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + 2 * self.scales.numel() + (0 if self.zeros is None else self.zeros.numel())

    def to(self, device) -> Int4Matrix:
        return Int4Matrix(*(None if t is None else t.to(device) for t in (self.codes, self.scales, self.zeros)), self.shape, self.group)

    def __getitem__(self, g: int) -> Int4Matrix:
        """Matrix g of a stack."""
        if len(self.shape) != 3:
            raise ValueError("Int4Matrix: only a stack of matrices is indexed")
        return Int4Matrix(*(None if t is None else t[g] for t in (self.codes, self.scales, self.zeros)), self.shape[1:], self.group)

    def __repr__(self) -> str:
        return f"Int4Matrix(shape={tuple(self.shape)}, group={self.group}, zeros={self.zeros is not None}, device={self.device})"


def _laid_out(q: torch.Tensor) -> torch.Tensor:
    """Values q (..., R, K) of 0 .. 15 as an Int4Matrix's codes."""
    *lead, R, K = q.shape
    s = torch.nn.functional.pad(q ^ 8, (0, -K % 128, 0, -R % 16))  # q - 8 as a nibble
    s = s.reshape(*lead, -(-R // 16), 16, -(-K // 128), 4, 4, 8)  # rows, chunks, h, p, e
    n = len(lead)
    s = s.permute(*range(n), n, n + 2, n + 4, n + 1, n + 3, n + 5)[..., _NIBBLES]
    s = s.reshape(*lead, -(-R // 16), -(-K // 128), 1024, 2)
    return s[..., 0] | s[..., 1] << 4


def _values_of(codes: torch.Tensor) -> torch.Tensor:
    """The values q (..., rows, columns), whole blocks of them, of an Int4Matrix's codes."""
    *lead, blocks, chunks, _ = codes.shape
    s = torch.stack([codes & 15, codes >> 4], -1).reshape(*lead, blocks, chunks, 4, 16, 4, 8)  # p, r, h, nibble
    s = s[..., [_NIBBLES.index(e) for e in range(8)]]
    n = len(lead)
    s = s.permute(*range(n), n, n + 3, n + 1, n + 4, n + 2, n + 5)
    return s.reshape(*lead, blocks * 16, chunks * 128) ^ 8


def _blocked(t: torch.Tensor, K: int, group: int) -> torch.Tensor:
    """Scales or zero points (..., R, ceil(K / group)) as an Int4Matrix's."""
    *lead, R, n = t.shape
    t = torch.nn.functional.pad(t, (0, -(-K // 128) * (128 // group) - n, 0, -R % 16))
    return t.reshape(*lead, -(-R // 16), 16, -(-K // 128), 128 // group).transpose(-3, -2).contiguous()


def _quantize_torch(X, group, zeros, scale_dtype) -> Int4Matrix:
    K = X.shape[-1]
    x = torch.nn.functional.pad(X.float(), (0, -K % group)).unflatten(-1, (-1, group))
    top = x.abs().amax(-1)  # NaN with a NaN among the values
    if zeros:
        lo, hi = x.amin(-1).clamp_max(0.0), x.amax(-1).clamp_min(0.0)
        s = (hi - lo) / torch.full_like(hi, 15.0)
    else:
        s = top / torch.full_like(top, 7.0)
    s = s.to(scale_dtype)
    bad = ~(top.isfinite() & s.isfinite())
    f = s.float()
    some = (f > 0) & ~bad
    by = torch.where(some, f, 1.0)
    v = torch.round(x.nan_to_num(0.0, 0.0, 0.0) / by.unsqueeze(-1))
    if zeros:
        z = torch.where(some, torch.round(-lo.nan_to_num(0.0, 0.0, 0.0) / by).clamp(0, 15), 0.0)
        q = (v + z.unsqueeze(-1)).clamp(0, 15)
        q = torch.where(some.unsqueeze(-1), q, 0.0)
    else:
        z, q = None, torch.where(some.unsqueeze(-1), v.clamp(-8, 7) + 8, 8.0)
    q = q.flatten(-2)[..., :K].to(torch.uint8)
    s = torch.where(bad, float("nan"), s)
    z = None if z is None else _blocked(z.to(torch.uint8), K, group)
    return Int4Matrix(_laid_out(q), _blocked(s, K, group), z, X.shape, group)


def _dequantize_torch(Q: Int4Matrix, dtype: torch.dtype) -> torch.Tensor:
    R, K = Q.shape[-2:]
    spread = lambda t: Q._rows(t).float().repeat_interleave(Q.group, -1)[..., :K]
    z = 8.0 if Q.zeros is None else spread(Q.zeros)
    return ((_values_of(Q.codes)[..., :R, :K].float() - z) * spread(Q.scales)).to(dtype)


def int4_quantize(
    X: torch.Tensor,
    group: int = 128,
    zeros: bool = False,
    trans: bool = False,
    scale_dtype: torch.dtype = torch.bfloat16,
) -> Int4Matrix:
    """X (R, K) or (G, R, K) as 4-bit integer weights with a scale for each `group` values along K.

    zeros: a zero point for each group too: s = (hi - lo) / 15, z = -lo / s, q = z + x / s, lo and hi the least and
    largest value and zero. Without: s = max |x| / 7, q = 8 + x / s. Quotients go to the nearest whole number
    (even at ties), within 4 bits. A group with an infinity or a NaN, or whose scale passes its type's range,
    becomes NaN as a whole. trans: X is stored the other way round, (K, R) or (G, K, R), and read in
    place, as any strided view is. float32, bfloat16 or float16 (others are rounded to float32
    first). The result carries no gradient.
    """
    if not isinstance(X, torch.Tensor) or X.dim() not in (2, 3):
        raise ValueError("int4_quantize: X must be a 2-D or 3-D tensor")
    if not X.is_floating_point():
        raise TypeError(f"int4_quantize: X must be a real floating tensor, got {X.dtype}")
    _check_group("int4_quantize", group)
    if scale_dtype not in _SCALES:
        raise TypeError(f"int4_quantize: scale_dtype {scale_dtype} (bfloat16 or float16)")
    if X.requires_grad:
        X = X.detach()
    if X.dtype not in _FLOATS:
        X = X.float()
    if trans_flag(trans):
        X = X.mT
    zeros = bool(zeros)
    if _d.mx_on_hip(X):
        try:
            parts = _gk().quantize_fast(X, group, zeros, scale_dtype)
            return Int4Matrix._of(parts or _gk().quantize(X, group, zeros, scale_dtype), X.shape, group)
        except Exception as exc:  # noqa: BLE001
            _d._kernel_failed(exc)
    return _quantize_torch(X, group, zeros, scale_dtype)


def int4_dequantize(Q: Int4Matrix, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The weights of Q, rounded to nearest even in `dtype` (float32 holds them exactly)."""
    if not isinstance(Q, Int4Matrix):
        raise TypeError(f"int4_dequantize: an Int4Matrix is needed, got {type(Q).__name__}")
    if dtype not in _FLOATS:
        raise TypeError(f"int4_dequantize: dtype {dtype} (float32, bfloat16 or float16)")
    if _d.mx_on_hip(Q.codes):
        try:
            q = Q.codes, Q.scales, Q.zeros
            D = _gk().dequantize_fast(q, Q.shape, Q.group, dtype)
            return _gk().dequantize(q, Q.shape, Q.group, dtype) if D is None else D
        except Exception as exc:  # noqa: BLE001
            _d._kernel_failed(exc)
    return _dequantize_torch(Q, dtype)


def _fast_product(alpha, A, B, offsets, dtype, dims, act=None):
    """The short way (`int4_gemm_fast`); None: something is out of the ordinary."""
    if (
        type(A) is torch.Tensor and A.is_cuda and type(B) is Int4Matrix and len(B.shape) == dims
        and (offsets is None if dims == 2 else type(offsets) is torch.Tensor)
        and not (A.requires_grad and torch.is_grad_enabled()) and _fwd._current_level < 0 and _d._use_hip()
    ):  # fmt: skip
        try:
            return _gk().int4_gemm_fast(alpha, A, B, offsets, dtype, act)
        except _d.HipKernelError as exc:
            _d._kernel_failed(exc)
    return None


def _product(what: str, alpha, A, B, offsets, beta, C, dtype, gate=None, grouped=False) -> torch.Tensor:
    """gate: None, or (activation, its function of [G | U]) for B of 2 N rows."""
    dims = 3 if grouped else 2
    if beta == 0.0:
        D = _fast_product(alpha, A, B, offsets, dtype, dims, gate and gate[0])
        if D is not None:
            return D
    if not isinstance(B, Int4Matrix) or len(B.shape) != dims:
        raise ValueError(f"{what}: B must be an Int4Matrix of {dims} dimensions (see int4_quantize)")
    if not isinstance(A, torch.Tensor) or A.dim() != 2:
        raise ValueError(f"{what}: A must be a 2-D tensor")
    if A.dtype not in _FLOATS:
        raise TypeError(f"{what}: A is {A.dtype} (float32, bfloat16 or float16)")
    if _d._wants_grad(A):
        raise NotImplementedError(f"{what}: no gradient through 4-bit weights (detach A, or use no_grad)")
    if A.shape[1] != B.shape[-1]:
        raise ValueError(f"{what}: inner dimensions differ: A {tuple(A.shape)}, B {tuple(B.shape)}")
    if A.device != B.device:
        raise ValueError(f"{what}: operands on different devices: {A.device} and {B.device}")
    if grouped:
        _check_offsets(what, offsets, A, B.shape[0])
    N = B.shape[-2]
    if gate is not None:
        if N % 2:
            raise ValueError(f"{what}: B must have the gates' rows and as many again, got {N}")
        N //= 2
    shape = (A.shape[0], N)
    out = _check_result(what, shape, dtype, beta, C, A, _FLOATS)
    if beta != 0.0 and _d._wants_grad(C):
        raise NotImplementedError(f"{what}: no gradient (detach C, or use no_grad)")
    c = C.expand(shape) if beta != 0.0 else None
    if _d.mx_on_hip(A, B.codes):
        try:
            q = (B.codes, B.scales, B.zeros)
            return _gk().int4_gemm(A, q, N, B.group, out, offsets, alpha, beta, c, gate and gate[0])
        except Exception as exc:  # noqa: BLE001
            _d._kernel_failed(exc)
    W = _dequantize_torch(B, torch.float32).mT
    P = _d.grouped_gemm(1.0, A.float(), W if grouped else W[None], offsets, 0.0, None, torch.float32)
    return gate[1](P).to(out) if gate is not None else _d._scaled_sum(P, alpha, beta, c, out)


def int4_gemm(
    alpha: float,
    A: torch.Tensor,
    B: Int4Matrix,
    beta: float = 0.0,
    C: torch.Tensor | None = None,
    dtype: torch.dtype | None = None,
) -> torch.Tensor:
    """alpha * A @ B^T + beta * C for A (M, K) and an Int4Matrix B (N, K).

    The result (M, N) has `dtype` (float32, bfloat16 or float16), A's by default. K is at most 2^22 on a GPU, where
    a group's products are summed before its scale: values of A beyond 2^116 (8e34) may make infinite sums there.
    """
    return _product("int4_gemm", alpha, A, B, None, beta, C, dtype)


def int4_grouped_gemm(
    alpha: float,
    A: torch.Tensor,
    B: Int4Matrix,
    offsets: torch.Tensor,
    beta: float = 0.0,
    C: torch.Tensor | None = None,
    dtype: torch.dtype | None = None,
) -> torch.Tensor:
    """D[r] = alpha * A[r] @ B[g]^T + beta * C[r] for the rows r of group g: `grouped_gemm` with
    such weights, A (R, K), B (G, N, K). Rows of no group come out as beta * C[r]."""
    return _product("int4_grouped_gemm", alpha, A, B, offsets, beta, C, dtype, grouped=True)
