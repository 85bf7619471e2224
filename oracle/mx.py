"""Microscaled 4-bit floats by their definition in 64 bits: nearest of the eight magnitudes, ties to the even code."""

import torch

VALUES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def quantize(X):
    """(values, codes 0 .. 15 without the sign of zeros, scale bytes) of X (..., K), float64 / int64, blocks padded with zeros."""
    x = X.double()
    K = x.shape[-1]
    x = torch.cat([x, x.new_zeros(*x.shape[:-1], -K % 32)], -1).reshape(*x.shape[:-1], -1, 32)
    bad = ~x.isfinite().all(-1)
    top = x.abs().nan_to_num(0.0, 0.0, 0.0).amax(-1)
    e = torch.where(top > 0, torch.frexp(top).exponent.long() - 3, -127).clamp_min(-127)
    y = torch.ldexp(x, -e.unsqueeze(-1).double()).nan_to_num(0.0, 0.0, 0.0)
    dist = (y.abs().unsqueeze(-1) - VALUES).abs()
    best = dist == dist.amin(-1, keepdim=True)  # one code, or two neighbours at the same distance
    even = best & (torch.arange(8) % 2 == 0)
    code = torch.where(best.sum(-1) > 1, even.long().argmax(-1), best.long().argmax(-1))
    values = torch.copysign(VALUES[code], y) * torch.exp2(e.double()).unsqueeze(-1)
    values = torch.where(bad.unsqueeze(-1), torch.nan, values)
    byte = torch.where(bad, 255, e + 127)
    return values.flatten(-2)[..., :K], code.flatten(-2), byte


def product(alpha, A, B, offsets=None, beta=0.0, C=None):
    """(D, |A| |B|) of quantised values A (R, K), B (N, K) or (G, N, K)."""
    if offsets is None:
        A, B = A.double(), B.double()
        D, den = alpha * (A @ B.mT), abs(alpha) * (A.abs() @ B.abs().mT)
        if beta != 0.0:
            D, den = D + beta * C.double(), den + abs(beta) * C.double().abs()
        return D, den
    from . import grouped

    return grouped.grouped_gemm(alpha, A, B, offsets, beta, C, True)


def wide(g, *shape, dtype=torch.float32):
    """Values over many powers of two, halfway cases among them."""
    x = torch.randn(*shape, generator=g) * torch.exp2(torch.randint(-12, 13, (*shape[:-1], 1), generator=g).float())
    half = torch.randint(-28, 29, shape, generator=g).float() / 4
    return torch.where(torch.rand(shape, generator=g) < 0.3, half, x).to(dtype)
