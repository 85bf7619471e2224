"""4-bit integer weights by their definition: quotients and scales rounded to fp32 where it says so, the rest in 64 bits."""

import torch

from . import grouped


def quantize(X, group, zeros, scale_dtype):
    """(values float64, q, scales, z) of X (..., K); scales float64 (..., groups), NaN where a group is one; z 8 without zeros."""
    K = X.shape[-1]
    x = X.double()
    x = torch.cat([x, x.new_zeros(*x.shape[:-1], -K % group)], -1).reshape(*x.shape[:-1], -1, group)
    finite = x.isfinite().all(-1)
    x = torch.where(finite.unsqueeze(-1), x, 0.0)
    lo, hi = x.amin(-1).clamp_max(0.0), x.amax(-1).clamp_min(0.0)
    # a difference or quotient of fp32 numbers rounded from 64 bits is the rounded one
    s = ((hi - lo).float().double() / 15).float() if zeros else (torch.maximum(hi, -lo) / 7).float()
    s = s.to(scale_dtype).double()
    good = finite & s.isfinite()
    live = good & (s > 0)
    by = torch.where(live, s, 1.0)
    v = torch.round((x / by.unsqueeze(-1)).float().double())
    if zeros:
        z = torch.where(live, torch.round((-lo / by).float().double()).clamp(0, 15), 0.0)
        q = torch.where(live.unsqueeze(-1), (v + z.unsqueeze(-1)).clamp(0, 15), 0.0)
    else:
        z = torch.full_like(s, 8.0)
        q = torch.where(live.unsqueeze(-1), v.clamp(-8, 7) + 8, 8.0)
    s = torch.where(good, s, torch.nan)
    w = ((q - z.unsqueeze(-1)) * s.unsqueeze(-1)).flatten(-2)[..., :K]
    return w, q.flatten(-2)[..., :K], s, z


def product(alpha, A, W, offsets=None, beta=0.0, C=None):
    """(D, |A| |W|) of values A (R, K), W (N, K) or (G, N, K)."""
    if offsets is None:
        return grouped.grouped_gemm(alpha, A, W[None], torch.tensor([0, A.shape[0]]), beta, C, True)
    return grouped.grouped_gemm(alpha, A, W, offsets, beta, C, True)


def wide(g, *shape, dtype=torch.float32):
    """Values over many powers of two, whole and halfway steps of a scale among them."""
    x = torch.randn(*shape, generator=g) * torch.exp2(torch.randint(-12, 13, (*shape[:-1], 1), generator=g).float())
    half = torch.randint(-14, 15, shape, generator=g).float() / 2
    half[..., :1] = 7.0  # a scale of one for the first group
    return torch.where(torch.rand(*shape[:-1], 1, generator=g) < 0.4, half, x).to(dtype)


def random_matrix(g, *shape, group, zeros, scale_dtype, device="cpu", z_max=15):
    """An Int4Matrix of random codes, scales and zero points, and its values in float64."""
    import trnblas_amd as tb

    *lead, R, K = shape
    n = -(-K // group)
    codes = torch.randint(0, 256, (*lead, R, -(-K // 2)), generator=g, device=device).to(torch.uint8)
    scales = ((torch.rand(*lead, R, n, generator=g, device=device) + 0.25) * K**-0.5 / 4).to(scale_dtype)
    scales *= torch.where(torch.rand(scales.shape, generator=g, device=device) < 0.1, -1.0, 1.0).to(scale_dtype)
    z = torch.randint(0, z_max + 1, (*lead, R, n), generator=g, device=device).to(torch.uint8) if zeros else None
    q = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)[..., :K].double()
    spread = lambda t: t.double().repeat_interleave(group, -1)[..., :K]
    W = (q - (8.0 if z is None else spread(z))) * spread(scales)
    return tb.Int4Matrix.from_parts(codes, scales, K, group, z), W
