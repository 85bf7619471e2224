"""Gated projections in 64 bits, and the error that fp32 arithmetic may make in them."""

import math

import torch

from .grouped import rows_of

ACTS = ("silu", "gelu", "gelu_tanh", "relu", "sigmoid")
EPS = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TINY = {torch.float32: 2.0**-126, torch.bfloat16: 2.0**-126, torch.float16: 2.0**-24}


def gate(act, x):
    """(act(x), act'(x)) in float64."""
    if act == "silu":
        s = torch.sigmoid(x)
        return x * s, s + x * s * torch.sigmoid(-x)
    if act == "gelu":
        p = 0.5 * torch.erfc(-x / math.sqrt(2.0))
        return x * p, p + x * torch.exp(-0.5 * x * x) / math.sqrt(2.0 * math.pi)
    if act == "gelu_tanh":
        c = 2.0 * math.sqrt(2.0 / math.pi)
        u = c * (x + 0.044715 * x**3)
        s = torch.sigmoid(u)
        return x * s, s + x * s * torch.sigmoid(-u) * c * (1.0 + 3.0 * 0.044715 * x * x)
    if act == "relu":
        return x.clamp_min(0.0), (x > 0).double()
    s = torch.sigmoid(x)
    return s, s * torch.sigmoid(-x)


# Largest |act'| and |act''|: silu 1.0998 and 0.5; gelu 1.129 and 0.798; gelu_tanh 1.13 and 0.8; relu 1 and none (its
# kink: a slope of 1 there bounds the change of act, that of act' is not bounded and not asked for); sigmoid 0.25 and 0.0963.
LIP = {"silu": 1.1, "gelu": 1.13, "gelu_tanh": 1.14, "relu": 1.0, "sigmoid": 0.25}
BEND = {"silu": 0.5, "gelu": 0.8, "gelu_tanh": 0.82, "relu": 0.0, "sigmoid": 0.1}
# fp32 evaluation of act and act': a handful of operations, each within two units of 2^-23 of values of the size of 1 + |x|
# (exp of -x is off by |x| 2^-24 from its argument's rounding besides its own).
FN = 24 * 2.0**-23


def products(A, B, offsets, transB=False):
    """(P, |A| |B|) in float64, A (R, K), B (G, K, 2 N) ((G, 2 N, K) with transB)."""
    A, B = A.double(), (B.mT if transB else B).double()
    P = torch.zeros(A.shape[0], B.shape[2], dtype=torch.float64, device=A.device)
    den = torch.zeros_like(P)
    for g, a, b in rows_of(offsets, A.shape[0]):
        W = B[g].contiguous()
        P[a:b], den[a:b] = A[a:b] @ W, A[a:b].abs() @ W.abs()
    return P, den


def forward(act, P, den, k, dtype):
    """(H, bound on its error in `dtype`): the products are k fp32 sums (each addition within 2^-23 of |A||B|)."""
    (G, U), (dG, dU) = P.chunk(2, -1), ((k + 2) * 2.0**-23 * den).chunk(2, -1)
    y, _ = gate(act, G)
    H = y * U
    ey = LIP[act] * dG + FN * (1.0 + G.abs())
    err = ey * (U.abs() + dU) + y.abs() * dU + 2.0**-23 * H.abs()
    return H, err + EPS[dtype] * (H.abs() + err) + TINY[dtype]


def backward(act, P, dH):
    """dP in float64."""
    G, U = P.chunk(2, -1)
    y, slope = gate(act, G)
    return torch.cat([dH.double() * U * slope, dH.double() * y], -1)


def gradient_bounds(act, P, den, dH, k, dtype):
    """Bound on the error of the kernels' dP in `dtype`, from P rounded to it (errors of P: its sums' and one rounding)."""
    (G, U), e = P.chunk(2, -1), (k + 2) * 2.0**-23 * den
    e = e + EPS[dtype] * (P.abs() + e) + TINY[dtype]
    eG, eU = e.chunk(2, -1)
    y, slope = gate(act, G)
    d = dH.double().abs()
    es, ey = BEND[act] * eG + FN * (1.0 + G.abs()), LIP[act] * eG + FN * (1.0 + G.abs())
    err = torch.cat([d * (es * (U.abs() + eU) + slope.abs() * eU), d * ey], -1)
    dP = backward(act, P, dH).abs()
    err = err + 2.0**-22 * (dP + err)
    return err + EPS[dtype] * (dP + err) + TINY[dtype]


def ratio(X, ref, bound):
    """Largest |X - ref| over the bound (<= 1 passes)."""
    return float(((X.detach().double().to(ref.device) - ref).abs() / bound).max()) if X.numel() else 0.0
