"""The grouped products in 64 bits, group by group, and the error that fp32 sums may make in them."""

import torch


def split(rows, sizes, lead=0):
    """Offsets of groups of `sizes` rows after `lead` rows of no group."""
    o = [lead]
    for s in sizes:
        o.append(o[-1] + s)
    assert o[-1] <= rows
    return torch.tensor(o, dtype=torch.int32)


# (rows, sizes of the groups, rows before the first): one row, empty groups, tiles that end inside, rows of no group
GROUPS = {
    "one": (1, [1], 0),
    "one_of_many": (1, [0] * 37 + [1] + [0] * 26, 0),
    "token": (6, [0, 1, 0, 2, 0, 0, 1, 1, 0, 1], 0),
    "gaps": (77, [0, 9, 0, 40, 3], 11),
    "all_gap": (19, [0, 0, 0], 7),
    "small": (150, [17, 33, 1, 64, 35], 0),
    "many": (300, [(3 * i) % 5 for i in range(140)], 2),
    "uneven": (700, [513, 0, 2, 185], 0),
    "single": (400, [400], 0),
}


def rows_of(offsets, rows):
    o = [min(max(int(x), 0), rows) for x in offsets.tolist()]
    return [(g, a, b) for g, (a, b) in enumerate(zip(o, o[1:])) if b > a]


def grouped_gemm(alpha, A, B, offsets, beta=0.0, C=None, transB=False):
    """(D, |alpha| |A| |B| + |beta C|) in float64."""
    A, B = A.double(), (B.mT if transB else B).double()
    D = torch.zeros(A.shape[0], B.shape[2], dtype=torch.float64)
    den = torch.zeros_like(D)
    for g, a, b in rows_of(offsets, A.shape[0]):
        D[a:b] = alpha * (A[a:b] @ B[g])
        den[a:b] = abs(alpha) * (A[a:b].abs() @ B[g].abs())
    if beta != 0.0:
        D, den = D + beta * C.double(), den + abs(beta) * C.double().abs()
    return D, den


def grouped_rank_k(alpha, A, B, offsets, beta=0.0, C=None):
    A, B = A.double(), B.double()
    D = torch.zeros(offsets.shape[0] - 1, A.shape[1], B.shape[1], dtype=torch.float64)
    den = torch.zeros_like(D)
    for g, a, b in rows_of(offsets, A.shape[0]):
        D[g] = alpha * (A[a:b].mT @ B[a:b])
        den[g] = abs(alpha) * (A[a:b].mT.abs() @ B[a:b].abs())
    if beta != 0.0:
        D, den = D + beta * C.double(), den + abs(beta) * C.double().abs()
    return D, den


def excess(D, ref, den, k):
    """Largest |D - ref| over what the arithmetic allows (<= 1 passes): k products summed in fp32 in any order, each
    addition off by at most one unit in the last place (2^-23, truncating adders included) of a partial sum
    that |A||B| bounds, two more for alpha and beta; then one rounding to D's type."""
    u = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}[D.dtype]
    tiny = {torch.float32: 2.0**-149, torch.bfloat16: 2.0**-133, torch.float16: 2.0**-25}[D.dtype]
    bound = (k + 2) * 2.0**-23 * den
    bound = bound + u * (ref.abs() + bound) + tiny
    return float(((D.detach().double().cpu() - ref).abs() / bound).max()) if D.numel() else 0.0


def plan(op, dtype, transB, groups, rows, M, N, K):
    from trnblas_amd.hip import _lib

    return _lib.load().trnblas_hip_grouped_plan(op, _lib.DTYPE_CODES[dtype], transB, groups, rows, M, N, K).decode()


def uneven(groups, rows, seed):
    """Offsets of `groups` uneven groups, one of them empty where there are several, some rows of no group."""
    g = torch.Generator().manual_seed(seed)
    w = torch.rand(groups, generator=g) + 0.2
    if groups > 2:
        w[1] = 0
    sizes = (w / w.sum() * (rows - 3)).long()
    return split(rows, sizes.tolist(), 2)


def rows_plan(op, dtype, transB, groups, rows, N, K):
    """(row blocks, waves along K, A quantised inside) of rows_kernel; zeros for another kernel."""
    import ctypes

    from trnblas_amd.hip import _lib

    out = (ctypes.c_int32 * 3)()
    _lib.call("trnblas_hip_grouped_rows_plan", op, _lib.DTYPE_CODES[dtype], transB, groups, rows, N, K, out)
    return tuple(out)
