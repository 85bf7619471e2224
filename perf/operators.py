"""The work that the grouped and the microscaled 4-bit products are measured on.

Families ("op"):
* grouped: rows sorted by expert times their expert's matrix (an expert layer's forward product, and, with
  trans, its gradient to the activations), from one token's rows to a long training batch.
* rank_k: the gradient to the experts' matrices, a product over each expert's rows, added to what is there.
* step: forward and both gradients through autograd, as a training step runs them.
* quant: values to 4-bit floats with one power-of-two scale per 32, and back (what training with quantised
  weights does in each step, and what writing a quantised checkpoint does once).
* mx: activations quantised on the way times 4-bit weights: one projection of a served model.
* mxg: the same with one matrix per expert.

"active" experts have rows, the others none; "tail" rows at the end belong to no expert (buffers of a fixed
size, as captured graphs need them) and come out as zeros.
"""

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # one token sent to eight of 64 experts: latency, and eight weight matrices to read
        dict(name="grouped_token", op="grouped", dtype="bf16", rows=8, groups=64, active=8, k=2048, n=1024, trans=True,
             skew=0.0, tail=0),
        # a serving batch: a few rows to each expert, two experts idle, some rows of the buffer unused
        dict(name="grouped_serve", op="grouped", dtype="f16", rows=384, groups=32, active=30, k=1536, n=2048, trans=False,
             skew=1.0, tail=21),
        # fp32 with sizes that are multiples of nothing, as odd layer widths give them
        dict(name="grouped_odd_f32", op="grouped", dtype="f32", rows=1501, groups=7, active=6, k=515, n=771, trans=False,
             skew=0.7, tail=0),
        # a long training batch over 16 experts of unequal load
        dict(name="grouped_train", op="grouped", dtype="bf16", rows=32768, groups=16, active=16, k=4096, n=4096, trans=True,
             skew=0.5, tail=0),
        # a training step of one expert projection: forward, gradient to the activations, gradient to the weights
        dict(name="step_bf16", op="step", dtype="bf16", rows=8192, groups=8, active=8, k=2048, n=4096, trans=False, skew=0.5,
             tail=0),
        # weight gradients of many experts, accumulated into the gradient of earlier micro-batches
        dict(name="rank_k_accum", op="rank_k", dtype="f16", rows=12288, groups=24, active=23, m=2048, n=1024, skew=0.8, tail=0,
             beta=1.0, out="f32"),
        # a weight matrix to 4 bits and back
        dict(name="quant_weight", op="quant", dtype="bf16", rows=8192, k=8192, trans=False),
        # a small fp32 matrix stored the other way round, its blocks cut short at the end
        dict(name="quant_odd_trans", op="quant", dtype="f32", rows=129, k=2056, trans=True),
        # one token through a projection: reads the weights once
        dict(name="mx_token", op="mx", dtype="bf16", rows=1, n=8192, k=8192, out="bf16"),
        # a prompt through the same projection
        dict(name="mx_prompt", op="mx", dtype="bf16", rows=4096, n=8192, k=8192, out="bf16"),
        # a serving batch over 4-bit experts
        dict(name="mxg_serve", op="mxg", dtype="bf16", rows=256, groups=64, active=57, k=2048, n=1536, skew=1.0, tail=0,
             out="bf16"),
        # prompts over 4-bit experts, a width whose last block is cut short
        dict(name="mxg_prompt", op="mxg", dtype="f16", rows=8191, groups=16, active=15, k=2056, n=4104, skew=0.7, tail=0,
             out="f16"),
    ]  # fmt: skip


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """Even over the logarithm; half the time a multiple of 64, as layer widths are."""
    n = _log(rng, lo, hi)
    return max(64, n // 64 * 64) if rng.random() < 0.5 else n


def draw(rng):
    op = rng.choice(["grouped", "grouped", "rank_k", "step", "quant", "mx", "mxg", "mxg"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "quant":
        return dict(op=op, dtype=dtype, rows=_size(rng, 1, 8192), k=_size(rng, 32, 8192), trans=rng.random() < 0.4)
    if op == "mx":
        return dict(op=op, dtype=dtype, rows=_log(rng, 1, 4096), n=_size(rng, 128, 8192), k=_size(rng, 128, 8192),
                    out=dtype if rng.random() < 0.7 else "f32")  # fmt: skip
    groups = _log(rng, 1, 64)
    k, n = _size(rng, 64, 4096), _size(rng, 64, 4096)
    groups = max(1, min(groups, (1 << 27) // (k * n)))
    rows = _log(rng, 1, {"grouped": 16384, "rank_k": 16384, "step": 8192, "mxg": 16384}[op])
    if dtype == "f32":
        rows = min(rows, 4096)
    active = max(1, min(rows, groups - (rng.randrange(groups + 1) // 2 if rng.random() < 0.5 else 0)))
    tail = rng.randrange(1, 1 + max(1, rows // 8)) if op in ("grouped", "mxg") and rng.random() < 0.3 else 0
    tail = min(tail, rows - active)
    c = dict(op=op, dtype=dtype, rows=rows, groups=groups, active=active, skew=round(rng.uniform(0.0, 1.5), 2), tail=tail)
    if op == "rank_k":
        return dict(c, m=k, n=n, beta=rng.choice([0.0, 1.0]), out=dtype if rng.random() < 0.5 else "f32")
    if op == "mxg":
        return dict(c, k=k, n=n, out=dtype if rng.random() < 0.7 else "f32")
    return dict(c, k=k, n=n, trans=rng.random() < 0.5)


def _group_sizes(case, seed):
    """Rows of each expert: `active` of them have one or more, by unequal chances."""
    g = torch.Generator().manual_seed(seed + 7919)
    groups, active, rows = case["groups"], case["active"], case["rows"] - case["tail"]
    p = torch.softmax(case["skew"] * torch.randn(active, generator=g), 0)
    extra = torch.bincount(torch.multinomial(p, rows - active, replacement=True, generator=g), minlength=active) if (
        rows > active
    ) else torch.zeros(active, dtype=torch.int64)  # fmt: skip
    sizes = torch.zeros(groups, dtype=torch.int64)
    sizes[torch.randperm(groups, generator=g)[:active]] = extra + 1
    return sizes.tolist()


def _ranges(sizes):
    a = 0
    for g, s in enumerate(sizes):
        yield g, a, a + s
        a += s


def _activations(g, rows, k, dt):
    """Normal values with a few channels far above the rest, as hidden states have them."""
    x = torch.randn(rows, k, generator=g, device="cuda")
    x[:, :: max(1, k // 8)] *= 12.0
    return x.to(dt)


def _weights(g, dt, *shape, fan):
    w = torch.empty(*shape, device="cuda", dtype=dt)
    for part in w.unbind(0) if len(shape) == 3 else (w,):  # one matrix at a time: no fp32 copy of all of them
        part.copy_(torch.randn(part.shape, generator=g, device="cuda") * fan**-0.5)
    return w


# ── microscaled 4-bit values in plain torch ──────────────────────────────────

_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _pow2(e):
    """2^e in fp32 for whole e of -127 .. 127, from its bits (torch's ldexp rounds its power of two)."""
    return torch.where(e < -126, 1 << 22, (e + 127) << 23).to(torch.int32).view(torch.float32)


def _quantise(x):
    """Codes 0 .. 15 (sign above three bits of magnitude) and one scale exponent per 32 values of the last axis."""
    x = x.float()
    k = x.shape[-1]
    x = torch.nn.functional.pad(x, (0, -k % 32)).unflatten(-1, (-1, 32))
    top = x.abs().amax(-1)
    e = torch.where(top > 0, torch.frexp(top).exponent - 3, -127).clamp(-127, 127)
    y = x * _pow2(-e).unsqueeze(-1)
    a = y.abs()
    # halfway values go to the code whose last bit is zero
    code = (a > 0.25).to(torch.uint8)
    for up in (a >= 0.75, a > 1.25, a >= 1.75, a > 2.5, a >= 3.5, a > 5.0):
        code += up
    return code + 8 * (y < 0).to(torch.uint8), e


def _dequantise(q, k):
    codes, e = q
    table = torch.tensor(_VALUES + tuple(-v for v in _VALUES), device=codes.device)
    return (table[codes.int()] * _pow2(e).unsqueeze(-1)).flatten(-2)[..., :k]


# ── inputs ───────────────────────────────────────────────────────────────────


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    dt = DTYPES[case["dtype"]]
    op, rows = case["op"], case["rows"]
    if "groups" in case:
        sizes = _group_sizes(case, seed)
        s["sizes"] = sizes
        s["offsets"] = torch.tensor([0] + sizes).cumsum(0).to(torch.int32).cuda()
    if op == "quant":
        shape = (case["k"], rows) if case["trans"] else (rows, case["k"])
        s["X"] = _weights(g, dt, *shape, fan=case["k"])
        return s
    if op == "rank_k":
        s["A"] = _activations(g, rows, case["m"], dt)
        s["B"] = (torch.randn(rows, case["n"], generator=g, device="cuda") * 0.1).to(dt)
        s["C"] = _weights(g, DTYPES[case["out"]], case["groups"], case["m"], case["n"], fan=1.0) if case["beta"] else None
        return s
    k, n = case["k"], case["n"]
    s["A"] = _activations(g, rows, k, dt)
    if op in ("mx", "mxg"):
        W = _weights(g, dt, *((case["groups"],) if op == "mxg" else ()), n, k, fan=k)
        if own:
            import trnblas_amd as tb

            s["B"] = tb.mx_quantize(W)
        else:
            s["B"] = _quantise(W) if op == "mx" else [_quantise(w) for w in W]
        return s
    s["B"] = _weights(g, dt, case["groups"], *((n, k) if case["trans"] else (k, n)), fan=k)
    if op == "step":
        s["dD"] = (torch.randn(rows, n, generator=g, device="cuda") * 0.1).to(dt)
    return s


# ── one pass ─────────────────────────────────────────────────────────────────


def _run_own(s):
    import trnblas_amd as tb

    op = s["op"]
    if op == "grouped":
        return tb.grouped_gemm(1.0, s["A"], s["B"], s["offsets"], transB=s["trans"])
    if op == "rank_k":
        return tb.grouped_rank_k(1.0, s["A"], s["B"], s["offsets"], s["beta"], s["C"], dtype=DTYPES[s["out"]])
    if op == "step":
        A, B = s["A"].detach().requires_grad_(), s["B"].detach().requires_grad_()
        D = tb.grouped_gemm(1.0, A, B, s["offsets"], transB=s["trans"])
        return (D.detach(), *torch.autograd.grad(D, (A, B), s["dD"]))
    if op == "quant":
        return tb.mx_quantize(s["X"], trans=s["trans"]).dequantize(torch.bfloat16)
    if op == "mx":
        return tb.mx_gemm(1.0, s["A"], s["B"], dtype=DTYPES[s["out"]])
    return tb.mx_grouped_gemm(1.0, s["A"], s["B"], s["offsets"], dtype=DTYPES[s["out"]])


def _plain_grouped(A, B, sizes, trans):
    D = torch.zeros(A.shape[0], B.shape[1 if trans else 2], device=A.device)
    for g, a, b in _ranges(sizes):
        if b > a:
            D[a:b] = A[a:b].float() @ (B[g].mT if trans else B[g]).float()
    return D


def _plain_rank_k(A, B, sizes):
    return torch.stack([A[a:b].float().mT @ B[a:b].float() for _, a, b in _ranges(sizes)])


def run(s):
    if own:
        return _run_own(s)
    op, dt = s["op"], DTYPES[s.get("out", s["dtype"])]
    if op == "grouped":
        return _plain_grouped(s["A"], s["B"], s["sizes"], s["trans"]).to(dt)
    if op == "rank_k":
        D = _plain_rank_k(s["A"], s["B"], s["sizes"])
        return (D + s["beta"] * s["C"].float() if s["beta"] else D).to(dt)
    if op == "step":
        D = _plain_grouped(s["A"], s["B"], s["sizes"], s["trans"])
        dA = _plain_grouped(s["dD"], s["B"], s["sizes"], not s["trans"])
        dB = _plain_rank_k(s["dD"], s["A"], s["sizes"]) if s["trans"] else _plain_rank_k(s["A"], s["dD"], s["sizes"])
        return D.to(dt), dA.to(dt), dB.to(dt)
    if op == "quant":
        X = s["X"].mT.contiguous() if s["trans"] else s["X"]
        return _dequantise(_quantise(X), s["k"]).to(torch.bfloat16)
    A = _dequantise(_quantise(s["A"]), s["k"])
    if op == "mx":
        return (A @ _dequantise(s["B"], s["k"]).mT).to(dt)
    D = torch.zeros(s["rows"], s["n"], device=A.device)
    for g, a, b in _ranges(s["sizes"]):
        if b > a:
            D[a:b] = A[a:b] @ _dequantise(s["B"][g], s["k"]).mT
    return D.to(dt)


def work(case):
    op, rows, e = case["op"], case["rows"], BYTES[case["dtype"]]
    if op == "quant":
        # values in, 4-bit values and scales out and in again, 16-bit values out
        n = rows * case["k"]
        return {"bytes": n * (e + 2) + 2 * n * 17 / 32, "flops": 2.0 * n}
    if op == "rank_k":
        o = BYTES[case["out"]] * case["groups"] * case["m"] * case["n"]
        return {"bytes": e * rows * (case["m"] + case["n"]) + o * (2 if case["beta"] else 1),
                "flops": 2.0 * rows * case["m"] * case["n"]}  # fmt: skip
    k, n = case["k"], case["n"]
    covered = rows - case.get("tail", 0)
    if op in ("mx", "mxg"):
        weights = case.get("active", 1) * n * k * 17 / 32
        return {"bytes": e * covered * k + weights + BYTES[case["out"]] * rows * n, "flops": 2.0 * covered * k * n}
    one = {"bytes": e * (covered * k + case["active"] * k * n + rows * n), "flops": 2.0 * covered * k * n}
    if op == "grouped":
        return one
    # the step reads A, B and dD and writes D, dA and dB (a matrix for every expert)
    return {"bytes": e * (2 * rows * (k + n) + (case["active"] + case["groups"]) * k * n), "flops": 3 * one["flops"]}


# ── the definitions in 64 bits ───────────────────────────────────────────────


def _mx64(x):
    """The values that x becomes: x / 2^e to the nearest multiple of the spacing at its size (ties to even), at most 6."""
    x = x.double()
    k = x.shape[-1]
    pad = -(-k // 32) * 32 - k
    b = torch.cat([x, x.new_zeros(*x.shape[:-1], pad)], -1).reshape(*x.shape[:-1], -1, 32)
    top = b.abs().amax(-1, keepdim=True)

    def power(n):  # 2^n from its bits
        return ((n.long() + 1023) << 52).view(torch.float64)

    e = torch.where(top > 0, torch.frexp(top).exponent - 3, -127).clamp(-127, 127)
    v = b / power(e)
    step = power(torch.frexp(v.abs().clamp(1.0, 6.0)).exponent - 2)
    v = (torch.round(v / step) * step).clamp(-6.0, 6.0)
    return (v * power(e)).reshape(*x.shape[:-1], k + pad)[..., :k]


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    op = case["op"]
    if op == "quant":
        return _mx64(s["X"].mT if case["trans"] else s["X"])
    if op in ("mx", "mxg"):
        A = _mx64(s["A"])
        if op == "mx":
            return A @ _dequantise(s["B"], case["k"]).double().mT.contiguous()
        D = torch.zeros(case["rows"], case["n"], dtype=torch.float64, device="cuda")
        for g, a, b in _ranges(s["sizes"]):
            if b > a:
                torch.matmul(A[a:b], _dequantise(s["B"][g], case["k"]).double().mT.contiguous(), out=D[a:b])
        return D
    A = s["A"].double()
    outs = []
    if op in ("grouped", "step"):
        D = torch.zeros(case["rows"], case["n"], dtype=torch.float64, device="cuda")
        dA = torch.zeros(case["rows"], case["k"], dtype=torch.float64, device="cuda")
        for g, a, b in _ranges(s["sizes"]):
            W = (s["B"][g].T if case["trans"] else s["B"][g]).double().contiguous()
            D[a:b] = A[a:b] @ W
            if op == "step":
                dA[a:b] = s["dD"][a:b].double() @ W.T.contiguous()
        if op == "grouped":
            return D
        outs = [D, dA]
    other = (s["dD"] if op == "step" else s["B"]).double()
    left, right = (other, A) if case.get("trans") else (A, other)
    dB = torch.zeros(case["groups"], left.shape[1], right.shape[1], dtype=torch.float64, device="cuda")
    for g, a, b in _ranges(s["sizes"]):
        dB[g] = left[a:b].T.contiguous() @ right[a:b]
        if op == "rank_k" and case["beta"]:
            dB[g] += case["beta"] * s["C"][g].double()
    return (*outs, dB) if op == "step" else dB
