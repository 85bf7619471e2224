"""The work that gated feed-forward projections and products of 4-bit integer weights are measured on.

Families ("op"):
* gated: H = act(A G) * (A U), the first half of a gated feed-forward block: both projections (G and U side by side in one
  matrix of 2 n columns), the activation and the product. Forward only, as a served model or an evaluation runs it.
* step: the same in a training step: H and the gradients of the rows and of the weights, through autograd.
* int4: rows times 4-bit integer weights with a scale (and a zero point, where "zeros" says so) for each group of "group"
  values along k: one projection of a served model.
* int4_gated: the gated projections of such weights.
* quant: values to such weights and back.

"groups" > 0: rows sorted by expert, each expert with weights of its own; "active" experts have rows, the others none, and
"tail" rows at the end belong to no expert (buffers of a fixed size) and come out as zeros. "trans": weights stored
(columns, k), as linear layers keep them, else (k, columns).
"""

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # one token sent to eight of 64 experts: latency, and eight pairs of weight matrices to read
        dict(name="gated_token", op="gated", dtype="bf16", act="silu", rows=8, groups=64, active=8, k=2048, n=1024, trans=True,
             skew=0.0, tail=0),
        # fp32 with sizes that are multiples of nothing, as odd layer widths give them
        dict(name="gated_odd_f32", op="gated", dtype="f32", act="gelu", rows=301, groups=0, k=515, n=771, trans=False),
        # a long prompt through a dense block's gate and up projections
        dict(name="gated_prompt", op="gated", dtype="f16", act="gelu_tanh", rows=4096, groups=0, k=4096, n=8192, trans=True),
        # a training step of a dense block's first half
        dict(name="step_bf16", op="step", dtype="bf16", act="silu", rows=8192, groups=0, k=2048, n=4096, trans=True),
        # a training step over experts of unequal load, one of them idle, weights stored the other way round
        dict(name="step_experts", op="step", dtype="f16", act="gelu", rows=4093, groups=8, active=7, k=1032, n=2048, trans=False,
             skew=0.5, tail=0),
        # one token through a projection: reads the weights once
        dict(name="int4_token", op="int4", dtype="bf16", rows=1, groups=0, k=8192, n=8192, group=128, zeros=False, scale="bf16",
             out="bf16"),
        # a decoding batch over weights with zero points, as post-training quantisation gives them
        dict(name="int4_batch", op="int4", dtype="f16", rows=23, groups=0, k=4096, n=8192, group=64, zeros=True, scale="f16",
             out="f16"),
        # a prompt through the same kind of projection
        dict(name="int4_prompt", op="int4", dtype="bf16", rows=2048, groups=0, k=4096, n=8192, group=128, zeros=False,
             scale="bf16", out="bf16"),
        # a few tokens through the gated projections of a served block
        dict(name="int4_gated_token", op="int4_gated", dtype="bf16", act="silu", rows=4, groups=0, k=4096, n=8192, group=128,
             zeros=True, scale="bf16", out="bf16"),
        # a decoding batch over 4-bit experts, groups of 32, some rows of the buffer unused
        dict(name="int4_gated_experts", op="int4_gated", dtype="f16", act="silu", rows=160, groups=32, active=29, k=2048, n=1032,
             group=32, zeros=False, scale="f16", out="f16", skew=0.7, tail=9),
        # a weight matrix to 4 bits and back
        dict(name="quant_weight", op="quant", dtype="bf16", rows=8192, k=8192, group=128, zeros=False, scale="bf16", trans=False),
        # a small fp32 matrix stored the other way round, its groups cut short at the end, with zero points
        dict(name="quant_odd_trans", op="quant", dtype="f32", rows=129, k=2056, group=64, zeros=True, scale="f16", trans=True),
    ]  # fmt: skip


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """Even over the logarithm; half the time a multiple of 64, as layer widths are."""
    n = _log(rng, lo, hi)
    return max(64, n // 64 * 64) if rng.random() < 0.5 else n


def draw(rng):
    op = rng.choice(["gated", "gated", "step", "step", "int4", "int4", "int4_gated", "quant"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    fine = dict(group=rng.choice([32, 64, 128]), zeros=rng.random() < 0.5, scale=rng.choice(["bf16", "f16"]))
    if op == "quant":
        return dict(op=op, dtype=dtype, rows=_size(rng, 64, 8192), k=_size(rng, 64, 8192), trans=rng.random() < 0.4, **fine)
    groups = _log(rng, 1, 64) if rng.random() < 0.5 else 0
    k, n = _size(rng, 64, 8192), _size(rng, 64, 8192)
    groups = min(groups, (1 << 26) // (k * n))
    # as much work as the listed cases have at most
    most = {"gated": 1 << 37, "step": 1 << 36, "int4": 1 << 36, "int4_gated": 1 << 35}[op] >> (3 if dtype == "f32" else 0)
    rows = max(1, min(_log(rng, 1, 8192), most // (k * n)))
    c = dict(op=op, dtype=dtype, rows=rows, groups=groups, k=k, n=n)
    if op in ("gated", "step"):
        c["trans"] = rng.random() < 0.6
    if op != "int4":
        c["act"] = rng.choice(["silu", "silu", "gelu", "gelu_tanh"])
    if op in ("int4", "int4_gated"):
        c.update(fine, out=dtype if rng.random() < 0.7 else "f32")
    if groups:
        active = max(1, min(rows, groups - (rng.randrange(groups + 1) // 2 if rng.random() < 0.5 else 0)))
        tail = rng.randrange(1, 1 + max(1, rows // 8)) if op != "step" and rng.random() < 0.3 else 0
        c.update(active=active, skew=round(rng.uniform(0.0, 1.0), 2), tail=min(tail, rows - active))
    return c


def _group_sizes(case, seed):
    """Rows of each expert: `active` of them have one or more, by unequal chances."""
    g = torch.Generator().manual_seed(seed + 7919)
    groups, active, rows = case["groups"], case["active"], case["rows"] - case["tail"]
    p = torch.softmax(case["skew"] * torch.randn(active, generator=g), 0)
    extra = torch.zeros(active, dtype=torch.int64)
    if rows > active:
        extra = torch.bincount(torch.multinomial(p, rows - active, replacement=True, generator=g), minlength=active)
    sizes = torch.zeros(groups, dtype=torch.int64)
    sizes[torch.randperm(groups, generator=g)[:active]] = extra + 1
    return sizes


def _activations(g, rows, k, dt):
    """Normal values with a few channels far above the rest, as hidden states have them."""
    x = torch.randn(rows, k, generator=g, device="cuda")
    x[:, :: max(1, k // 8)] *= 4.0
    return x.to(dt)


def _weights(g, dt, *shape, fan):
    w = torch.empty(*shape, device="cuda", dtype=dt)
    for part in w.unbind(0) if len(shape) == 3 else (w,):  # one matrix at a time: no fp32 copy of all of them
        part.copy_(torch.randn(part.shape, generator=g, device="cuda") * fan**-0.5)
    return w


def _stored_int4(g, case, *lead, n):
    """Weights as a checkpoint holds them: codes two to a byte (the even one low), scales and zero points of groups along k."""
    k, parts = case["k"], -(-case["k"] // case["group"])
    codes = torch.randint(0, 16, (*lead, n, -(-k // 2) * 2), generator=g, device="cuda", dtype=torch.uint8)
    codes[..., k:] = 0
    scales = (torch.rand(*lead, n, parts, generator=g, device="cuda") + 0.5) * (k**-0.5 / 4)
    zeros = torch.randint(5, 12, (*lead, n, parts), generator=g, device="cuda", dtype=torch.uint8) if case["zeros"] else None
    return codes[..., ::2] | codes[..., 1::2] << 4, scales.to(DTYPES[case["scale"]]), zeros


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    dt, op = DTYPES[case["dtype"]], case["op"]
    if op == "quant":
        shape = (case["k"], case["rows"]) if case["trans"] else (case["rows"], case["k"])
        s["X"] = _weights(g, dt, *shape, fan=case["k"])
        return s
    rows, k, n, lead = case["rows"], case["k"], case["n"], ()
    if case["groups"]:
        lead = (case["groups"],)
        sizes = _group_sizes(case, seed)
        s["sizes"] = sizes.tolist()
        s["offsets"] = torch.cat([torch.zeros(1, dtype=torch.int64), sizes.cumsum(0)]).to(torch.int32).cuda()
    s["A"] = _activations(g, rows, k, dt)
    if op in ("int4", "int4_gated"):
        s["codes"], s["scales"], s["zeros"] = _stored_int4(g, case, *lead, n=2 * n if op == "int4_gated" else n)
        if own:  # laid out once, when a program loads its weights
            import trnblas_amd as tb

            s["B"] = tb.Int4Matrix.from_parts(s["codes"], s["scales"], k, case["group"], s["zeros"])
        return s
    s["B"] = _weights(g, dt, *lead, *((2 * n, k) if case["trans"] else (k, 2 * n)), fan=k)
    if op == "step":
        s["dH"] = (torch.randn(rows, n, generator=g, device="cuda") * 0.1).to(dt)
    return s


# ── one pass ─────────────────────────────────────────────────────────────────


def _run_own(s):
    import trnblas_amd as tb

    op = s["op"]
    if op == "quant":
        Q = tb.int4_quantize(s["X"], s["group"], zeros=s["zeros"], trans=s["trans"], scale_dtype=DTYPES[s["scale"]])
        return tb.int4_dequantize(Q, DTYPES[s["dtype"]])
    if op == "int4":
        out = DTYPES[s["out"]]
        if s["groups"]:
            return tb.int4_grouped_gemm(1.0, s["A"], s["B"], s["offsets"], dtype=out)
        return tb.int4_gemm(1.0, s["A"], s["B"], dtype=out)
    if op == "int4_gated":
        out = DTYPES[s["out"]]
        if s["groups"]:
            return tb.grouped_gated_gemm(s["A"], s["B"], s["offsets"], s["act"], dtype=out)
        return tb.gated_gemm(s["A"], s["B"], s["act"], dtype=out)
    A, B = s["A"], s["B"]
    if op == "step":
        A, B = A.detach().requires_grad_(), B.detach().requires_grad_()
    if s["groups"]:
        H = tb.grouped_gated_gemm(A, B, s["offsets"], s["act"], transB=s["trans"])
    else:
        H = tb.gated_gemm(A, B, s["act"], transB=s["trans"])
    return H if op == "gated" else (H.detach(), *torch.autograd.grad(H, (A, B), s["dH"]))


def _dequantise(codes, scales, zeros, k, group):
    """(q - z) s in fp32 for packed codes (..., n, k / 2)."""
    q = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)[..., :k].float()
    z = 8.0 if zeros is None else zeros.float().repeat_interleave(group, -1)[..., :k]
    return (q - z) * scales.float().repeat_interleave(group, -1)[..., :k]


def _by_expert(s):
    """Experts that have rows; of each of their rows the expert's place and the row's place in it; the longest."""
    sizes = torch.tensor(s["sizes"])
    active = sizes.nonzero()[:, 0]
    mine = sizes[active]
    place = torch.repeat_interleave(torch.arange(len(active)), mine)
    at = torch.arange(int(mine.sum())) - (mine.cumsum(0) - mine)[place]
    return active.cuda(), place.cuda(), at.cuda(), int(mine.max())


def _spread(X, where):
    """Rows sorted by expert as (experts, longest, columns), zeros behind the shorter ones."""
    active, place, at, longest = where
    P = X.new_zeros(len(active), longest, X.shape[1])
    P[place, at] = X[: len(place)]
    return P


def _gather(P, where, rows):
    _, place, at, _ = where
    X = P.new_zeros(rows, P.shape[2])
    X[: len(place)] = P[place, at]
    return X


def _act(x, name):
    if name == "silu":
        return x / (1.0 + torch.exp(-x))
    if name == "gelu":
        return 0.5 * x * (1.0 + torch.erf(x * 0.5**0.5))
    return 0.5 * x * (1.0 + torch.tanh((2.0 / math.pi) ** 0.5 * (x + 0.044715 * x * x * x)))


def _act_slope(x, name):
    if name == "silu":
        y = 1.0 / (1.0 + torch.exp(-x))
        return y * (1.0 + x * (1.0 - y))
    if name == "gelu":
        return 0.5 * (1.0 + torch.erf(x * 0.5**0.5)) + x * torch.exp(-0.5 * x * x) * (2.0 * math.pi) ** -0.5
    c = (2.0 / math.pi) ** 0.5
    t = torch.tanh(c * (x + 0.044715 * x * x * x))
    return 0.5 * (1.0 + t) + 0.5 * x * (1.0 - t * t) * c * (1.0 + 3.0 * 0.044715 * x * x)


def _quantise(X, group, zeros, scale):
    """Values to codes and back: whole steps of the group's scale, at most 4 bits of them, in fp32."""
    rows, k = X.shape
    x = torch.nn.functional.pad(X.float(), (0, -k % group)).reshape(rows, -1, group)
    if zeros:
        lo, hi = x.amin(-1, keepdim=True).clamp_max(0.0), x.amax(-1, keepdim=True).clamp_min(0.0)
        step = ((hi - lo) / torch.full_like(hi, 15.0)).to(scale).float()
        some = torch.where(step > 0, step, 1.0)
        z = torch.round(-lo / some).clamp(0, 15)
        q = (torch.round(x / some) + z).clamp(0, 15) - z
    else:
        top = x.abs().amax(-1, keepdim=True)
        step = (top / torch.full_like(top, 7.0)).to(scale).float()
        q = torch.round(x / torch.where(step > 0, step, 1.0)).clamp(-8, 7)
    return (torch.where(step > 0, q, 0.0) * step).reshape(rows, -1)[:, :k]


def run(s):
    if own:
        return _run_own(s)
    op, dt = s["op"], DTYPES[s.get("out", s["dtype"])]
    if op == "quant":
        return _quantise(s["X"].mT if s["trans"] else s["X"], s["group"], s["zeros"], DTYPES[s["scale"]]).to(dt)
    A, rows, n = s["A"].float(), s["rows"], s["n"]
    where = _by_expert(s) if s["groups"] else None
    if where:
        A = _spread(A, where)
    pick = (lambda t: t if t is None or not where else t[where[0]])  # noqa: E731
    if op in ("int4", "int4_gated"):
        W = _dequantise(pick(s["codes"]), pick(s["scales"]), pick(s["zeros"]), s["k"], s["group"]).mT
    else:
        W = pick(s["B"]).float()
        W = W.mT if s["trans"] else W
    P = A @ W
    if op == "int4":
        return (_gather(P, where, rows) if where else P).to(dt)
    G, U = P[..., :n], P[..., n:]
    H = _act(G, s["act"]) * U
    if op != "step":
        return (_gather(H, where, rows) if where else H).to(dt)
    dH = s["dH"].float()
    if where:
        dH = _spread(dH, where)
    dP = torch.cat([dH * U * _act_slope(G, s["act"]), dH * _act(G, s["act"])], -1)
    dA = dP @ W.mT
    dB = dP.mT @ A if s["trans"] else A.mT @ dP
    if not where:
        return H.to(dt), dA.to(dt), dB.to(dt)
    all_dB = torch.zeros(s["B"].shape, dtype=dt, device=A.device)
    all_dB[where[0]] = dB.to(dt)
    return _gather(H, where, rows).to(dt), _gather(dA, where, rows).to(dt), all_dB


def work(case):
    op, rows, k, e = case["op"], case["rows"], case["k"], BYTES[case["dtype"]]
    if op == "quant":
        # values in; codes, scales and zero points out and in again; values out
        cells = rows * k
        held = cells / 2 + rows * -(-k // case["group"]) * (2.5 if case["zeros"] else 2)
        return {"bytes": 2 * e * cells + 2 * held, "flops": 2.0 * cells}
    n, covered = case["n"], rows - case.get("tail", 0)
    active = case["active"] if case["groups"] else 1
    columns = n if op == "int4" else 2 * n
    flops = 2.0 * covered * k * columns
    if op in ("int4", "int4_gated"):
        weights = columns * (k / 2 + -(-k // case["group"]) * (2.5 if case["zeros"] else 2))
        return {"bytes": e * covered * k + active * weights + BYTES[case["out"]] * rows * n, "flops": flops}
    if op == "gated":
        return {"bytes": e * (covered * k + active * k * columns + rows * n), "flops": flops}
    # a step reads A, B and dH and writes H, dA and dB (a matrix for every expert)
    return {"bytes": e * (2 * rows * k + 2 * rows * n + (active + max(1, case["groups"])) * k * columns), "flops": 3 * flops}


# ── the definitions in 64 bits ───────────────────────────────────────────────


def _exact_values(codes, scales, zeros, k, group):
    n = codes.shape[0]
    q = torch.empty(n, 2 * codes.shape[1], dtype=torch.float64, device=codes.device)
    q[:, 0::2], q[:, 1::2] = (codes % 16).double(), (codes // 16).double()
    of = torch.arange(k, device=codes.device) // group
    return (q[:, :k] - (8.0 if zeros is None else zeros.double()[:, of])) * scales.double()[:, of]


def _exact_rounded(X, group, zeros, scale):
    """The values that X becomes. Scales and quotients are by definition rounded to fp32, scales then to their type."""
    rows, k = X.shape
    out = torch.empty(rows, k, dtype=torch.float64, device=X.device)
    for a in range(0, k, group):
        x = X[:, a : a + group].double()
        zero = torch.zeros(rows, 1, dtype=torch.float64, device=X.device)
        lo, hi = torch.minimum(x.amin(1, keepdim=True), zero), torch.maximum(x.amax(1, keepdim=True), zero)
        span = (hi - lo).float().double() / 15 if zeros else torch.maximum(hi, -lo) / 7
        step = span.float().to(scale).double()
        q = torch.round((x / step).float().double())
        if zeros:
            z = torch.round((-lo / step).float().double()).clamp(0, 15)
            q = (q + z).clamp(0, 15) - z
        else:
            q = q.clamp(-8, 7)
        out[:, a : a + group] = torch.where(step > 0, q * step, 0.0)
    return out


def _exact_gate(G, act):
    """(act(G), its derivative) in 64 bits."""
    if act == "silu":
        y = torch.sigmoid(G)
        return G * y, y + G * y * torch.sigmoid(-G)
    if act == "gelu":
        phi = 0.5 * torch.erfc(-G / math.sqrt(2.0))
        return G * phi, phi + G * torch.exp(-G * G / 2) / math.sqrt(2.0 * math.pi)
    c = math.sqrt(2.0 / math.pi)
    y = torch.sigmoid(2.0 * c * (G + 0.044715 * G**3))
    return G * y, y + G * y * (1.0 - y) * 2.0 * c * (1.0 + 0.134145 * G**2)


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    op, rows, k = case["op"], case["rows"], case["k"]
    if op == "quant":
        X = s["X"].T if case["trans"] else s["X"]
        return _exact_rounded(X, case["group"], case["zeros"], DTYPES[case["scale"]])
    n, A = case["n"], s["A"].double()
    sizes = s.get("sizes", [rows])
    make = lambda *shape: torch.zeros(*shape, dtype=torch.float64, device="cuda")  # noqa: E731
    H, dA = make(rows, n), make(rows, k)
    dB = make(*s["B"].shape) if op == "step" else None
    a = 0
    for g, size in enumerate(sizes):
        b, of = a + size, (lambda t: t[g] if case["groups"] and t is not None else t)  # noqa: E731
        if size:
            if op in ("int4", "int4_gated"):
                W = _exact_values(of(s["codes"]), of(s["scales"]), of(s["zeros"]), k, case["group"]).T.contiguous()
            else:
                W = (of(s["B"]).T if case["trans"] else of(s["B"])).double().contiguous()
            P = A[a:b] @ W
            if op == "int4":
                H[a:b] = P
            else:
                G, U = P[:, :n], P[:, n:]
                y, slope = _exact_gate(G, case["act"])
                H[a:b] = y * U
                if op == "step":
                    d = s["dH"][a:b].double()
                    dP = torch.cat([d * U * slope, d * y], 1)
                    dA[a:b] = dP @ W.T.contiguous()
                    grad = A[a:b].T.contiguous() @ dP
                    of(dB).copy_(grad.T if case["trans"] else grad)
        a = b
    return (H, dA, dB) if op == "step" else H
