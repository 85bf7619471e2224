"""An expert layer trained on ragged groups of rows, then served from 4-bit weights.

    python -m examples.expert_layer [--device cpu|cuda] [--steps 40]

A router sends each token to its best `top` experts; rows sorted by expert go
through `grouped_gemm`. In training the gradients of the experts' matrices are
`grouped_rank_k`'s, summed over the micro-batches in fp32. For serving the experts
and the output projection become 4-bit floats (`mx_quantize`) and tokens go
through `mx_grouped_gemm` and `mx_gemm`; on a GPU one decoding step is a captured
graph, as no call waits for the router's counts.
"""

import argparse

import torch

import trnblas_amd as tb


class ExpertLinear(torch.autograd.Function):
    """x W[g] for the rows of group g; dW goes to `grad` (fp32), on top of what is there."""

    @staticmethod
    def forward(ctx, x, W, offsets, grad):
        ctx.save_for_backward(x, W, offsets)
        ctx.grad = grad
        return tb.grouped_gemm(1.0, x, W, offsets)

    @staticmethod
    def backward(ctx, dy):
        x, W, offsets = ctx.saved_tensors
        ctx.grad.copy_(tb.grouped_rank_k(1.0, x, dy, offsets, 1.0, ctx.grad, dtype=torch.float32))
        dx = tb.grouped_gemm(1.0, dy, W, offsets, transB=True) if ctx.needs_input_grad[0] else None
        return dx, None, None, None


class ExpertLayer:
    """y = Wo sum_e p_e(x) W2[e] silu(W1[e] x) over each token's best `top` experts; the router stays as it is."""

    def __init__(self, width, hidden, experts, top, device, dtype, seed=0):
        g = torch.Generator().manual_seed(seed)
        make = lambda *shape: torch.randn(*shape, generator=g).mul_(shape[-2] ** -0.5).to(device)
        self.top, self.dtype = top, dtype
        self.router = make(width, experts)
        # fp32 weights that the optimiser steps, their gradients, and what the products read
        self.master = [make(experts, width, hidden), make(experts, hidden, width), make(width, width)]
        self.grads = [torch.zeros_like(w) for w in self.master]
        self.weights = [w.to(dtype, copy=True).requires_grad_() for w in self.master]

    def route(self, x):
        """Rows' order by expert, the way back, the groups' offsets, the experts' shares."""
        share, expert = (x.float() @ self.router).softmax(-1).topk(self.top)
        expert, order = expert.flatten().sort(stable=True)
        offsets = torch.searchsorted(expert, torch.arange(self.router.shape[1] + 1, device=x.device))
        return order, order.argsort(), offsets, (share / share.sum(-1, keepdim=True)).to(x.dtype)

    def combine(self, rows, back, share):
        return (rows[back].view(*share.shape, -1) * share[..., None]).sum(1)

    def train_forward(self, x):
        W1, W2, Wo = self.weights
        order, back, offsets, share = self.route(x)
        h = ExpertLinear.apply(x[order // self.top], W1, offsets, self.grads[0])
        h = ExpertLinear.apply(torch.nn.functional.silu(h), W2, offsets, self.grads[1])
        return tb.grouped_gemm(1.0, self.combine(h, back, share), Wo[None], offsets[[0, -1]] // self.top)

    def step(self, micro_batches, rate):
        """One descent step over the micro-batches (x, target); returns the mean loss."""
        total = 0.0
        for grad in self.grads:
            grad.zero_()
        self.weights[2].grad = None
        for x, target in micro_batches:
            loss = (self.train_forward(x).float() - target).square().mean() / len(micro_batches)
            loss.backward()
            total += loss.detach()
        self.grads[2] += self.weights[2].grad
        for master, weight, grad in zip(self.master, self.weights, self.grads):
            master -= rate * grad / grad.square().mean().sqrt().clamp_min(1e-12)
            weight.data.copy_(master)
        return float(total)

    def quantised(self):
        """Weights stored (K, N): 4-bit floats along K, as (N, K)."""
        return [tb.mx_quantize(w.detach(), trans=True) for w in self.weights]

    def serve(self, x, quantised):
        E1, E2, Qo = quantised
        order, back, offsets, share = self.route(x)
        h = tb.mx_grouped_gemm(1.0, x[order // self.top], E1, offsets, dtype=self.dtype)
        h = tb.mx_grouped_gemm(1.0, torch.nn.functional.silu(h), E2, offsets, dtype=self.dtype)
        return tb.mx_gemm(1.0, self.combine(h, back, share), Qo, dtype=self.dtype)


def captured(layer, x, quantised):
    """serve() as a graph: a function of the tokens."""
    tokens = x.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer.serve(tokens, quantised)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer.serve(tokens, quantised)

    def run(x):
        tokens.copy_(x)
        graph.replay()
        return out.clone()

    return run


def main(argv=None):
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--device", default="cuda" if torch.cuda.is_available() else "cpu")
    p.add_argument("--steps", type=int, default=40)
    p.add_argument("--width", type=int, default=256)
    p.add_argument("--hidden", type=int, default=384)
    p.add_argument("--experts", type=int, default=8)
    p.add_argument("--tokens", type=int, default=512)
    args = p.parse_args(argv)
    dev, dtype = torch.device(args.device), torch.bfloat16
    layer = ExpertLayer(args.width, args.hidden, args.experts, 2, dev, dtype)
    teacher = ExpertLayer(args.width, args.hidden, args.experts, 2, dev, dtype, seed=1)
    teacher.router = layer.router
    g = torch.Generator().manual_seed(2)
    tokens = lambda n: torch.randn(n, args.width, generator=g).to(dev, dtype)
    losses = []
    for i in range(args.steps):
        batches = [(x, teacher.train_forward(x).detach().float()) for x in (tokens(args.tokens), tokens(args.tokens))]
        losses.append(layer.step(batches, 0.004 * (1.0 - i / args.steps)))
        if i % 10 == 0 or i == args.steps - 1:
            print(f"step {i:3d}  loss {losses[-1]:.5f}", flush=True)
    quantised = layer.quantised()
    bits = sum(8 * (q.codes.numel() + q.scales.numel()) for q in quantised) / sum(w.numel() for w in layer.weights)
    error = []
    with torch.no_grad():
        for n in (1, 7, args.tokens):
            x = tokens(n)
            exact, served = layer.train_forward(x).float(), layer.serve(x, quantised).float()
            error.append(float((served - exact).norm() / exact.norm()))
            print(f"served {n:4d} tokens from {bits:.2f} bits a weight: {100 * error[-1]:.1f} % from bfloat16", flush=True)
        same = True
        if dev.type == "cuda":
            x = tokens(7)
            run = captured(layer, x, quantised)
            for _ in range(3):
                x = tokens(7)
                same &= torch.equal(run(x), layer.serve(x, quantised))
            print("captured decoding step:", "same bits" if same else "differs", flush=True)
    return losses, error, same


if __name__ == "__main__":
    main()
