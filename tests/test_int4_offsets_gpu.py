"""Gated products with 4-bit weights at the last size that the tile kernel's 32-bit offsets reach, and the first past it."""

import pytest
import torch
from test_gated_int4_limits_gpu import _blocks
from test_int4_offsets_host import BF16, last_inside, plan

import trnblas_amd as tb
from oracle import gated as oa
from trnblas_amd.int4 import Int4Matrix

pytestmark = pytest.mark.gpu


def test_ups_at_the_end_of_reach(dev):
    # 34 GB of codes; K no multiple of 128
    K, group, rows = 1032, 32, 32
    N = last_inside(K, group)
    assert plan(BF16, 1, 1, rows, N, K, group)[0] == 64 and plan(BF16, 1, 1, rows, N + 16, K, group)[0] == 0
    blocks, chunks = 2 * (N + 16) // 16, -(-K // 128)
    g = torch.Generator(device=dev).manual_seed(0)
    codes = torch.empty(blocks, chunks, 1024, dtype=torch.uint8, device=dev)
    codes.view(torch.int64).random_(generator=g)
    scales = torch.empty(blocks, chunks, 16, 4, dtype=torch.bfloat16, device=dev).uniform_(0.5, 1.5, generator=g)
    zeros = torch.empty(blocks, chunks, 16, 4, dtype=torch.uint8, device=dev).random_(0, 16, generator=g)
    A = torch.randn(rows, K, generator=torch.Generator().manual_seed(1)).to(dev, torch.bfloat16) / 64
    for n in (N, N + 16):  # the tile kernel, the few-rows kernel
        for z in (None, zeros):
            cut = lambda t: None if t is None else t[: 2 * n // 16]
            Q = Int4Matrix(cut(codes), cut(scales), cut(z), (2 * n, K), group)
            H = tb.gated_gemm(A, Q, "silu")
            for a in (0, n // 32 - 4, n // 16 - 8):
                W = torch.cat([_blocks(Q, a + up, a + up + 8).dequantize() for up in (0, n // 16)])[None]
                P, den = oa.products(A, W, torch.tensor([0, rows]), True)
                assert oa.ratio(H[:, 16 * a : 16 * a + 128], *oa.forward("silu", P, den, K, torch.bfloat16)) <= 1, (n, a)
            del H, Q
