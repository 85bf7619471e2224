"""The expert layer of examples/: the grouped and the 4-bit products run together, as a user would."""

import pytest
import torch
from examples import expert_layer as ex

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
def test_layer_and_its_gradients(device):
    """fp32 against every token through every expert in 64 bits. Values and gradients of order one or less pass three sums
    of up to 48 fp32 products and, in the gradients, one over 64 rows: below 1e-4 of the largest."""
    layer = ex.ExpertLayer(32, 48, 5, 2, torch.device(device), torch.float32)
    g = torch.Generator().manual_seed(3)
    x, target = torch.randn(33, 32, generator=g).to(device), torch.randn(33, 32, generator=g).to(device)
    W1, W2, Wo = (w.cpu().double().requires_grad_() for w in layer.master)
    p, e = (x.cpu().double() @ layer.router.cpu().double()).softmax(-1).topk(2)
    p = torch.zeros(33, 5, dtype=torch.float64).scatter(1, e, p / p.sum(-1, keepdim=True))
    h = torch.nn.functional.silu(torch.matmul(x.cpu().double()[None], W1)) @ W2
    y = (p.T[..., None] * h).sum(0) @ Wo
    (y - target.cpu().double()).square().mean().backward()
    got = layer.train_forward(x)
    assert (got.cpu().double() - y).abs().max() <= 1e-4 * y.abs().max()
    layer.step([(x, target)], 0.0)
    for grad, want in zip(layer.grads, (W1.grad, W2.grad, Wo.grad)):
        assert (grad.cpu().double() - want).abs().max() <= 1e-4 * want.abs().max()
    # two micro-batches of the same rows: their mean is the same gradient
    once = [grad.clone() for grad in layer.grads]
    layer.step([(x, target), (x, target)], 0.0)
    for grad, want in zip(layer.grads, once):
        assert (grad - want).abs().max() <= 1e-4 * want.abs().max()


@pytest.mark.parametrize("device", DEVICES)
def test_trains_and_serves(device, capsys):
    """The loss falls; 4-bit serving is near. Rounding to e2m1 moves a normal value by about a tenth of its size, both
    operands of three products: sqrt(6) / 10, twice that allowed. A captured step repeats the eager one's bits."""
    losses, error, same = ex.main(["--device", device, "--steps", "12", "--width", "64", "--hidden", "96", "--tokens", "256"])
    assert losses[-1] < 0.8 * losses[0]
    assert max(error) < 0.5
    assert same
    assert "served" in capsys.readouterr().out
