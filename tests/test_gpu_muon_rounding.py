"""GPU tests of the update's roundings, bit by bit: p = fma(-rate, O, p decay) where the direction O is known exactly, and
m = fma(momentum, m, (1 - momentum) g)."""
import numpy as np
import pytest
import torch

from laser_amd import grad_ops as G

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,cols", [(16, 16), (64, 64), (16, 128), (100, 128), (128, 250), (60, 900), (900, 60), (100, 1000), (200, 301), (301, 200),
                                       (300, 300), (700, 260), (768, 768), (256, 1024)])
def test_two_roundings(rows, cols):
    """One step with (a, 0, 0) gives a U / |U|.  U holds 4^k ones among zeros, so that O is a / 2^k there; a has 20 bits."""
    torch.manual_seed(rows * cols)
    n = 1
    while 4 * n <= rows * cols:
        n *= 4
    a = round(1.2345678 * 2 ** 19) / 2 ** 19
    g = torch.zeros(2, rows * cols, device="cuda")
    for i in range(2):
        g[i, torch.randperm(rows * cols, device="cuda")[:n]] = 1.0
    g = g.view(2, rows, cols)
    p = 0.5 + 0.5 * torch.rand(2, rows, cols, device="cuda")
    lr, decay, scale = np.float32(7.1), np.float32(0.0123), np.float32(0.9 * n ** 0.5 / 16)
    rate, keep = np.float32(np.float64(lr) * np.float64(scale)), np.float32(1.0 - np.float64(lr) * np.float64(decay))
    o = g.double() * (a / n ** 0.5)
    # at most 24 + 20 bits of the product and 24 of p beside it: 64 bits hold the difference exactly
    want = ((p * float(keep)).double() - float(rate) * o).float()
    G.muon_step(list(p), list(g), torch.zeros_like(p), lr=float(lr), momentum=0.0, nesterov=False, weight_decay=float(decay), scale=float(scale), steps=1,
                coefficients=(a, 0.0, 0.0), eps=0.0)
    assert torch.equal(p, want)


@pytest.mark.parametrize("rows,cols", [(16, 16), (100, 128), (128, 250), (60, 900), (900, 60), (200, 301), (768, 768)])
def test_momentum_is_rounded_twice(rows, cols):
    torch.manual_seed(rows * cols)
    g, m, p = (0.5 + 0.5 * torch.rand(2, rows, cols, device="cuda") for _ in range(3))
    mu = np.float32(0.9)
    # products of 48 bits below 1, sums of 49: exact in 64 bits
    want = (float(mu) * m.double() + (float(np.float32(1) - mu) * g).double()).float()
    G.muon_step(list(p), list(g), m, lr=0.1, momentum=float(mu))
    assert torch.equal(m, want)
