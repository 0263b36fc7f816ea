"""Accuracy of the linear layer and the MLP where bounds by magnitudes or norms would not see a loss."""

from __future__ import annotations

import math

import pytest
import torch

from dabsn_amd import fused_linear, fused_mlp
from test_linear import Val, activated
from test_norm import U, within

BF16, FP32 = torch.bfloat16, torch.float32

# ---- slopes far from zero ---------------------------------------------------------------------
# GELU's slope is 2^-25 at -5.5 and 2^-39 at -7.7, SiLU's at -20.5 and -30.7.
TAILS = {"gelu": (-7.5, -4.5), "silu": (-30.0, -14.0)}


def _tail(act):
    z = torch.linspace(*TAILS[act], 4096).to(BF16)
    _, slope = activated(Val(z.cuda()), act)
    # Kept with 2^-11 of itself or 2^-39; GELU's fit 1.7e-5 of a term below half the slope there;
    # exp's argument (up to 30) u of itself off, some more operations.
    tol = (2.0 ** -11 + 2e-5 + 64 * U) * slope.v.abs() + 2.0 ** -39
    return z, slope.v, tol


@pytest.mark.gpu
@pytest.mark.parametrize("act", TAILS)
def test_gradients_of_tails(cuda_device, act):
    """Small slopes relative to themselves: through a product with one term, in the gradient's pass."""
    z, slope, tol = _tail(act)
    x = z.cuda()[:, None].requires_grad_(True)
    one = torch.ones(1, 1, device=cuda_device, dtype=BF16)
    (dx,) = torch.autograd.grad(fused_linear(x, one, activation=act), x, torch.ones_like(x))
    within(dx[:, 0], slope, tol + 2.0 ** -8 * (slope.abs() + tol))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 256])
@pytest.mark.parametrize("act", TAILS)
def test_gradients_of_tails_of_the_mlp(cuda_device, act, m):
    """The same in the products' epilogues: a first layer without weights, whose arguments are its bias."""
    z, slope, tol = _tail(act)
    f, h = z.numel(), 8
    x = torch.randn(m, h, device=cuda_device).to(BF16)
    b1 = z.cuda().requires_grad_(True)
    w1 = torch.zeros(f, h, device=cuda_device, dtype=BF16)
    w2 = torch.zeros(h, f, device=cuda_device, dtype=BF16)
    w2[0] = 1
    up = torch.zeros(m, h, device=cuda_device, dtype=BF16)
    up[:, 0] = 1
    (db,) = torch.autograd.grad(fused_mlp(x, w1, w2, b1, activation=act), b1, up)
    # All rows have the same dz, rounded to bf16; their number is a power of two.
    within(db / m, slope, tol + 2.0 ** -8 * (slope.abs() + tol))
