"""Gradients of linear_cross_entropy that are asked for one by one, of any scale, over many rows."""
import math

import pytest
import torch

import protenix_b200 as px
from protenix_b200 import ops

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def _inputs(rows, c, v, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, c, generator=g, device="cuda").to(dtype).requires_grad_()
    w = (torch.randn(v, c, generator=g, device="cuda") * 2 / math.sqrt(c)).to(dtype).requires_grad_()
    b = (torch.randn(v, generator=g, device="cuda") * 0.5).requires_grad_()
    t = torch.randint(0, v, (rows,), generator=g, device="cuda").masked_fill(torch.rand(rows, generator=g, device="cuda") < 0.2, -100)
    return x, w, b, t


@pytest.mark.parametrize("rows", [1, 129, 40000])
@pytest.mark.parametrize("v", [64, 128])
def test_small_heads_without_dw(rows, v):
    """The products for dW are formed all the same: launches that follow one another, on two shapes in turn, find tensor memory and barriers at rest."""
    x, w, b, t = _inputs(rows, 128, v, BF16, seed=v)
    y, u, a, s = _inputs(700, 72, 192 - v, BF16, seed=rows)
    loss, other = px.linear_cross_entropy(x, w, t, bias=b, reduction="sum"), px.linear_cross_entropy(y, u, s, bias=a, reduction="sum")
    dx, _, db = torch.autograd.grad(loss, (x, w, b), retain_graph=True)
    dy, du, da = torch.autograd.grad(other, (y, u, a), retain_graph=True)
    for _ in range(20):
        assert torch.equal(torch.autograd.grad(loss, x, retain_graph=True)[0], dx)
        assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(other, (y, u, a), retain_graph=True), (dy, du, da)))
        assert torch.equal(torch.autograd.grad(loss, b, retain_graph=True)[0], db)
    ops.device_error_flags()
