"""Windowed attention in fp16 where all weights but one are far below the smallest normal number of the type."""
import math

import pytest
import torch

import protenix_b200 as px
from window_reference import reference

FP16 = torch.float16
U = 2.0 ** -11


def _one_large(n, d, at):
    """Key `at` stands 14.28 above the others, whose weights are 10.5 steps of 2^-24 then: in the middle between two subnormal numbers, 4.8 % from either."""
    q = torch.ones(1, 2, n, d, dtype=FP16, device="cuda")
    k = torch.zeros_like(q)
    k[:, :, at] = math.log(2.0 ** 24 / 10.5) / d
    g = torch.Generator(device="cuda").manual_seed(d)
    some = (torch.rand(1, 2, n, d, generator=g, device="cuda") + 0.5) * 100
    return q, k, some.to(FP16)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("at", [0, 150, 299])
def test_output_of_small_weights(d, at):
    """The large key's value is zero, so that o is what the others add up to.  Each term: the weight rounded (U), fp32 steps and an exponential of a logit of
    14.3 (2^-20 (1 + 14.3) < 2^-16); then the result rounded (U)."""
    n = 300
    q, k, v = _one_large(n, d, at)
    v[:, :, at] = 0
    o = px.window_attention(q, k, v, n, scale=1.0)
    want = reference(q, k, v, n, n, scale=1.0)["o"][0]
    assert bool(((o.double() - want).abs() <= (2.01 * U + 2.0 ** -16) * want.abs()).all())


@pytest.mark.gpu
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("n,window,sinks,at", [(300, (300, 300), 0, 0), (300, (300, 300), 0, 150), (4300, (33, 0), 3, 1)])
def test_gradient_of_values_with_small_weights(d, n, window, sinks, at):
    """dV of the other keys, whose terms all have one sign: the same roundings."""
    q, k, grad = _one_large(n, d, at)
    v = torch.zeros_like(q).requires_grad_()
    if n > 300:
        grad = grad * 2.0 ** -5      # many queries see the sink: its own gradient stays a number of the type
    dv, = torch.autograd.grad(px.window_attention(q, k, v, window, sinks=sinks, scale=1.0), v, grad)
    want = reference(q, k, v.detach(), *window, sinks, scale=1.0, grad=grad)["dv"][0]
    smallest = torch.finfo(FP16).smallest_normal * U      # a result that is subnormal itself
    assert bool(torch.isfinite(dv).all())
    assert bool(((dv.double() - want).abs() <= (2.01 * U + 2.0 ** -16) * want.abs() + smallest).all())
