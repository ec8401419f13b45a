"""Gradients of windowed attention that fp16 cannot hold: they leave the kernels as infinities or NaN, which is how a loss scaler learns that its
scale is too large, and never as the largest finite number."""
import pytest
import torch

import protenix_b200 as px
from protenix_b200 import ops
from window_reference import reference

FP16 = torch.float16


def _grads(q, k, v, grad, window, sinks=0, mask=None):
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    o = px.window_attention(*leaves, window, sinks=sinks, mask=mask)
    got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(o, leaves, grad)))
    ops.device_error_flags()
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("d", [24, 32, 64, 128])
@pytest.mark.parametrize("n,window,sinks", [(200, (200, 0), 0), (4300, (33, 0), 1)])
def test_sums_beyond_the_type(d, n, window, sinks):
    """All weights alike and all gradients 60000: dV of the keys that many queries see passes 65504 (the second case: a sink, whose queries several CTAs share).
    V is zero, so nothing but the result is large.  A sum is off by its roundings, two of half a step: entries nearer than that to the border may go either way."""
    q = torch.zeros(1, 2, n, d, dtype=FP16, device="cuda")
    grad = torch.full_like(q, 60000.0)
    got = _grads(q, q, q, grad, window, sinks)
    want = reference(q, q, q, *window, sinks, grad=grad)["dv"][0]
    slack = 2.02 * 2.0 ** -11
    beyond, within = want > 65520 * (1 + slack), want < 65520 * (1 - slack)
    assert bool(beyond.any()) and bool(within.any())
    assert bool((got["dv"][beyond] == float("inf")).all())
    assert bool(((got["dv"].double() - want).abs() <= slack * want)[within].all())
    assert not got["dq"].any() and not got["dk"].any()


@pytest.mark.gpu
@pytest.mark.parametrize("d", [32, 64, 128])
def test_gradients_of_the_logits_beyond_the_type(d):
    """dS itself passes 65504 in most places: each gradient is right or not finite, and not finite where its value has no finite fp16."""
    g = torch.Generator(device="cuda").manual_seed(d)
    q, k, v, grad = (torch.randn(1, 2, 260, d, generator=g, device="cuda").to(FP16) for _ in range(4))
    v, grad = v * 100, grad * 4000
    got = _grads(q, k, v, grad, (3, 2))
    want = reference(q, k, v, 3, 2, grad=grad)
    for name in ("dq", "dk", "dv"):
        value, bound, _ = want[name]
        x = got[name].double()
        finite = torch.isfinite(x)
        assert bool(((x - value).abs() <= bound)[finite].all()), name
        assert not bool(finite[value.abs() - bound > 65520].any()), name
    assert not torch.isfinite(got["dq"]).all() and not torch.isfinite(got["dk"]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [FP16, torch.bfloat16])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
def test_a_gradient_that_is_not_finite_stays_so(bad, d, dtype):
    g = torch.Generator(device="cuda").manual_seed(d)
    q, k, v, grad = (torch.randn(1, 2, 260, d, generator=g, device="cuda").to(dtype) for _ in range(4))
    grad[0, 1, 140] = bad
    got = _grads(q, k, v, grad, (3, 2))
    assert not torch.isfinite(got["dq"][0, 1, 140]).any()
    for name in ("dk", "dv"):
        assert not torch.isfinite(got[name][0, 1, 137:143]).any(), name
        assert torch.isfinite(got[name][0, 0]).all(), name
