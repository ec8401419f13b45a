"""dropout_add against its formula in 64 bits, with the mask from the tests' own generator."""
import numpy as np
import pytest
import torch

import protenix_b200 as px
from philox import keep

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}   # finfo.eps / 2
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _inputs(shape, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(shape, generator=g).to(dtype).cuda() for _ in range(3)]


def _check(got, residual, x, mask, p, dtype):
    """One rounding of the result to its type; before it, those of 1 / (1 - p), of the product and of the sum to fp32."""
    m = torch.from_numpy(mask).cuda()
    prod = torch.where(m, x.double() / (1 - p) if p < 1 else x.double() * 0, torch.zeros((), dtype=torch.float64, device="cuda"))
    want = prod + (residual.double() if residual is not None else 0)
    # a value in the subnormal range is off by half of its step, whatever its size
    bound = HALF_STEP[dtype] * want.abs() * (1 + 2.0 ** -10) + 2.0 ** -23 * prod.abs() + 2.0 ** -24 * want.abs() + torch.finfo(dtype).smallest_normal * HALF_STEP[dtype]
    assert got.dtype == dtype and bool(((got.double() - want).abs() <= bound).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,dim", [((1,), None), ((3,), None), ((384, 384), None), ((1001, 3), None), ((5, 7, 3), -3), ((5, 7, 3), 1),
                                       ((2, 37, 20, 128), -3), ((2, 37, 20, 128), -2), ((2, 37, 20, 128), 0), ((2, 37, 20, 128), -1),
                                       ((0, 4), None), ((3, 0, 8), -2), ((1, 1, 128), -3), ((70000, 8), 0), ((97, 97, 128), None)])
def test_against_the_formula(shape, dim, dtype):
    residual, x, grad = _inputs(shape, dtype)
    p, seed, offset = 0.3, (5 << 40) + 11, (1 << 33) + 2
    mask = keep(shape, p, seed, offset, dim)
    xr, rr = x.clone().requires_grad_(), residual.clone().requires_grad_()
    out = px.dropout_add(rr, xr, p, seed, offset=offset, shared_dim=dim)
    _check(out.detach(), residual, x, mask, p, dtype)
    _check(px.dropout_add(None, x, p, seed, offset=offset, shared_dim=dim), None, x, mask, p, dtype)
    dr, dx = torch.autograd.grad(out, (rr, xr), grad)
    assert torch.equal(dr, grad)
    _check(dx, None, grad, mask, p, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("p", [0.0, 1e-9, 0.5, 1 - 1e-9, 1.0])
def test_extreme_probabilities(p):
    residual, x, _ = _inputs((33, 128), torch.float32)
    _check(px.dropout_add(residual, x, p, 9), residual, x, keep((33, 128), p, 9, 0), p, torch.float32)


@pytest.mark.gpu
def test_dropped_elements_may_hold_anything():
    residual, x, _ = _inputs((64, 64), torch.bfloat16)
    mask = torch.from_numpy(keep((64, 64), 0.5, 4, 0)).cuda()
    bad = torch.where(mask, x, torch.full_like(x, float("nan")))
    assert torch.equal(px.dropout_add(residual, bad, 0.5, 4), px.dropout_add(residual, x, 0.5, 4))
    assert bool((px.dropout_add(residual, x, 0.5, 4)[~mask] == residual[~mask]).all())


@pytest.mark.gpu
def test_places_count_not_memory_order():
    """Strided, misaligned and transposed tensors drop what their contiguous copies drop."""
    residual, x, grad = _inputs((48, 40, 16), torch.float16)
    want = px.dropout_add(residual, x, 0.25, 3, shared_dim=-2)
    turned = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(px.dropout_add(turned(residual), turned(x), 0.25, 3, shared_dim=-2), want)
    off = torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")[1:].view(x.shape).copy_(x)
    assert off.data_ptr() % 16 and torch.equal(px.dropout_add(residual, off, 0.25, 3, shared_dim=-2), want)
    assert torch.equal(px.dropout_add(residual, off, 0.25, 3), px.dropout_add(residual, x, 0.25, 3))
    xr = x.clone().requires_grad_()
    out = px.dropout_add(None, xr, 0.25, 3)
    assert torch.equal(torch.autograd.grad(out, xr, turned(grad))[0], px.dropout_add(None, grad, 0.25, 3))
    # one gradient for all elements, as sum() gives it
    xr = x.clone().requires_grad_()
    px.dropout_add(None, xr, 0.25, 3).sum().backward()
    assert torch.equal(xr.grad, px.dropout_add(None, torch.ones_like(x), 0.25, 3))


@pytest.mark.gpu
def test_seeds_and_offsets():
    x = torch.ones(1 << 16, device="cuda")
    a = px.dropout_add(None, x, 0.5, 1)
    assert torch.equal(a, px.dropout_add(None, x, 0.5, 1))
    for other in (px.dropout_add(None, x, 0.5, 2), px.dropout_add(None, x, 0.5, 1 + (1 << 32)), px.dropout_add(None, x, 0.5, 1, offset=1),
                  px.dropout_add(None, x, 0.5, 1, offset=1 << 32)):
        assert abs(float((a == other).float().mean()) - 0.5) < 0.02      # ten standard deviations


@pytest.mark.gpu
def test_seed_on_the_device():
    residual, x, grad = _inputs((40, 128), torch.float32)
    state = torch.tensor([77, 5], device="cuda")
    xr = x.clone().requires_grad_()
    out = px.dropout_add(residual, xr, 0.4, state)
    state += 1                                            # the backward pass drops what the forward pass dropped
    assert torch.equal(out.detach(), px.dropout_add(residual, x, 0.4, 77, offset=5))
    assert torch.equal(torch.autograd.grad(out, xr, grad)[0], px.dropout_add(None, grad, 0.4, 77, offset=5))
    assert torch.equal(px.dropout_add(residual, x, 0.4, state), px.dropout_add(residual, x, 0.4, 78, offset=6))


@pytest.mark.gpu
def test_captured_step_draws_anew():
    x = torch.randn(128, 128, device="cuda").requires_grad_()
    grad, state = torch.randn(128, 128, device="cuda"), torch.tensor([3, 0], device="cuda")

    def step():
        out = px.dropout_add(None, x, 0.5, state)
        dx, = torch.autograd.grad(out, x, grad)
        state[1:].add_(1)
        return out, dx

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, dx = step()
    for i in range(1, 4):
        graph.replay()
        assert torch.equal(out, px.dropout_add(None, x.detach(), 0.5, 3, offset=i))
        assert torch.equal(dx, px.dropout_add(None, grad, 0.5, 3, offset=i))


@pytest.mark.gpu
def test_second_derivative():
    x = torch.randn(6, 8, dtype=torch.float32, device="cuda", requires_grad=True)
    out = px.dropout_add(None, x, 0.5, 3)
    dx, = torch.autograd.grad((out ** 2).sum(), x, create_graph=True)
    ddx, = torch.autograd.grad(dx.sum(), x)
    mask = torch.from_numpy(keep((6, 8), 0.5, 3, 0)).cuda()
    assert torch.equal(ddx, mask * 8.0)                   # d/dx of 2 m (m x) with m = 2 where kept


@pytest.mark.gpu
def test_other_stream_and_eval():
    residual, x, _ = _inputs((300, 128), torch.bfloat16)
    want = px.dropout_add(residual, x, 0.1, 6)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = px.dropout_add(residual, x, 0.1, 6)
    s.synchronize()
    assert torch.equal(got, want)
    assert torch.equal(px.dropout_add(residual, x, 0.1, 6, training=False), residual + x)


def test_cpu_tensors_and_bad_seeds_are_refused():
    x = torch.zeros(4)
    with pytest.raises(RuntimeError, match="no CPU path"):
        px.dropout_add(None, x, 0.1, 3)


@pytest.mark.gpu
def test_refusals():
    x = torch.zeros(4, 8, device="cuda")
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(RuntimeError, match="probability"):
            px.dropout_add(None, x, p, 3)
    for seed in (-1, 1 << 63, 0.5):
        with pytest.raises(RuntimeError, match="seed"):
            px.dropout_add(None, x, 0.1, seed)
    with pytest.raises(RuntimeError, match="offset"):
        px.dropout_add(None, x, 0.1, 3, offset=-1)
    with pytest.raises(RuntimeError, match="holds the offset"):
        px.dropout_add(None, x, 0.1, torch.zeros(2, dtype=torch.long, device="cuda"), offset=1)
    for state in (torch.zeros(3, dtype=torch.long, device="cuda"), torch.zeros(2, device="cuda"), torch.zeros(2, dtype=torch.long)):
        with pytest.raises(RuntimeError, match="seed"):
            px.dropout_add(None, x, 0.1, state)
    with pytest.raises(RuntimeError, match="out of range"):
        px.dropout_add(None, x, 0.1, 3, shared_dim=2)
    with pytest.raises(RuntimeError, match="match"):
        px.dropout_add(x[:2], x, 0.1, 3)
    with pytest.raises(RuntimeError, match="float"):
        px.dropout_add(None, x.double(), 0.1, 3)
