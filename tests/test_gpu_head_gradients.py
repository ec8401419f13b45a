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


def _one_sign(rows, c, dtype):
    """Numbers between 0.5 and 3, column by column in other binades."""
    g = torch.Generator(device="cuda").manual_seed(rows + c)
    x = torch.empty(rows, c, dtype=dtype, device="cuda")
    spread = 1 + torch.arange(c, device="cuda") / c
    for part in x.split(max(1, 2 ** 27 // c)):
        part.copy_((torch.rand(part.shape, generator=g, device="cuda") + 0.5) * spread)
    total = sum(part.double().sum(0) for part in x.split(max(1, 2 ** 27 // c)))
    return x, total


def _even(v, dtype):
    """1 / v as dl holds it: rounded to 16 bits, in fp16 times 2^14."""
    scale = 16384.0 if dtype == FP16 else 1.0
    return float((torch.tensor(1.0 / v, dtype=torch.float32) * scale).to(dtype).double()) / scale


def _mean_error(got, want, dtype):
    """Results are off by half a step u at most, 0.58 u in the root mean square: four times that over the root of their number, and a quarter of u for what the cuts of
    an accumulator take off a sum of one sign."""
    u = torch.finfo(dtype).eps / 2
    assert abs(float(((got.double() - want) / want).mean())) <= u * (0.25 + 4 * 0.58 / got.numel() ** 0.5)


@pytest.mark.parametrize("rows,c,v,dtype", [(2 ** 19, 4096, 250, FP16), (2 ** 20, 4096, 250, BF16), (2 ** 24, 64, 120, FP16), (2 ** 25, 64, 60, FP16), (2 ** 25, 64, 120, BF16), (2 ** 17 + 77, 512, 300, FP16)])
def test_sums_of_one_sign_over_many_rows(rows, c, v, dtype):
    """Weights of zero: all classes are as likely, and dW of those that are no target is a plain sum of x."""
    x, total = _one_sign(rows, c, dtype)
    w = torch.zeros(v, c, dtype=dtype, device="cuda", requires_grad=True)
    b = torch.zeros(v, device="cuda", requires_grad=True)
    dw, db = torch.autograd.grad(px.linear_cross_entropy(x, w, torch.zeros(rows, dtype=torch.long, device="cuda"), bias=b), (w, b))
    ops.device_error_flags()
    _mean_error(dw[1], total * _even(v, dtype) / rows, dtype)
    assert bool((dw[1:] == dw[1]).all())
    # db is formed from dl before it is rounded: fp32 over a lane's rows of up to 1024 tiles, and what is left of the exponentials
    assert float((db[1:].double() * v - 1).abs().max()) <= 1024 * 2.0 ** -24


@pytest.mark.parametrize("rows,c,v,dtype", [(2048, 4096, 131072, FP16), (600, 1024, 2 ** 19 + 3, FP16)])
def test_sums_of_one_sign_over_many_classes(rows, c, v, dtype):
    w, total = _one_sign(v, c, dtype)
    total = total - w[0].double()
    w[0] = 0.0
    x = torch.zeros(rows, c, dtype=dtype, device="cuda", requires_grad=True)
    dx = torch.autograd.grad(px.linear_cross_entropy(x, w, torch.zeros(rows, dtype=torch.long, device="cuda"), reduction="sum"), x)[0]
    ops.device_error_flags()
    _mean_error(dx[0], total * _even(v, dtype), dtype)
    assert bool((dx == dx[0]).all())


@pytest.mark.parametrize("rows", [148 * 128 * 128 + 1, 3 * 148 * 128 * 128 - 200])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_small_heads_in_several_launches(rows, reduction):
    """More rows than the accumulators of one launch take in fp16: every row's gradient, and sums over all of them."""
    x, w, b, t = _inputs(rows, 16, 20, FP16, seed=rows)
    each = torch.randn(rows, device="cuda") if reduction == "none" else None
    dx, dw, db = torch.autograd.grad(px.linear_cross_entropy(x, w, t, bias=b, reduction=reduction), (x, w, b), each)
    ops.device_error_flags()
    counts = t != -100
    g = torch.where(counts, (each if each is not None else torch.full((rows,), 1 / float(counts.sum()), device="cuda")).double(), 0.0)
    p = torch.softmax(x.detach().double() @ w.detach().double().t() + b.detach().double(), -1)
    y = torch.zeros_like(p).scatter_(1, t.clamp_min(0)[:, None], 1.0)
    dl, u = g[:, None] * (p - y), 2.0 ** -11
    # dl is off by u of itself and by what fp32 leaves of p, the results by u of themselves, and what they lose to fp16's smallest numbers
    for got, want, size, most in ((dx, dl @ w.detach().double(), dl.abs() @ w.detach().double().abs(), g.abs()[:, None] * 2 * w.detach().double().abs().sum(0)),
                                  (dw, dl.t() @ x.detach().double(), dl.abs().t() @ x.detach().double().abs(), 2 * (g.abs()[:, None] * x.detach().double().abs()).sum(0))):
        assert bool(((got.double() - want).abs() <= u * (1 + u) * size + u * want.abs() + 2.0 ** -17 * most + 2.0 ** -25).all())
    assert bool(((db.double() - dl.sum(0)).abs() <= 2.0 ** -14 * g.abs().sum()).all())


@pytest.mark.parametrize("rows,c,v", [(300, 264, 300), (9000, 136, 700), (70000, 64, 9000)])
@pytest.mark.parametrize("which", [(0, 1, 2), (0, 1), (1,), (1, 2), (0,)])
def test_ignored_rows_that_are_not_finite(rows, c, v, which):
    """The rows without them are kept where dx will be, or in the workspace of a call without dx; classes in one piece and in several."""
    x, w, b, t = _inputs(rows, c, v, BF16, seed=2)
    dirty = x.detach().clone()
    x.data[t == -100] = 0.0
    dirty[t == -100] = math.inf
    dirty.requires_grad_()
    out = []
    for y in (x, dirty):
        leaves = (y, w, b)
        out.append(torch.autograd.grad(px.linear_cross_entropy(y, w, t, bias=b), [leaves[i] for i in which]))
    ops.device_error_flags()
    assert all(bool(g.isfinite().all()) and torch.equal(g, z) for g, z in zip(*out))


@pytest.mark.parametrize("c,v", [(64, 90), (136, 300)])
@pytest.mark.parametrize("reduction", ["none", "mean"])
@pytest.mark.parametrize("dtype,power", [(BF16, -90), (BF16, -20), (BF16, 20), (BF16, 100), (FP16, -4), (FP16, 8)])
def test_the_scale_of_the_loss_enters_at_the_end(c, v, reduction, dtype, power):
    """All three gradients of a loss times a power of two are those of the loss times it, to the bit, where both are normal numbers of their type."""
    x, w, b, t = _inputs(150, c, v, dtype, seed=4)
    loss = px.linear_cross_entropy(x, w, t, bias=b, reduction=reduction)
    up = torch.randn(loss.shape, device="cuda")
    one = torch.autograd.grad(loss, (x, w, b), up, retain_graph=True)
    for g, z in zip(torch.autograd.grad(loss, (x, w, b), up * 2.0 ** power), one):
        least = torch.finfo(z.dtype).tiny
        normal = (z.abs() > least) & (g.abs() > least) & g.isfinite()      # the least itself may have come from below, where steps are wider
        assert float(normal.float().mean()) > 0.1 and torch.equal(g[normal].double(), z[normal].double() * 2.0 ** power)


@pytest.mark.parametrize("rows,c,v", [(300, 264, 300), (70000, 64, 9000), (300, 64, 50)])
def test_a_captured_pass_whose_ignored_rows_change(rows, c, v):
    """Replays find ignored rows that are finite, then not, then finite again, and other rows ignored."""
    x, w, b, t = _inputs(rows, c, v, BF16, seed=6)
    fixed, target = x.detach().clone().requires_grad_(), t.clone()
    for _ in range(2):
        torch.autograd.grad(px.linear_cross_entropy(fixed, w, target, bias=b), (fixed, w, b))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = px.linear_cross_entropy(fixed, w, target, bias=b)
        out = [loss.detach(), *torch.autograd.grad(loss, (fixed, w, b))]
    for hold, shift in ((0.0, 0), (math.nan, 0), (math.inf, 1), (1.0, 1)):
        with torch.no_grad():
            target.copy_(t.roll(shift))
            fixed.copy_(torch.where((target == -100)[:, None], hold, x))
        graph.replay()
        leaves = [l.detach().clone().requires_grad_() for l in (fixed, w, b)]
        want = px.linear_cross_entropy(leaves[0], leaves[1], target, bias=leaves[2])
        for a, z in zip(out, [want.detach(), *torch.autograd.grad(want, leaves)]):
            assert bool(z.isfinite().all()) and torch.equal(a, z)
    ops.device_error_flags()
