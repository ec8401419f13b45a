"""linear_cross_entropy against the formula in 64 bits, at the sizes, targets and values where it can go wrong."""
import math

import pytest
import torch

import protenix_b200 as px
from protenix_b200 import ops

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def _inputs(rows, c, v, dtype, bias=None, ignored=0.2, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, c, generator=g, device="cuda").to(dtype).requires_grad_()
    w = (torch.randn(v, c, generator=g, device="cuda") * 2 / math.sqrt(c)).to(dtype).requires_grad_()
    b = (torch.randn(v, generator=g, device="cuda") * 0.5).to(bias).requires_grad_() if bias is not None else None
    t = torch.randint(0, v, (rows,), generator=g, device="cuda")
    t = t.masked_fill(torch.rand(rows, generator=g, device="cuda") < ignored, -100)
    t[0] = v - 1
    return x, w, b, t


def _formula(x, w, b, t, smooth=0.0, weight=None):
    """Losses of the rows, and for gradients `weight` of them those of x, w and b, in 64 bits; with the sums of absolute values that bound the
    kernels' roundings.  Rows that do not count are left out of everything."""
    x, w = x.detach().double(), w.detach().double()
    b = torch.zeros(len(w), dtype=torch.float64, device="cuda") if b is None else b.detach().double()
    counts = (t != -100)[:, None]
    x = torch.where(counts, x, 0.0)
    v = len(w)
    logits = x @ w.t() + b
    y = torch.zeros_like(logits).scatter_(1, t.clamp_min(0)[:, None], 1.0) * (1.0 - smooth) + smooth / v
    lse = torch.logsumexp(logits, -1)
    losses = torch.where(counts[:, 0], lse - (y * logits).sum(-1), 0.0)
    out = {"losses": losses, "size": (x.abs() @ w.abs().t() + b.abs()).amax(-1)}
    if weight is not None:
        g = torch.where(counts, weight.double()[:, None], 0.0)
        p = torch.exp(logits - lse[:, None])
        dl, most = g * (p - y), g.abs() * (p + y)
        out.update(dx=dl @ w, dw=dl.t() @ x, db=dl.sum(0), dx_abs=dl.abs() @ w.abs(), dw_abs=dl.abs().t() @ x.abs(),
                   dx_most=most @ w.abs(), dw_most=most.t() @ x.abs(), db_most=most.sum(0))
    return out


def _loss_close(got, want, c, share=1.0):
    # An fp32 sum of c products loses at most half a step for each of c / 16 additions and each of the products; lse, its logarithm and the
    # difference are a few steps of numbers of that size.
    tol = 2.0 ** -23 * (c / 16 + 24) * (want["size"].max() + math.log(2 ** 17)) * share
    assert float((got.double() - want["losses"]).abs().max()) <= float(tol)


def _grad_close(name, got, want, dtype, c):
    """dl is off by half a step of `dtype`, and by what fp32 logits and exponentials leave of p; the result by half a step of its own."""
    u = torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == FP16 else 0.0
    fp32 = 2.0 ** -23 * (c / 16 + 24) * 40          # 40: logits are below that, and an error of l is a relative one of p
    bound = (u * (1 + u)) * want[name + "_abs"] + fp32 * want[name + "_most"] + u * want[name].abs() + tiny
    assert bool(((got.detach().double() - want[name]).abs() <= bound * (1 + 1e-9) + 1e-30).all()), name


SIZES = [(1, 8, 2), (5, 8, 3), (128, 64, 64), (129, 72, 65), (384, 384, 32), (300, 128, 257), (31, 1024, 1000), (257, 264, 256), (1000, 136, 4999), (4096, 256, 8192),
         (1000, 128, 128), (257, 128, 127), (300, 64, 128), (130, 120, 129), (40000, 128, 64), (41001, 96, 100), (20000, 264, 70)]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("rows,c,v", SIZES)
@pytest.mark.parametrize("reduction,smooth,bias", [("mean", 0.0, None), ("sum", 0.1, "own"), ("none", 0.3, "fp32")])
def test_against_64_bits(rows, c, v, dtype, reduction, smooth, bias):
    x, w, b, t = _inputs(rows, c, v, dtype, {None: None, "own": dtype, "fp32": torch.float32}[bias], seed=rows + v)
    loss = px.linear_cross_entropy(x, w, t, bias=b, label_smoothing=smooth, reduction=reduction)
    counts = t != -100
    each = torch.randn(rows, device="cuda") if reduction == "none" else torch.ones(rows, device="cuda") / (counts.sum() if reduction == "mean" else 1)
    leaves = [y for y in (x, w, b) if y is not None]
    grads = torch.autograd.grad(loss, leaves, each if reduction == "none" else None)
    ops.device_error_flags()
    want = _formula(x, w, b, t, smooth, each)
    assert loss.dtype == torch.float32
    if reduction == "none":
        _loss_close(loss.detach(), want, c)
        assert not bool(loss[~counts].any())
    else:
        want["losses"] = want["losses"].sum() / (counts.sum() if reduction == "mean" else 1)
        _loss_close(loss.detach(), want, c, 1.0 if reduction == "mean" else float(counts.sum()))
    _grad_close("dx", grads[0], want, dtype, c)
    _grad_close("dw", grads[1], want, dtype, c)
    assert not bool(grads[0][~counts].any())
    for y, g in zip(leaves, grads):
        assert g.dtype == y.dtype and g.shape == y.shape
    if b is not None:
        u = torch.finfo(b.dtype).eps / 2
        fp32 = 2.0 ** -23 * (c / 16 + 24) * 40
        tiny = 2.0 ** -25 if b.dtype == FP16 else 0.0
        assert bool(((grads[2].double() - want["db"]).abs() <= fp32 * want["db_most"] + u * want["db"].abs() + tiny + 1e-30).all())
    plain = px.linear_cross_entropy(x.detach(), w.detach(), t, bias=b, label_smoothing=smooth, reduction=reduction)
    assert torch.equal(plain, loss.detach())
    again = torch.autograd.grad(px.linear_cross_entropy(x, w, t, bias=b, label_smoothing=smooth, reduction=reduction), leaves, each if reduction == "none" else None)
    for a, z in zip(grads, again):
        assert torch.equal(a, z)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_more_classes_than_a_piece(dtype):
    """70 000 rows and 9 000 classes: dl in three pieces, the gradient of x added up over them."""
    x, w, b, t = _inputs(70000, 64, 9000, dtype, torch.float32, seed=3)
    loss = px.linear_cross_entropy(x, w, t, bias=b)
    grads = torch.autograd.grad(loss, (x, w, b))
    ops.device_error_flags()
    counts = t != -100
    want = _formula(x, w, b, t, 0.0, torch.ones(len(t), device="cuda") / counts.sum())
    want["losses"] = want["losses"].sum() / counts.sum()
    _loss_close(loss.detach(), want, 64)
    _grad_close("dx", grads[0], want, dtype, 64)
    _grad_close("dw", grads[1], want, dtype, 64)


@pytest.mark.parametrize("rows,v", [(2048, 19990), (19990, 2048)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_a_last_round_of_few_tiles(rows, v, dtype):
    """79 tiles of 256 x 256 for dW, or for dx: two rounds, or parts of them."""
    x, w, b, t = _inputs(rows, 248, v, dtype, torch.float32, seed=6)
    loss = px.linear_cross_entropy(x, w, t, b, reduction="sum")
    grads = torch.autograd.grad(loss, (x, w, b))
    want = _formula(x, w, b, t, weight=torch.ones(rows, device="cuda"))
    for name, got in zip(("dx", "dw"), grads):
        _grad_close(name, got, want, dtype, 248)
    bound = 2.0 ** -23 * ((248 / 16 + 24) * 40 + 64) * want["db_most"]
    assert bool(((grads[2].double() - want["db"]).abs() <= bound + 1e-30).all())
    assert not bool(grads[0][t == -100].any())
    again = torch.autograd.grad(px.linear_cross_entropy(x, w, t, b, reduction="sum"), (x, w, b))
    assert all(torch.equal(y, z) for y, z in zip(grads, again))


@pytest.mark.parametrize("rows,c,v", [(200, 64, 50), (200, 136, 700)])
@pytest.mark.parametrize("hold", [math.nan, math.inf, -math.inf])
def test_ignored_rows_have_no_influence(rows, c, v, hold):
    x, w, b, t = _inputs(rows, c, v, BF16, BF16, ignored=0.4, seed=8)
    zeros, dirty = x.detach().clone(), x.detach().clone()
    zeros[t == -100] = 0.0
    dirty[t == -100] = hold
    out = []
    for y in (zeros, dirty):
        y.requires_grad_()
        loss = px.linear_cross_entropy(y, w, t, bias=b)
        out.append((loss.detach(), *torch.autograd.grad(loss, (y, w, b))))
    for a, z in zip(*out):
        assert bool(torch.isfinite(z).all()) and torch.equal(a, z)


@pytest.mark.parametrize("rows,c,v", [(70, 128, 130), (300, 264, 300), (9000, 136, 700)])
@pytest.mark.parametrize("sign", [0.0, 1.0, -1.0])
def test_one_element_of_an_ignored_row(rows, c, v, sign):
    """Infinite logits of one sign, or NaN, in a single ignored row; its neighbours and the rows of other tiles keep their part."""
    x, w, b, t = _inputs(rows, c, v, BF16, torch.float32, ignored=0.3, seed=4)
    t[rows - 2] = -100
    with torch.no_grad():
        w[:, 5] = sign
    outs = []
    for hold in (0.0, math.inf):
        x.data[rows - 2, 5] = hold
        loss = px.linear_cross_entropy(x, w, t, b, label_smoothing=0.1)
        outs.append((loss.detach(), *torch.autograd.grad(loss, (x, w, b))))
    for y, z in zip(*outs):
        assert bool(y.isfinite().all()) and torch.equal(y, z)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_all_rows_ignored(reduction):
    x, w, b, t = _inputs(140, 64, 70, FP16, FP16)
    t[:] = -100
    x.data[3] = math.nan
    loss = px.linear_cross_entropy(x, w, t, bias=b, reduction=reduction)
    assert bool(torch.isnan(loss)) if reduction == "mean" else not bool(loss.any())
    for g in torch.autograd.grad(loss, (x, w, b), torch.ones_like(loss)):
        assert not bool(g.any())


def test_no_rows():
    x, w, _, _ = _inputs(1, 64, 70, BF16)
    none = torch.zeros(0, 64, dtype=BF16, device="cuda", requires_grad=True)
    t = torch.zeros(0, dtype=torch.long, device="cuda")
    for reduction in ("mean", "sum", "none"):
        loss = px.linear_cross_entropy(none, w, t, reduction=reduction)
        assert loss.dtype == torch.float32 and loss.shape == (() if reduction != "none" else (0,))
        assert bool(torch.isnan(loss)) if reduction == "mean" else not bool(loss.any())
        dx, dw = torch.autograd.grad(loss, (none, w), torch.ones_like(loss))
        assert dx.shape == (0, 64) and not bool(dw.any())


def test_targets_outside_the_classes():
    """They fault nothing: their rows' losses are NaN, the other rows' losses and gradients what they are."""
    x, w, _, t = _inputs(150, 64, 300, BF16, ignored=0.0)
    good = t.clone()
    good[[3, 77]] = -100
    t[3], t[77] = 300, -5
    for bad in (t, torch.where(t == 300, 1 << 40, t)):
        loss = px.linear_cross_entropy(x, w, bad, reduction="none")
        keep = torch.ones(150, dtype=torch.bool, device="cuda")
        keep[[3, 77]] = False
        assert bool(torch.isnan(loss[~keep]).all())
        other = px.linear_cross_entropy(x, w, good, reduction="none")
        assert torch.equal(loss[keep], other[keep])
        dx, dw = torch.autograd.grad(loss.sum(), (x, w))
        ox, _ = torch.autograd.grad(other.sum(), (x, w))
        assert torch.equal(dx[keep], ox[keep]) and bool(torch.isnan(dx[~keep]).all()) and bool(torch.isnan(dw).all())


def test_hidden_classes():
    """A bias of minus infinity takes a class out: as if it were not there."""
    x, w, _, t = _inputs(140, 64, 600, BF16, ignored=0.0)
    b = torch.zeros(600, device="cuda")
    b[256:512] = -math.inf           # a whole tile of classes among them
    t = t % 256
    kept = torch.cat([torch.arange(256), torch.arange(512, 600)]).cuda()
    loss = px.linear_cross_entropy(x, w, t, bias=b)
    dx, dw = torch.autograd.grad(loss, (x, w))
    want = _formula(x, w.detach()[kept], None, t, 0.0, torch.ones(140, device="cuda") / 140)
    want["losses"] = want["losses"].mean()
    _loss_close(loss.detach(), want, 64)
    _grad_close("dx", dx, want, BF16, 64)
    _grad_close("dw", dw[kept], want, BF16, 64)
    assert not bool(dw[256:512].any())


@pytest.mark.parametrize("v", [40, 5000])
def test_one_class_far_ahead(v):
    """Logits of hundreds: the exponentials neither overflow nor vanish into NaN; a row that is certain and right has no loss."""
    x, w, _, t = _inputs(140, 64, v, BF16, ignored=0.0)
    big = (x.detach() * 64).requires_grad_()
    t = (big.detach().float() @ w.detach().float().t()).argmax(-1)
    loss = px.linear_cross_entropy(big, w, t, reduction="none")
    dx, dw = torch.autograd.grad(loss.sum(), (big, w))
    want = _formula(big, w, None, t, 0.0, torch.ones(140, device="cuda"))
    _loss_close(loss.detach(), want, 64)
    assert bool(torch.isfinite(dx).all()) and bool(torch.isfinite(dw).all()) and float(loss.detach().min()) >= 0.0
    certain = want["losses"] < 1e-9      # the class is its own reference there, and the others add nothing: what is left is an exponential's rounding
    assert int(certain.sum()) > 10 and float(loss.detach()[certain].max()) <= 2.0 ** -21


def test_one_class():
    x, w, b, t = _inputs(140, 64, 1, FP16, FP16, ignored=0.0)
    loss = px.linear_cross_entropy(x, w, t, bias=b, label_smoothing=0.2, reduction="none")
    assert float(loss.abs().max()) <= 1e-5
    for g in torch.autograd.grad(loss.sum(), (x, w, b)):
        assert float(g.abs().max()) <= 1e-3


@pytest.mark.parametrize("size", [0.0, 1e-38, 1e-30, 1e30])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_gradients_of_any_size(size, dtype):
    """The scale of the loss's gradient does not reach the 16-bit values."""
    x, w, b, t = _inputs(150, 64, 90, dtype, torch.float32)
    each = torch.randn(150, device="cuda")
    one = torch.autograd.grad(px.linear_cross_entropy(x, w, t, bias=b, reduction="none"), b, each)[0]
    loss = px.linear_cross_entropy(x, w, t, bias=b, reduction="none")
    got = torch.autograd.grad(loss, b, each * size)[0]
    assert float((got.double() - one.double() * size).abs().max()) <= 1e-5 * float(one.abs().max()) * size + 1e-40


def test_a_gradient_that_is_not_finite_stays_in_its_row():
    x, w, _, t = _inputs(150, 64, 90, BF16, ignored=0.0)
    each = torch.ones(150, device="cuda")
    each[7] = math.inf
    dx, dw = torch.autograd.grad(px.linear_cross_entropy(x, w, t, reduction="none"), (x, w), each)
    ox, _ = torch.autograd.grad(px.linear_cross_entropy(x, w, t, reduction="none"), (x, w), torch.ones(150, device="cuda"))
    keep = torch.arange(150, device="cuda") != 7
    assert torch.equal(dx[keep], ox[keep]) and not bool(torch.isfinite(dx[7]).any()) and not bool(torch.isfinite(dw).any())


@pytest.mark.parametrize("rows,c,v", [(150, 64, 90), (150, 136, 300)])
@pytest.mark.parametrize("size", [math.inf, math.nan, 0.0])
def test_a_scale_that_is_not_finite(rows, c, v, size):
    """Rows that are ignored have gradients of zero all the same."""
    x, w, _, t = _inputs(rows, c, v, BF16)
    dx, dw = torch.autograd.grad(px.linear_cross_entropy(x, w, t) * size, (x, w))
    assert not bool(dx[t == -100].any())
    assert not bool(dx.any() or dw.any()) if size == 0.0 else not bool(torch.isfinite(dx[t != -100]).any())


@pytest.mark.parametrize("c,v", [(128, 16), (1024, 200)])
def test_offsets_beyond_32_bits(c, v):
    """Rows that begin beyond 2^31 elements of x, and beyond 2^32 bytes of its gradient."""
    rows = 2 ** 31 // c + 300
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.zeros(rows, c, dtype=BF16, device="cuda")
    at = torch.cat([torch.arange(200), torch.arange(rows - 200, rows)]).cuda()
    x[at] = torch.randn(400, c, generator=g, device="cuda").to(BF16)
    x.requires_grad_()
    w = (torch.randn(v, c, generator=g, device="cuda") / math.sqrt(c)).to(BF16).requires_grad_()
    t = torch.full((rows,), -100, device="cuda")
    t[at] = torch.randint(0, v, (400,), generator=g, device="cuda")
    each = px.linear_cross_entropy(x, w, t, reduction="none")
    dx, dw = torch.autograd.grad(each.sum(), (x, w))
    want = _formula(x.detach()[at], w, None, t[at], 0.0, torch.ones(400, device="cuda"))
    _loss_close(each.detach()[at], want, c)
    want_dx = {k: want[k] for k in ("dx", "dx_abs", "dx_most")}
    _grad_close("dx", dx[at], want_dx, BF16, c)
    _grad_close("dw", dw, want, BF16, c)
    assert int(torch.count_nonzero(dx)) == int(torch.count_nonzero(dx[at]))


def test_two_streams_at_once():
    sets = [_inputs(700, 128, v, BF16, BF16, seed=v) for v in (64, 3000)]
    call = lambda s: [(loss := px.linear_cross_entropy(s[0], s[1], s[3], bias=s[2])).detach(), *torch.autograd.grad(loss, s[:3])]  # noqa: E731
    want = [call(s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (s, st) in enumerate(zip(sets, streams)):
            with torch.cuda.stream(st):
                got[i].append(call(s))
    torch.cuda.synchronize()
    for w, many in zip(want, got):
        for g in many:
            assert all(torch.equal(a, b) for a, b in zip(w, g))


def test_layouts():
    """Rows inside larger rows, transposed weights, targets of other types and several batch axes."""
    x, w, b, t = _inputs(6 * 50, 64, 130, BF16, BF16, seed=5)
    want = px.linear_cross_entropy(x, w, t, bias=b, reduction="none").detach()
    dx, dw = torch.autograd.grad(px.linear_cross_entropy(x, w, t, bias=b), (x, w))
    wide = torch.full((300, 3, 64), math.nan, dtype=BF16, device="cuda")
    wide[:, 1] = x.detach()
    inside = wide[:, 1].requires_grad_()
    wide_w = torch.cat([w.detach(), w.detach()], 1)[:, :64].requires_grad_()
    odd = torch.zeros(130 * 64 + 1, dtype=BF16, device="cuda")[1:].view(130, 64).copy_(w.detach()).requires_grad_()
    turned = w.detach().t().contiguous().t().requires_grad_()
    for y in (inside, x.detach().view(6, 50, 64).requires_grad_(), x.detach().t().contiguous().t().requires_grad_()):
        for z in (wide_w, odd, turned):
            for tt in (t, t.int()):
                tt = tt.view(y.shape[:-1])
                loss = px.linear_cross_entropy(y, z, tt, bias=b, reduction="none")
                assert loss.shape == tt.shape and torch.equal(loss.detach().flatten(), want)
                gx, gw = torch.autograd.grad(px.linear_cross_entropy(y, z, tt, bias=b), (y, z))
                assert torch.equal(gx.reshape(300, 64), dx) and torch.equal(gw, dw)
    one = px.linear_cross_entropy(x.detach()[1], w, t[1], bias=b, reduction="none")
    assert one.shape == () and torch.equal(one.detach(), want[1])


def test_gradients_of_some_inputs():
    x, w, b, t = _inputs(150, 64, 90, BF16, BF16)
    full = torch.autograd.grad(px.linear_cross_entropy(x, w, t, bias=b), (x, w, b))
    for which in range(1, 8):
        leaves = [y.detach().requires_grad_(bool(which >> i & 1)) for i, y in enumerate((x, w, b))]
        loss = px.linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2])
        loss.backward()
        for y, f in zip(leaves, full):
            assert torch.equal(y.grad, f) if y.requires_grad else y.grad is None


@pytest.mark.parametrize("v", [90, 300])
@pytest.mark.parametrize("bias", [None, torch.float32])
def test_some_of_the_gradients(v, bias):
    """All inputs are leaves, and a call asks for some of their gradients."""
    x, w, b, t = _inputs(150, 136, v, BF16, bias)
    leaves = [y for y in (x, w, b) if y is not None]
    loss = px.linear_cross_entropy(x, w, t, bias=b)
    full = torch.autograd.grad(loss, leaves, retain_graph=True)
    for which in range(1, 1 << len(leaves)):
        some = [i for i in range(len(leaves)) if which >> i & 1]
        for i, g in zip(some, torch.autograd.grad(loss, [leaves[i] for i in some], retain_graph=True)):
            # db alone is added up by a kernel of its own, in another order
            assert torch.equal(g, full[i]) if i < 2 else torch.allclose(g, full[i], rtol=0, atol=2.0 ** -20 * float(full[i].abs().max()))


@pytest.mark.parametrize("v,smooth", [(24, 0.0), (700, 0.1)])
def test_against_differences(v, smooth):
    """Along a direction whose steps x's type holds exactly; the third derivative of the loss along it is below 40, so that the quotient is off by h^2 / 6 of that."""
    x, w, b, t = _inputs(60, 64, v, FP16, FP16, seed=9)
    x = (torch.round(x.detach() * 64) / 64).requires_grad_()
    d = torch.sign(torch.randn(60, 64, device="cuda")).to(FP16)
    loss = px.linear_cross_entropy(x, w, t, bias=b, label_smoothing=smooth)
    along = float((torch.autograd.grad(loss, x)[0].double() * d.double()).sum())
    h = 1 / 64
    far = [float(px.linear_cross_entropy((x + s * h * d).detach(), w, t, bias=b, label_smoothing=smooth)) for s in (1, -1)]
    # fp32 losses of about 5 are off by 1e-6, over 2 h; the gradient of 64 channels by its roundings
    assert abs((far[0] - far[1]) / (2 * h) - along) <= 40 * h * h / 6 + 1e-6 / h + 2e-3 * 64 ** 0.5


def test_streams_and_capture():
    x, w, b, t = _inputs(300, 128, 1000, BF16, BF16)
    want = [px.linear_cross_entropy(x, w, t, bias=b).detach(), *torch.autograd.grad(px.linear_cross_entropy(x, w, t, bias=b), (x, w, b))]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        loss = px.linear_cross_entropy(x, w, t, bias=b)
        got = [loss.detach(), *torch.autograd.grad(loss, (x, w, b))]
    side.synchronize()
    for a, z in zip(want, got):
        assert torch.equal(a, z)
    del loss
    fixed = [y.detach().clone().requires_grad_() for y in (x, w, b)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = px.linear_cross_entropy(fixed[0], fixed[1], t, bias=fixed[2])
        out = [loss.detach(), *torch.autograd.grad(loss, fixed)]
    for scale in (1.0, 0.5):
        with torch.no_grad():
            fixed[0].copy_(x * scale)
        graph.replay()
        y = (x.detach() * scale).requires_grad_()
        loss = px.linear_cross_entropy(y, w, t, bias=b)
        for a, z in zip(out, [loss.detach(), *torch.autograd.grad(loss, (y, w, b))]):
            assert torch.equal(a, z)


def test_refusals():
    x, w, b, t = _inputs(10, 64, 20, BF16, BF16)
    call = px.linear_cross_entropy
    for args, kw in (((x.float(), w.float(), t), {}), ((x, w.half(), t), {}), ((x, w[:, :32], t), {}), ((x[:, :12], w[:, :12], t), {}), ((x, w, t[:5]), {}),
                     ((x, w, t.float()), {}), ((x, w, t), {"bias": b[:5]}), ((x, w, t), {"bias": b.double()}), ((x, w, t), {"label_smoothing": 1.5}),
                     ((x, w, t), {"label_smoothing": math.nan}), ((x, w, t), {"reduction": "median"}), ((x, w, t.cpu()), {}), ((x, w.cpu(), t), {}), ((x.cpu(), w, t), {}),
                     ((x, w[:0], t), {})):
        with pytest.raises(RuntimeError):
            call(*args, **kw)
    loss = call(x, w, t, bias=b)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(loss, x, create_graph=True)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x.detach(), torch.ones_like(x))
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(dual, w, t)
