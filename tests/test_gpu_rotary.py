"""rotary_embedding against complex multiplication in 64 bits."""
import math

import pytest
import torch

import protenix_b200 as px

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _turned(x, positions, sections, base=10000.0, interleaved=False, per_axis=False, sign=1.0):
    p = sum(sections)
    e = [(i / s if per_axis else (i + sum(sections[:a])) / p, a) for a, s in enumerate(sections) for i in range(s)]
    ladder = torch.tensor([base ** -x for x, _ in e], dtype=torch.float64, device=x.device)
    angle = sign * positions.double()[..., [a for _, a in e]] * ladder
    circle = torch.polar(torch.ones_like(angle), angle).unsqueeze(-3)
    y = x.detach().double()
    pairs = y[..., : 2 * p]
    pairs = pairs.unflatten(-1, (p, 2)) if interleaved else torch.stack(pairs.split(p, -1), -1)
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * circle)
    z = z.flatten(-2) if interleaved else torch.cat([z[..., 0], z[..., 1]], -1)
    size = pairs.abs().sum(-1, keepdim=True).expand_as(pairs)      # |u| + |v|
    size = size.flatten(-2) if interleaved else torch.cat([size[..., 0], size[..., 1]], -1)
    return torch.cat([z, y[..., 2 * p:]], -1), torch.cat([size, torch.zeros_like(y[..., 2 * p:])], -1)


def _close(got, x, positions, sections, far=0, **kw):
    """Sine and cosine are off by two steps and by what a turn in 31 bits leaves of the angle, five 2^-24 in all, products and sum by half a step each; `far`: what
    64-bit angles of the comparison itself lose."""
    want, size = _turned(x, positions, sections, **kw)
    u = torch.finfo(got.dtype).eps / 2
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 0.0
    assert bool(((got.detach().double() - want).abs() <= u * want.abs() + (8 * 2.0 ** -24 + far) * size * (1 + u) + tiny).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("per_axis", [False, True])
@pytest.mark.parametrize("batch,n,h,hk,d,sections", [(1, 1, 1, 1, 2, (1,)), (1, 97, 4, 4, 32, (16,)), (2, 50, 6, 2, 40, (5, 8, 7)), (3, 33, 3, 1, 24, (3, 3)), (2, 129, 5, 5, 34, (4, 0, 9)),
                                                     (1, 300, 16, 4, 128, (16, 24, 24)), (2, 7, 2, 2, 256, (100, 28)), (2, 64, 2, 1, 26, (13,)), (1, 20, 1, 1, 600, (256,))])
def test_against_64_bits(batch, n, h, hk, d, sections, interleaved, per_axis, dtype):
    g = torch.Generator(device="cuda").manual_seed(n)
    q, k = (torch.randn(batch, x, n, d, generator=g, device="cuda").to(dtype).requires_grad_() for x in (h, hk))
    at = torch.randint(-1000, 1000, (batch, n, len(sections)), generator=g, device="cuda")
    kw = {"interleaved": interleaved, "per_axis": per_axis}
    got = px.rotary_embedding(q, k, at, sections=sections, **kw)
    up = [torch.randn(y.shape, generator=g, device="cuda").to(dtype) for y in got]
    grads = torch.autograd.grad(got, (q, k), up)
    for y, x, dx, dy in zip(got, (q, k), grads, up):
        assert y.dtype == dtype and y.shape == x.shape
        _close(y, x, at, sections, **kw)
        _close(dx, dy, at, sections, sign=-1.0, **kw)
    assert torch.equal(px.rotary_embedding(q.detach(), None, at, sections=sections, **kw), got[0].detach())


@pytest.mark.parametrize("far", [10 ** 6, -10 ** 9, 2 ** 40])
def test_far_positions(far):
    """Exact modulo a turn: far positions give what the same offsets give near zero, turned by a constant."""
    x = torch.randn(1, 2, 64, 32, device="cuda")
    at = torch.arange(64, device="cuda")[:, None] + far
    got = px.rotary_embedding(x, None, at)
    _close(got, x, at[None], (16,), far=abs(far) * 2.0 ** -52 if abs(far) < 2 ** 31 else 2.0)
    back = px.rotary_embedding(got, None, -at)
    assert float((back - x).abs().max()) <= 16 * 2.0 ** -24 * float(x.abs().max()) * 2
    # logits depend on the offset alone
    near = px.rotary_embedding(x, None, at - far)
    a, b = ((t[0, 0].double() @ t[0, 1].double().t()) for t in (got, near))
    assert float((a - b).abs().max()) <= 32 * 2 * 8 * 2.0 ** -24 * float(x.abs().max()) ** 2 * 4


def test_more_rows_than_one_thread_each():
    """Large enough for the form in which a thread takes four heads; a number of heads that four does not divide."""
    q, k = torch.randn(2, 2100, 13, 128, device="cuda").bfloat16().transpose(1, 2), torch.randn(2, 5, 2100, 128, device="cuda").bfloat16()
    at = torch.randint(0, 3000, (2, 2100, 2), device="cuda")
    for x, y in zip((q, k), px.rotary_embedding(q, k, at, sections=(30, 10), interleaved=True)):
        _close(y, x, at, (30, 10), interleaved=True)
        assert y.stride()[1:] == x.stride()[1:]


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(dtype):
    """Heads inside the rows of a projection, odd strides and addresses, broadcast samples, several batch axes, other integer types."""
    n, h, hk, d = 45, 4, 2, 32
    qkv = torch.randn(3, n, h + 2 * hk, d, device="cuda").to(dtype)
    q, k, _ = (t.transpose(1, 2) for t in qkv.split([h, hk, hk], 2))
    at = torch.randint(0, 100, (n, 2), device="cuda")
    want = px.rotary_embedding(q.contiguous(), k.contiguous(), at, sections=(10, 6))
    _close(want[0], q, at[None], (10, 6))
    odd = torch.empty(3 * n * (h * d + 1) + 1, dtype=dtype, device="cuda")[1:].view(3, n, h * d + 1)[..., 1:].unflatten(-1, (h, d)).copy_(q.transpose(1, 2)).transpose(1, 2)
    for qq in (q, odd, q.transpose(-1, -2).contiguous().transpose(-1, -2)):
        for p in (at, at.int(), at[None].expand(3, n, 2), at.short()[None], torch.stack([at[:, 0], at[:, 1]], 0).t()):
            got = px.rotary_embedding(qq, k, p, sections=(10, 6))
            for a, b in zip(got, want):
                assert torch.equal(a, b)
    got = px.rotary_embedding(q, k, at, sections=(10, 6))
    assert got[0].transpose(1, 2).is_contiguous()      # like q: heads inside the rows
    one = q[:1].expand(3, h, n, d)
    assert torch.equal(px.rotary_embedding(one, None, at, sections=(10, 6)), want[0][:1].expand(3, h, n, d))
    here = torch.full((1, 2), 7, device="cuda")      # one place for all rows
    assert torch.equal(px.rotary_embedding(q, None, here, sections=(10, 6)), px.rotary_embedding(q, None, here.expand(n, 2).contiguous(), sections=(10, 6)))
    each = torch.randint(0, 50, (3, n, 2), device="cuda")
    want3 = px.rotary_embedding(q, k, each, sections=(10, 6))
    for i in range(3):
        assert torch.equal(px.rotary_embedding(q[i:i + 1], None, each[i], sections=(10, 6)), want3[0][i:i + 1])
    six = px.rotary_embedding(q[None].expand(2, 3, h, n, d), None, each.expand(2, 3, n, 2), sections=(10, 6))
    assert torch.equal(six, want3[0].expand(2, 3, h, n, d))
    mixed = px.rotary_embedding(q[None].expand(2, 3, h, n, d), None, each[:1, :, :].unsqueeze(1).expand(1, 1, n, 2), sections=(10, 6))
    assert torch.equal(mixed[1], px.rotary_embedding(q, None, each[0], sections=(10, 6)))
    five = px.rotary_embedding(q[None], k[None], at.expand(1, 3, n, 2), sections=(10, 6))
    assert five[0].shape == (1, 3, h, n, d) and torch.equal(five[0][0], want[0]) and torch.equal(five[1][0], want[1])
    three = px.rotary_embedding(q[0], k[0], at, sections=(10, 6))
    assert torch.equal(three[0], want[0][0])


def test_untouched_channels_and_special_values():
    """Channels behind the pairs keep every bit; an infinity or a NaN stays in its pair."""
    x = torch.randn(1, 2, 10, 24, device="cuda")
    x[0, 0, 3, 20], x[0, 1, 4, 2], x[0, 0, 5, 1] = math.nan, math.inf, math.nan
    at = torch.arange(10, device="cuda")[:, None] + 1
    y = px.rotary_embedding(x, None, at, sections=(8,))
    assert torch.equal(y[..., 16:].nan_to_num(7.0), x[..., 16:].nan_to_num(7.0))
    bad = ~torch.isfinite(y[..., :16])
    want = torch.zeros_like(bad)
    want[0, 1, 4, [2, 10]] = want[0, 0, 5, [1, 9]] = True
    assert torch.equal(bad, want)


def test_empty():
    for shape in ((0, 2, 5, 16), (2, 2, 0, 16)):
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        y = px.rotary_embedding(x, None, torch.zeros(shape[0], shape[2], 1, dtype=torch.long, device="cuda"))
        assert y.shape == shape and torch.autograd.grad(y.sum(), x)[0].shape == shape


def test_gradients():
    """Of q alone, of k alone, of the gradient, and by differences (the operator is linear)."""
    q, k = (torch.randn(1, 2, 9, 16, device="cuda", requires_grad=True) for _ in range(2))
    at = torch.arange(9, device="cuda")[:, None]
    for which in range(3):
        yq, yk = px.rotary_embedding(q, k, at)
        up = torch.randn_like(yq)
        loss = (yq * up).sum() * (which != 1) + (yk * up).sum() * (which != 0) if which == 2 else ((yq, yk)[which] * up).sum()
        grads = torch.autograd.grad(loss, (q, k), allow_unused=True)
        want = px.rotary_embedding(up, None, -at)
        for i, g in enumerate(grads):
            if which in (i, 2):      # the angle is cut to 32 bits on its way down, on the other side for the negated position
                assert float((g - want).abs().max()) <= (8 * 2.0 ** -24 + math.pi * 2.0 ** -31) * 2 * float(up.abs().max())
            else:
                assert g is None or not bool(g.any())
    d, up = torch.randn_like(q), torch.randn_like(q)
    f = lambda x: float((px.rotary_embedding(x.detach(), None, at).double() * up.double()).sum())  # noqa: E731
    g = torch.autograd.grad(px.rotary_embedding(q, None, at), q, up)[0]
    assert abs((f(q + d) - f(q - d)) / 2 - float((g.double() * d.double()).sum())) <= 1e-4
    up = up.requires_grad_()
    g = torch.autograd.grad(px.rotary_embedding(q, None, at), q, up, create_graph=True)[0]
    assert torch.equal(torch.autograd.grad(g, up, d)[0], px.rotary_embedding(d, None, at))
    only = px.rotary_embedding(q, k.detach(), at)
    assert torch.autograd.grad(only[0].sum(), q)[0].shape == q.shape


def test_one_of_two_gradients():
    q, k = (torch.randn(2, 3, 50, 32, device="cuda", requires_grad=True) for _ in range(2))
    out = px.rotary_embedding(q, k, torch.arange(50, device="cuda")[:, None])
    full = torch.autograd.grad(out, (q, k), out, retain_graph=True)
    assert torch.equal(torch.autograd.grad(out, q, out, retain_graph=True)[0], full[0])
    assert torch.equal(torch.autograd.grad(out, k, out, retain_graph=True)[0], full[1])


def test_offsets_beyond_32_bits():
    """Rows that begin beyond 2^31 elements of q, and beyond 2^32 bytes."""
    n, h, d = 2 ** 31 // (16 * 128) + 700, 16, 128
    q = torch.zeros(1, n, h, d, dtype=torch.bfloat16, device="cuda").transpose(1, 2)
    rows = torch.tensor([0, 1, n // 2, n - 600, n - 1], device="cuda")
    q[:, :, rows] = torch.randn(1, h, 5, d, device="cuda").to(torch.bfloat16)
    got = px.rotary_embedding(q, None, torch.arange(n, device="cuda")[:, None])
    _close(got[:, :, rows], q[:, :, rows], rows[None, :, None], (64,), far=n * 2.0 ** -52)
    assert int(torch.count_nonzero(got)) == int(torch.count_nonzero(got[:, :, rows]))


def test_streams_and_capture():
    q, k = torch.randn(2, 4, 70, 64, device="cuda").half(), torch.randn(2, 2, 70, 64, device="cuda").half()
    at = torch.randint(0, 500, (2, 70, 1), device="cuda")
    want = px.rotary_embedding(q, k, at)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = px.rotary_embedding(q, k, at)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = px.rotary_embedding(q, k, at)
    for step in (0, 11):
        at += step
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, px.rotary_embedding(q, k, at)))


def test_refusals():
    q, k = torch.randn(2, 4, 10, 32, device="cuda"), torch.randn(2, 2, 10, 32, device="cuda")
    at = torch.zeros(2, 10, 2, dtype=torch.long, device="cuda")
    ok = {"sections": (8, 8)}
    px.rotary_embedding(q, k, at, **ok)
    for args, kw in (((q, k, at), {}), ((q, k, at), {"sections": (9, 8)}), ((q, k, at), {"sections": (16,)}), ((q, k, at), {"sections": (-1, 8)}),
                     ((q, k, at), {"sections": (0, 0)}), ((q, k, at.float()), ok), ((q, k, at[:, :5]), ok), ((q, k, at.cpu()), ok), ((q, k.half(), at), ok),
                     ((q, k[:1], at), ok), ((q, k[..., :16], at), ok), ((q.double(), None, at), ok), ((q[0, 0], None, at), ok), ((q.cpu(), None, at), ok),
                     ((q, k, at), {**ok, "base": 0.5}), ((q, k, at), {**ok, "base": math.nan}), ((q, k, at), {**ok, "base": math.inf}), ((q, k, at[0, 0, 0]), ok)):
        with pytest.raises(RuntimeError):
            px.rotary_embedding(*args, **kw)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(q, torch.ones_like(q))
        with pytest.raises(RuntimeError, match="forward-mode"):
            px.rotary_embedding(dual, k, at, **ok)
