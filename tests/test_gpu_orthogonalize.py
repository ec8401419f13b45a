"""orthogonalize against the iteration in 64 bits."""
import math

import pytest
import torch

import protenix_b200 as px
from protenix_b200 import ops

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
ABC = (3.4445, -4.7750, 2.0315)


def _iterated(g, steps=5, coefficients=ABC, eps=1e-7):
    x = g.double()
    x = x / (torch.linalg.matrix_norm(x)[..., None, None] + eps)
    one = torch.eye(min(x.shape[-2:]), dtype=torch.float64, device=x.device)
    for a, b, c in [coefficients] * steps if isinstance(coefficients[0], float) else coefficients:
        if x.shape[-2] <= x.shape[-1]:
            s = x @ x.mT
            x = (a * one + b * s + c * (s @ s)) @ x
        else:
            s = x.mT @ x
            x = x @ (a * one + b * s + c * (s @ s))
    return x


def _close(got, want, noise=4e-6):
    """Operands of 22 bits: half a step of 2^-22 enters with each of three operands a step, and fp32 sums of up to some hundred terms of a sign lose as much
    again; noise as large in all directions grows by 3.45 a step in those whose singular values are small, 200 times over the steps that follow the
    first, and a share of the singular values that is sqrt(1 / 200) at most is that small where the spectrum is that of noise."""
    u = torch.finfo(got.dtype).eps / 2
    assert bool(torch.isfinite(want).all())
    off = (got.double() - want).flatten(-2).norm(dim=-1)
    size = want.flatten(-2).norm(dim=-1)
    assert bool((off <= (u + noise) * size + 2.0 ** -25 * math.sqrt(want.shape[-1] * want.shape[-2])).all()), float((off / size).max())


SIZES = [(1, 1, 1), (3, 1, 5), (2, 7, 3), (5, 16, 16), (2, 33, 130), (2, 130, 33), (7, 128, 128), (3, 129, 127), (4, 512, 128), (4, 128, 512), (2, 384, 1536), (1, 1000, 257), (1, 301, 299),
         (2, 100, 500), (1, 128, 1000), (1, 1001, 90), (1, 90, 2000), (1, 2048, 64), (60, 128, 500), (60, 510, 100), (100, 256, 128), (40, 1000, 33), (150, 100, 100)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,m,n", SIZES)
def test_against_64_bits(batch, m, n, dtype):
    g = torch.randn(batch, m, n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(m + n)).to(dtype)
    keep = g.clone()
    got = px.orthogonalize(g)
    ops.device_error_flags()
    assert got.dtype == dtype and got.shape == g.shape and torch.equal(g, keep)
    _close(got, _iterated(g))
    assert torch.equal(got, px.orthogonalize(g))
    # a matrix does not depend on what lies beside it; on how many there are it does in its last bits (the work is split otherwise)
    others = torch.randn_like(g)
    others[batch - 1] = g[batch - 1]
    assert torch.equal(got[batch - 1], px.orthogonalize(others)[batch - 1])
    _close(px.orthogonalize(g[batch - 1])[None], _iterated(g[batch - 1:]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,m,n", [(1, 256, 4096), (1, 4100, 200), (3, 1500, 140), (2, 129, 1025), (1, 77, 9000), (1, 9001, 131), (5, 300, 1500)])
def test_long_sides(batch, m, n, dtype):
    """The sum over the long side in parts."""
    g = torch.randn(batch, m, n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(m + n)).to(dtype)
    got = px.orthogonalize(g)
    ops.device_error_flags()
    _close(got, _iterated(g))
    assert torch.equal(got, px.orthogonalize(g))
    g[0, 3, 5] = math.nan
    assert bool(px.orthogonalize(g)[0].isnan().all())


@pytest.mark.parametrize("m,n", [(2048, 2048), (3000, 700), (1100, 4100)])
def test_large(m, n):
    """Tiles of pairs of CTAs, and whole rounds of them."""
    g = torch.randn(3, m, n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    _close(px.orthogonalize(g), _iterated(g), 1e-5)


@pytest.mark.parametrize("m,n", [(128, 128), (256, 700), (700, 256)])
def test_falling_spectra(m, n):
    """Eight strong directions and little else: what 16-bit iterates lose a third of.  Noise of 2^-22 grows by 200 beside directions that are there."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    g = torch.randn(m, 8, device="cuda", generator=gen) @ torch.randn(8, n, device="cuda", generator=gen)
    _close(px.orthogonalize(g[None]), _iterated(g[None]), 2e-4)
    g = g + 0.05 * torch.randn(m, n, device="cuda", generator=gen)
    _close(px.orthogonalize(g[None]), _iterated(g[None]), 2e-5)


def test_singular_values():
    """Between 0.7 and 1.2, for those above a hundredth of the norm."""
    u, _, v = torch.linalg.svd(torch.randn(96, 96, device="cuda", dtype=torch.float64))
    s = torch.linspace(1.0, 0.02, 96, device="cuda", dtype=torch.float64)
    s = s / s.norm()
    keep = s > 0.01
    got = torch.linalg.svdvals(px.orthogonalize((u * s @ v).float()).double())
    assert float(got[: int(keep.sum())].min()) > 0.65 and float(got.max()) < 1.25


@pytest.mark.parametrize("coefficients,steps", [([(1.5, -0.5, 0.0)] * 3, 0), ((1.875, -1.25, 0.375), 7), ([(8.287, -23.596, 17.300), (4.107, -2.948, 0.545), (3.949, -2.909, 0.552)], 1),
                                                ((1.0, 0.0, 0.0), 2), ((0.0, 0.0, 0.0), 1)])
def test_other_polynomials(coefficients, steps):
    g = torch.randn(2, 130, 200, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    got = px.orthogonalize(g, steps=steps, coefficients=coefficients)
    want = _iterated(g, steps, coefficients)
    _close(got, want, 2e-5)


@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e12, 1e30])
def test_size_does_not_matter(scale):
    g = torch.randn(2, 60, 90, device="cuda")
    _close(px.orthogonalize(g * scale, eps=0.0), _iterated((g * scale).double(), eps=0.0))
    _close(px.orthogonalize(g * scale), _iterated((g * scale).double()), 4e-6)


def test_zero_and_not_finite():
    """A zero matrix stays zero, one that is not finite gives NaN, and neither touches the others."""
    g = torch.randn(5, 130, 72, device="cuda")
    want = px.orthogonalize(g)
    g[1], g[2, 3, 4], g[4, 100, 0] = 0.0, math.nan, math.inf
    got = px.orthogonalize(g)
    assert not bool(got[1].any()) and bool(torch.isnan(got[[2, 4]]).all())
    assert torch.equal(got[[0, 3]], want[[0, 3]])
    assert bool(torch.isnan(px.orthogonalize(torch.zeros(4, 4, device="cuda"), eps=0.0)).all())


def test_layouts_and_empty():
    g = torch.randn(2, 3, 40, 64, device="cuda")
    want = px.orthogonalize(g)
    assert want.shape == g.shape
    assert torch.equal(px.orthogonalize(g.transpose(-1, -2).contiguous().transpose(-1, -2)), want)
    assert torch.equal(px.orthogonalize(g.transpose(0, 1)), want.transpose(0, 1))
    odd = torch.empty(g.numel() + 1, device="cuda")[1:].view(g.shape).copy_(g)
    assert torch.equal(px.orthogonalize(odd), want)
    half = torch.empty(g.numel() + 1, device="cuda", dtype=torch.float16)[1:].view(g.shape).copy_(g)
    assert torch.equal(px.orthogonalize(half), px.orthogonalize(g.half()))
    for shape in ((0, 4, 5), (2, 0, 5), (2, 4, 0)):
        assert px.orthogonalize(torch.zeros(shape, device="cuda")).shape == shape


@pytest.mark.parametrize("batch,m,n", [(34000, 64, 1000), (17000, 130, 1000)])
def test_offsets_beyond_32_bits(batch, m, n):
    g = torch.randn(batch, m, n, device="cuda", dtype=torch.bfloat16)
    got = px.orthogonalize(g)
    at = torch.tensor([0, batch // 2, batch - 1], device="cuda")
    _close(got[at], _iterated(g[at]))


def test_two_streams_at_once():
    sets = [torch.randn(s, device="cuda") for s in ((40, 128, 512), (3, 300, 400), (20, 100, 90))]
    want = [px.orthogonalize(g) for g in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], [], []]
    for _ in range(10):
        for i, (g, st) in enumerate(zip(sets, streams)):
            with torch.cuda.stream(st):
                got[i].append(px.orthogonalize(g))
    torch.cuda.synchronize()
    ops.device_error_flags()
    for w, many in zip(want, got):
        assert all(torch.equal(w, g) for g in many)


def test_many_steps():
    """More than the one launch of small matrices holds."""
    g = torch.randn(2, 30, 50, device="cuda")
    _close(px.orthogonalize(g, steps=40, coefficients=(1.5, -0.5, 0.0)), _iterated(g, 40, (1.5, -0.5, 0.0)), 2e-5)


def test_streams_and_capture():
    g = torch.randn(4, 150, 130, device="cuda").bfloat16()
    want = px.orthogonalize(g)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = px.orthogonalize(g)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = px.orthogonalize(g)
    for _ in range(2):
        g.copy_(torch.randn_like(g))
        graph.replay()
        assert torch.equal(out, px.orthogonalize(g))


def test_refusals():
    g = torch.randn(4, 8, device="cuda")
    for x, kw in ((g.cpu(), {}), (g.double(), {}), (g[0], {}), (g, {"steps": 0}), (g, {"coefficients": [(1.0,)]}), (g, {"coefficients": [(1.0, 2.0)]}), (g, {"coefficients": []}), (g, {"eps": -1.0}),
                  (g, {"eps": math.nan}), (g, {"coefficients": (math.inf, 0.0, 0.0)}), (g, {"steps": 1001}), (g.clone().requires_grad_(), {})):
        with pytest.raises(RuntimeError):
            px.orthogonalize(x, **kw)
    with torch.no_grad():
        px.orthogonalize(g.clone().requires_grad_())
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            px.orthogonalize(torch.autograd.forward_ad.make_dual(g, g))
