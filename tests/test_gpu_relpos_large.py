"""The relative position encoding at lengths of real use: more strips than warps, rings that turn, accumulators that change.

Weights and gradients are small whole numbers, so that every sum on the way is a number of fp32 (and of a 16-bit z): the results have to be equal, whatever the order."""
import pytest
import torch

import protenix_b200 as px
from test_gpu_relpos import DTYPES, _features, _one_hot


def _check(n, c, r, s, lead, dtype, wild=False):
    f = _features(n, n + c, lead, wild)
    g = torch.Generator(device="cuda").manual_seed(n)
    whole = lambda top, *shape: torch.randint(-top, top + 1, shape, generator=g, device="cuda")
    w = whole(9, c, 4 * r + 2 * s + 7).float().requires_grad_()
    z = px.relative_position_encoding(w, **{k: v.cuda() for k, v in f.items()}, r_max=r, s_max=s, dtype=dtype)
    dz = whole(3, *lead, n, n, c).to(dtype)
    dw, = torch.autograd.grad(z, w, dz)
    plain = px.relative_position_encoding(w.detach(), **{k: v.cuda() for k, v in f.items()}, r_max=r, s_max=s, dtype=dtype)
    assert torch.equal(plain, z.detach())
    want = torch.zeros(dw.shape, dtype=torch.float64, device="cuda")
    z, dz = z.detach().reshape(-1, n, n, c), dz.reshape(-1, n, n, c)
    for b, row in enumerate(torch.stack([f[k].reshape(-1, n) for k in f], 1).cuda()):
        sample = dict(zip(f, row))
        one = _one_hot(sample, r, s).reshape(n, n, -1)
        for i in range(0, n, 64):
            rows = one[i:i + 64]
            assert torch.equal(z[b, i:i + 64].double(), rows @ w.detach().double().t())
            want += dz[b, i:i + 64].double().reshape(-1, c).t() @ rows.reshape(-1, rows.shape[-1])
    assert float(want.abs().max()) < 2 ** 24
    assert torch.equal(dw.double(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("n,c,lead", [(193, 128, ()), (401, 128, ()), (701, 128, ()), (401, 136, (2,)), (300, 24, (3,)), (333, 384, ())])
def test_equal_to_the_one_hot_form(n, c, lead, dtype):
    _check(n, c, 32, 2, lead, DTYPES[dtype])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_wild_features_and_the_largest_tables(dtype):
    _check(401, 128, 32, 2, (), DTYPES[dtype], wild=True)
    _check(257, 64, 92, 2, (), DTYPES[dtype])


@pytest.mark.gpu
def test_sums_of_random_numbers():
    """fp32 sums in a chain of a few thousand steps at most: each within 2^-24 of the running sum, which is at most the sum of magnitudes; 4096 such steps are the
    bound of an entry.  Of the whole: rounded steps do not all err one way (1e-6 as at small sizes); for 16-bit gradients the 32 steps of a
    group of 512 pairs cut off, towards zero, by at most 2^-23 of a running sum that is smaller than the group's in the mean."""
    n, c = 601, 128
    f = _features(n, 5)
    g = torch.Generator(device="cuda").manual_seed(7)
    w = torch.randn(c, 139, generator=g, device="cuda").requires_grad_()
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        dz = torch.randn(n, n, c, generator=g, device="cuda").to(dtype)
        dw, = torch.autograd.grad(px.relative_position_encoding(w, **{k: v.cuda() for k, v in f.items()}, dtype=dtype), w, dz)
        one = _one_hot({k: v.cuda() for k, v in f.items()}, 32, 2).reshape(n * n, -1)
        want, size = dz.double().reshape(-1, c).t() @ one, dz.double().abs().reshape(-1, c).t() @ one
        assert bool(((dw.double() - want).abs() <= 2.0 ** -12 * size).all())
        assert float((dw.double() - want).norm()) <= (1e-6 if dtype == torch.float32 else 32 * 2.0 ** -23) * float(want.norm())
