"""Gradients of the relative position encoding that are not finite: they stay in their channel, and never come out as numbers in the columns of their pairs."""
import pytest
import torch

import protenix_b200 as px
from test_gpu_relpos import _features, _one_hot


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
@pytest.mark.parametrize("n", [97, 300])
def test_one_bad_gradient(n, bad, dtype):
    f = _features(n, 3)
    w = torch.randn(128, 139, device="cuda").requires_grad_()
    g = torch.Generator(device="cuda").manual_seed(n)
    dz = torch.randn(n, n, 128, generator=g, device="cuda").to(dtype)
    call = lambda grad: torch.autograd.grad(px.relative_position_encoding(w, **{k: v.cuda() for k, v in f.items()}, dtype=dtype), w, grad)[0]
    want = call(dz)
    i, j, c = n // 2, n // 3, 77
    dz[i, j, c] = bad
    got = call(dz)
    columns = _one_hot(f, 32, 2)[i, j].bool().cuda()
    assert not bool(torch.isfinite(got[c, columns]).any())
    others = torch.arange(128, device="cuda") != c
    assert torch.equal(got[others], want[others])
    if dtype == torch.float32:      # the form on the tensor cores multiplies it by the zeros of the other columns
        assert torch.equal(got[c, ~columns], want[c, ~columns])
        assert bool(got[c, columns].isnan().all()) if bad != bad else bool((got[c, columns] == bad).all())
