"""Entries of the learned bias that hide their offset: minus infinity, and what is minus infinity once it is multiplied by log2(e)."""
import math

import pytest
import torch

import protenix_b200 as px
from window_reference import check, reference


@pytest.mark.gpu
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("low", [-math.inf, torch.finfo(torch.float32).min])
@pytest.mark.parametrize("r", [3, 64])
def test_a_query_whose_offsets_are_all_hidden_sees_nothing(r, low, d):
    """Of three in front and itself a query sees those at offsets -3 and -2; the first two queries have none."""
    g = torch.Generator(device="cuda").manual_seed(d)
    q, k, v, grad = (torch.randn(2, 2, 200, d, generator=g, device="cuda").to(torch.bfloat16) for _ in range(4))
    bias = torch.randn(2, 2 * r + 1, generator=g, device="cuda")
    hidden = bias.clone()
    hidden[:, r - 1:r + 1] = low
    leaves = [t.clone().requires_grad_() for t in (q, k, v, hidden)]
    o = px.window_attention(*leaves[:3], (3, 0), rel_bias=leaves[3])
    dq, dk, dv, db = torch.autograd.grad(o, leaves, grad)
    assert not o[:, :, :2].any() and not dq[:, :, :2].any() and not db[:, r - 1:r + 1].any()
    # the same without the hidden offsets: keys moved two on, queries that see nothing left out
    moved = lambda t: torch.nn.functional.pad(t, (0, 0, 2, 0))[:, :, :200]
    at = torch.zeros(2, 2 * r + 1, device="cuda")
    at[:, r - 1:r + 1] = bias[:, r - 3:r - 1]      # offsets -3 and -2 as -1 and 0
    mask = (torch.arange(200, device="cuda") >= 2)[None].expand(2, 200)
    want = reference(q, moved(k), moved(v), 1, 0, 0, at, mask, grad=grad)
    check({"o": o.detach(), "dq": dq}, {x: want[x] for x in ("o", "dq")}, torch.bfloat16)
    back = lambda t: torch.nn.functional.pad(t[:, :, 2:], (0, 0, 0, 2))
    check({"dk": dk, "dv": dv}, {x: tuple(back(t) for t in want[x]) for x in ("dk", "dv")}, torch.bfloat16)
    value, bound, _ = want["drel_bias"]
    assert bool(((db[:, r - 3:r - 1].double() - value[:, r - 1:r + 1]).abs() <= bound[:, r - 1:r + 1]).all())
