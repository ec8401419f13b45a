"""A query of NaN that sees keys gives NaN to what it touches, whether there is a mask or not."""
import pytest
import torch

import protenix_b200 as px
from protenix_b200 import ops


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("masked", [False, True])
def test_a_query_of_nan_is_not_one_that_sees_nothing(masked, d, dtype):
    g = torch.Generator(device="cuda").manual_seed(d)
    q, k, v, grad = (torch.randn(1, 2, 260, d, generator=g, device="cuda").to(dtype) for _ in range(4))
    q[0, 1, 140] = float("nan")
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    mask = torch.ones(1, 260, dtype=torch.bool, device="cuda") if masked else None
    o = px.window_attention(*leaves, (3, 2), mask=mask)
    dq, dk, dv = torch.autograd.grad(o, leaves, grad)
    ops.device_error_flags()
    assert bool(o[0, 1, 140].isnan().all()) and bool(dq[0, 1, 140].isnan().all())
    for t in (dk, dv):
        assert bool(t[0, 1, 137:143].isnan().all()) and bool(torch.isfinite(t[0, 0]).all())
