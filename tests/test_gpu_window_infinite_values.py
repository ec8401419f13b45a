"""What visible keys hold reaches the output as it is: infinities too, and the largest finite numbers without becoming one."""
import pytest
import torch

import protenix_b200 as px

DTYPES = [torch.bfloat16, torch.float16]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [24, 64, 128])
def test_infinite_values_stay_infinite(d, dtype):
    g = torch.Generator(device="cuda").manual_seed(d)
    q, k, v = (torch.randn(1, 2, 200, d, generator=g, device="cuda").to(dtype) for _ in range(3))
    v[0, 0, 130] = float("inf")
    v[0, 1, 70, 1] = -float("inf")
    o = px.window_attention(q, k, v, 0)                     # each query sees its own key alone
    assert bool((o[0, 0, 130] == float("inf")).all()) and float(o[0, 1, 70, 1]) == -float("inf")
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    kept = px.window_attention(*leaves, 0)                  # with what the backward pass asks for
    assert bool((kept[0, 0, 130] == float("inf")).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [32, 64, 128])
def test_means_of_the_largest_values_stay_finite(d, dtype):
    """A mean of equal numbers is that number.  The rounded weights add up to one within half a step u, the result is rounded: two of them at most, and no infinity
    (65504 (1 + u) is nearer to 65536 than to 65504).  bf16 has the range of the fp32 sums, which the weights before their division make 2^8 n times
    as large as the values: 2^100 is well inside."""
    g = torch.Generator(device="cuda").manual_seed(d)
    q, k = (torch.randn(2, 2, 300, d, generator=g, device="cuda").to(dtype) for _ in range(2))
    top = 65504.0 if dtype == torch.float16 else 2.0 ** 100
    v = torch.full((2, 2, 300, d), top, dtype=dtype, device="cuda")
    for sign in (1, -1):
        o = px.window_attention(q, k, sign * v, 40)
        assert bool(torch.isfinite(o).all())
        assert bool(((o.double() - sign * top).abs() <= 2.02 * torch.finfo(dtype).eps / 2 * top).all())
