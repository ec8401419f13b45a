"""Backward passes of heads of 65 to 128, whose kernel for dK and dV takes all of an SM's tensor memory, on several streams at once."""
import pytest
import torch

import protenix_b200 as px
from protenix_b200 import ops


@pytest.mark.gpu
@pytest.mark.parametrize("d,other", [(128, 128), (72, 32), (128, 64)])
def test_same_bits_beside_one_another(d, other):
    g = torch.Generator(device="cuda").manual_seed(d)

    def inputs(size):
        rand = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16)
        return [rand(1, 8, 1500, size), rand(1, 2, 1500, size), rand(1, 2, 1500, size), rand(8, 65), rand(1, 8, 1500, size)]

    def step(q, k, v, bias, grad):
        leaves = [t.detach().clone().requires_grad_() for t in (q, k, v, bias)]
        o = px.window_attention(*leaves[:3], (300, 0), sinks=4, rel_bias=leaves[3])
        return (o.detach(), *torch.autograd.grad(o, leaves, grad))

    sets = [inputs(d), inputs(other)]
    want = [step(*x) for x in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    results = []
    for _ in range(6):
        for x, s in zip(sets, streams):
            with torch.cuda.stream(s):
                results.append(step(*x))
    torch.cuda.synchronize()
    ops.device_error_flags()
    for i, got in enumerate(results):
        assert all(torch.equal(a, b) for a, b in zip(got, want[i % 2]))
