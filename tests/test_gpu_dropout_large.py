"""dropout_add beyond one turn of its grid: 148 SMs x 32 blocks x 256 threads take 9.7 million 16-bit or 4.8 million fp32 elements at a time."""
import numpy as np
import pytest
import torch

import protenix_b200 as px
from philox import LOW, SHIFT, keep, philox
from test_gpu_counter_dropout import _check, _inputs

SEED, OFFSET, P = (5 << 40) + 11, (1 << 33) + 2, 0.3


@pytest.mark.gpu
@pytest.mark.parametrize("shape,dim,dtype", [((9_800_003,), None, torch.bfloat16), ((9_800_003,), None, torch.float16), ((4_900_001,), None, torch.float32),
                                             ((2, 5, 2_600_008), 1, torch.bfloat16), ((2, 5, 1_300_004), 1, torch.float32), ((2, 6, 400_001), 1, torch.float16)])
def test_second_turn_of_the_grid(shape, dim, dtype):
    residual, x, grad = _inputs(shape, dtype)
    mask = keep(shape, P, SEED, OFFSET, dim)
    xr, rr = x.clone().requires_grad_(), residual.clone().requires_grad_()
    out = px.dropout_add(rr, xr, P, SEED, offset=OFFSET, shared_dim=dim)
    _check(out.detach(), residual, x, mask, P, dtype)
    dr, dx = torch.autograd.grad(out, (rr, xr), grad)
    assert torch.equal(dr, grad)
    _check(dx, None, grad, mask, P, dtype)


def _keep_from(place, count):
    """Truth values of `count` places from `place` (a multiple of four) on."""
    block = np.arange(count // 4, dtype=np.uint64) + np.uint64(place // 4)
    words = philox([block & LOW, block >> SHIFT, np.full_like(block, OFFSET & 0xFFFFFFFF), np.full_like(block, OFFSET >> 32)], (SEED & 0xFFFFFFFF, SEED >> 32))
    return np.stack(words, -1).reshape(-1) >= np.uint64(round(P * 2 ** 32))


@pytest.mark.gpu
@pytest.mark.parametrize("shared", [False, True])
def test_places_beyond_32_bits(shared):
    """More than 2^32 elements: the last ones drop by their own places."""
    tail = 4096
    shape = (2, 3, (1 << 32) // 6 // 8 * 8 + 2 * tail) if shared else ((1 << 32) + tail,)
    x = torch.ones(shape, dtype=torch.bfloat16, device="cuda")
    out = px.dropout_add(None, x, P, SEED, offset=OFFSET, shared_dim=1 if shared else None)
    assert x.numel() > 1 << 32
    kept = torch.tensor(1 / (1 - P)).to(torch.bfloat16)
    inner = shape[-1]
    for row, first, place in [((1, 2), inner - tail, 2 * inner - tail), ((0, 1), 0, 0)] if shared else [((), (1 << 32), 1 << 32), ((), 0, 0)]:
        want = torch.from_numpy(_keep_from(place, tail)).cuda()
        assert torch.equal(out[row][first:first + tail], torch.where(want, kept.cuda(), torch.zeros_like(kept).cuda()))
    del x, out
    torch.cuda.empty_cache()
