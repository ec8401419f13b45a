"""The angles of rotary_embedding at positions of any size, against decimal arithmetic with 90 digits."""
import math
from decimal import Decimal, getcontext

import pytest
import torch

import protenix_b200 as px

pytestmark = pytest.mark.gpu
getcontext().prec = 90
TURN = Decimal("0.159154943091895335768883763372514362034459645740456448747667344058896797634226535090113802766253085956")      # 1 / 2 pi
PLACES = [0, 1, -1, 2 ** 20 + 1, 2 ** 31 + 5, 2 ** 40 + 3, -(2 ** 40) - 7, 2 ** 52 + 11, -(2 ** 57) + 1, 2 ** 62 + 12345, 2 ** 63 - 1, -(2 ** 63)]
# Sine and cosine are off by two steps and by what a turn in 31 bits leaves of the angle, five 2^-24 in all, a speed of 88 bits leaves 1.7 at 2^63; the product and
# the sum lose half a step each, of numbers up to |u| + |v|.
BOUND = 9 * 2.0 ** -24


def _angles(places, sections, base, per_axis):
    """[place][pair], reduced to a turn before they become 64-bit numbers."""
    exponents = [Decimal(i) / n for n in sections for i in range(n)] if per_axis else [Decimal(j) / sum(sections) for j in range(sum(sections))]
    speeds = [TURN * (-(e * Decimal(base).ln())).exp() for e in exponents]
    turned = [[p * s for s in speeds] for p in places]
    return torch.tensor([[float(t - t.to_integral_value()) for t in row] for row in turned], dtype=torch.float64, device="cuda") * (2 * math.pi)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("base", [10000.0, 2.0, 1.0, 500000.0, 1e30])
@pytest.mark.parametrize("sections,per_axis", [((64,), False), ((3, 0, 5), True), ((16, 24, 24), False), ((256,), False), ((1,), False), ((255, 1), True)])
def test_any_position(sections, per_axis, base, interleaved):
    pairs = sum(sections)
    x = torch.randn(1, 2, len(PLACES), 2 * pairs, device="cuda", generator=torch.Generator(device="cuda").manual_seed(pairs))
    at = torch.tensor(PLACES, device="cuda")[:, None].expand(-1, len(sections))
    got = px.rotary_embedding(x, None, at, sections=sections, base=base, interleaved=interleaved, per_axis=per_axis).double()
    split = (lambda t: (t[..., ::2], t[..., 1::2])) if interleaved else (lambda t: t.split(pairs, -1))
    angle = _angles(PLACES, sections, base, per_axis)
    (u, v), (gu, gv) = split(x.double()), split(got)
    bound = BOUND * (u.abs() + v.abs())
    assert bool(((gu - (u * angle.cos() - v * angle.sin())).abs() <= bound).all())
    assert bool(((gv - (v * angle.cos() + u * angle.sin())).abs() <= bound).all())


@pytest.mark.parametrize("far", [2 ** 45, -(2 ** 62), 2 ** 63 - 100])
def test_gradients_of_far_positions(far):
    x = torch.randn(1, 2, 40, 32, device="cuda", requires_grad=True)
    at = torch.arange(40, device="cuda")[:, None] + far
    up = torch.randn_like(x)
    grad = torch.autograd.grad(px.rotary_embedding(x, None, at), x, up)[0].double()
    angle = _angles([far + i for i in range(40)], (16,), 10000.0, False)
    u, v = up.double().split(16, -1)
    want = torch.cat([u * angle.cos() + v * angle.sin(), v * angle.cos() - u * angle.sin()], -1)
    assert bool(((grad - want).abs() <= BOUND * (u.abs() + v.abs()).repeat(1, 1, 1, 2)).all())
