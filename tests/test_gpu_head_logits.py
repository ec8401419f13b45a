"""The mean error of the logits of linear_cross_entropy: what the tensor core cuts off, and what is put back for it."""
import pytest
import torch

import protenix_b200 as px

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def _rows(kind, c, dtype, rows=8192):
    g = torch.Generator(device="cuda").manual_seed(c)
    if kind == "one sign":
        w = (torch.rand(c, generator=g, device="cuda") + 0.5) / c
        return ((torch.rand(rows, c, generator=g, device="cuda") + 0.5) * 20).to(dtype), w.to(dtype)
    w = torch.randn(c, generator=g, device="cuda")
    x = torch.randn(rows, c, generator=g, device="cuda") / c ** 0.5
    return (x * 3 + w * 20 / c if kind == "leaning" else x * 6).to(dtype), w.to(dtype)


def _mean(kind, c, dtype):
    """Of the relative error of logits above 9, from losses against a class whose logit is zero: log(1 + exp l); in units of 1e-8 (c / 16 + 1)."""
    x, w = _rows(kind, c, dtype)
    l = x.double() @ w.double()
    far = l > 9
    got = px.linear_cross_entropy(x, torch.stack([torch.zeros_like(w), w]), torch.zeros(len(x), dtype=torch.long, device="cuda"), reduction="none").double()
    assert int(far.sum()) > 300
    return float(((got - torch.nn.functional.softplus(l)) / l)[far].mean()) / (1e-8 * (c / 16 + 1))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("c", [512, 1024, 2048, 4096])
@pytest.mark.parametrize("kind", ["leaning", "noise"])
def test_what_the_cuts_take_is_put_back(kind, c, dtype):
    """Half of the smaller of the two corrections, 1.6: without one, or with twice as much, the mean is beyond it on either side."""
    assert abs(_mean(kind, c, dtype)) <= 0.8


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("c", [512, 1024, 2048, 4096])
def test_terms_of_one_sign(c, dtype):
    """They lose 1 to 4 (bf16) and 8 to 10 (fp16) of these units, and get 1.6 and 2.1 of them back: nothing becomes worse than the correction itself."""
    mean = _mean("one sign", c, dtype)
    assert -8.8 <= mean <= 2.1 if dtype == FP16 else -3.2 <= mean <= 1.6
