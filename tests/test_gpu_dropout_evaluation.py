"""dropout_add in evaluation refuses what it refuses in training."""
import pytest
import torch

import protenix_b200 as px


@pytest.mark.gpu
@pytest.mark.parametrize("training", [True, False])
def test_refusals(training):
    x = torch.zeros(4, 8, device="cuda")
    call = lambda residual=None, x=x, p=0.1, seed=3, **kw: px.dropout_add(residual, x, p, seed, training=training, **kw)
    state = lambda *v, **kw: torch.zeros(*v, dtype=torch.long, **kw)
    for match, kw in [("probability", {"p": 2.0}), ("probability", {"p": -0.1}), ("probability", {"p": float("nan")}), ("seed", {"seed": -1}), ("seed", {"seed": 0.5}),
                      ("seed", {"seed": 1 << 63}), ("offset", {"offset": -1}), ("holds the offset", {"seed": state(2, device="cuda"), "offset": 1}),
                      ("seed", {"seed": state(3, device="cuda")}), ("seed", {"seed": state(2)}), ("out of range", {"shared_dim": 2}), ("match", {"residual": x[:2]}),
                      ("match", {"residual": x.half()}), ("match", {"residual": x[:1]}), ("float", {"x": x.double()}), ("CUDA", {"residual": x.cpu()})]:
        with pytest.raises(RuntimeError, match=match):
            call(**kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_evaluation_is_the_sum_alone(dtype):
    residual, x = (torch.randn(5, 7, 8, device="cuda").to(dtype).requires_grad_() for _ in range(2))
    for kw in ({}, {"shared_dim": -2}, {"offset": 4}):
        out = px.dropout_add(residual, x, 0.4, 3, training=False, **kw)
        assert torch.equal(out, residual + x)
        assert all(bool((g == 1).all()) for g in torch.autograd.grad(out.sum(), (residual, x)))
    alone = px.dropout_add(None, x, 0.4, torch.zeros(2, dtype=torch.long, device="cuda"), training=False)
    assert torch.equal(alone, x) and alone.data_ptr() != x.data_ptr()
