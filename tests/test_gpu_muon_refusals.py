"""What Muon refuses, it refuses before anything has changed."""
import math

import pytest
import torch

import protenix_b200 as px

pytestmark = pytest.mark.gpu


def _good(seed):
    p = torch.nn.Parameter(torch.randn(8, 12, device="cuda"))
    p.grad = torch.randn(8, 12, device="cuda")
    return p


def _sparse():
    p = torch.nn.Parameter(torch.randn(6, 5, device="cuda"))
    p.grad = torch.randn(6, 5, device="cuda").to_sparse()
    return p


def _of(make):
    p = torch.nn.Parameter(make())
    p.grad = torch.ones_like(p)
    return p


@pytest.mark.parametrize("bad", [
    _sparse, lambda: _of(lambda: torch.randn(6, 5)), lambda: _of(lambda: torch.randn(6, 5, device="cuda", dtype=torch.float64)),
    lambda: _of(lambda: torch.zeros(65536, 1, 1, device="cuda")), lambda: _of(lambda: torch.zeros((1 << 20) + 1, 1, device="cuda")),
    lambda: _of(lambda: torch.zeros(0, (1 << 20) + 1, device="cuda"))])
@pytest.mark.parametrize("apart", [False, True])
def test_parameters(bad, apart):
    """Beside good ones of the same group, or of a group before it, that have been stepped already or not."""
    first, good, p = _good(1), _good(2), bad()
    opt = px.Muon([{"params": [first]}, {"params": [good]}] if apart else [first, good], weight_decay=0.1)
    opt.step()
    opt.add_param_group({"params": [p]})
    if not apart:
        opt.param_groups[0]["params"].append(opt.param_groups.pop()["params"][0])
    before = [t.detach().clone() for t in (first, good, p)]
    held = [opt.state[t]["momentum_buffer"].clone() for t in (first, good)]
    with pytest.raises(RuntimeError):
        opt.step()
    assert all(torch.equal(t.detach(), b) for t, b in zip((first, good, p), before))
    assert all(torch.equal(opt.state[t]["momentum_buffer"], b) for t, b in zip((first, good), held))
    assert "momentum_buffer" not in opt.state.get(p, {})


@pytest.mark.parametrize("changed", [{"steps": 0}, {"steps": 1001}, {"coefficients": (1.0, 2.0)}, {"coefficients": [(1.0,)]}, {"coefficients": []}, {"eps": -1.0}, {"eps": math.nan},
                                     {"coefficients": (math.inf, 0.0, 0.0)}])
def test_polynomials(changed):
    p, q = _good(1), _good(2)
    opt = px.Muon([{"params": [p]}, {"params": [q], **changed}])
    before = p.detach().clone(), q.detach().clone()
    with pytest.raises(RuntimeError):
        opt.step()
    assert torch.equal(p.detach(), before[0]) and torch.equal(q.detach(), before[1]) and not opt.state


def test_parameters_that_move_later():
    """A model may go to the device after its optimiser was made."""
    model = torch.nn.Linear(12, 8, bias=False)
    opt = px.Muon(model.parameters())
    model.cuda()
    model.weight.grad = torch.randn_like(model.weight)
    before = model.weight.detach().clone()
    opt.step()
    assert not torch.equal(model.weight.detach(), before)
