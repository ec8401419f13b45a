"""Muon over 16-bit parameters: the state, the change of the weights, and what a checkpoint holds."""
import copy
import math

import pytest
import torch

import protenix_b200 as px

pytestmark = pytest.mark.gpu
SHAPES = [(40, 24), (24, 40), (40, 24), (3, 16, 16), (130, 70)]


def _orthogonal(x):
    x = x / (torch.linalg.matrix_norm(x)[..., None, None] + 1e-7)
    for _ in range(5):
        s = x @ x.mT
        x = 3.4445 * x + (-4.7750 * s + 2.0315 * (s @ s)) @ x
    return x


def _parameters(dtype, seed=3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.nn.Parameter(torch.randn(s, device="cuda", generator=g).to(dtype)) for s in SHAPES]


def _give(params, step):
    g = torch.Generator(device="cuda").manual_seed(100 + step)
    for p in params:
        p.grad = torch.randn(p.shape, device="cuda", generator=g).to(p.dtype)


@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("decay", [0.0, 0.3])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_the_change_of_the_weights(nesterov, decay, dtype):
    """One step from the weights that are there: momentum and update in fp32 and one rounding of the weight, half a step of its type.  What fp32 leaves of the
    momentum and operands of 22 bits of the iteration is below 1e-4 of the update."""
    params, lr = _parameters(dtype), 0.1
    opt = px.Muon(params, lr=lr, momentum=0.9, nesterov=nesterov, weight_decay=decay)
    held = [torch.zeros(s, device="cuda", dtype=torch.float64) for s in SHAPES]
    u = torch.finfo(dtype).eps / 2
    for step in range(3):
        _give(params, step)
        before = [p.detach().double() for p in params]
        opt.step()
        for i, p in enumerate(params):
            g = p.grad.double()
            held[i] = 0.9 * held[i] + g
            change = -lr * math.sqrt(max(1.0, g.shape[-2] / g.shape[-1])) * _orthogonal(g + 0.9 * held[i] if nesterov else held[i])
            want = before[i] * (1 - lr * decay) + change
            # of fp32 weights a rounding more, that of the decay
            rounding = u * (1 + 2.0 ** -10) * (want.abs() + (before[i].abs() if dtype == torch.float32 else 0.0)) + 2.0 ** -25 * (dtype == torch.float16)
            off = (p.detach().double() - want).abs() - rounding
            assert float(off.clamp_min(0).norm()) <= 1e-4 * float(change.norm())
            buffer = opt.state[p]["momentum_buffer"]
            assert buffer.dtype == torch.float32 and float((buffer.double() - held[i]).abs().max()) <= 8 * 2.0 ** -24 * float(held[i].abs().max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_decay_alone(dtype):
    """A gradient of zero leaves the decay, rounded once."""
    params = _parameters(dtype)
    before = [p.detach().clone() for p in params]
    for p in params:
        p.grad = torch.zeros_like(p)
    px.Muon(params, lr=0.1, weight_decay=0.25).step()
    for p, b in zip(params, before):
        want = b.double() * (1 - 0.1 * 0.25)
        # the factor, a number of fp32, is off by up to 2^-24 of itself, the product by as much, before a 16-bit weight is rounded: (1 + 2^-24)^2 (1 + u) - 1
        u, fp32 = torch.finfo(dtype).eps / 2, 2.0 ** -24
        bound = 2.01 * fp32 if dtype == torch.float32 else u + 2.01 * fp32
        assert bool(((p.detach().double() - want).abs() <= bound * want.abs() + 2.0 ** -25 * (dtype == torch.float16)).all())
        assert bool((p.detach() != b).any())


def test_momentum_beyond_fp16():
    """A steady gradient adds up to twenty times itself, beyond what fp16 holds."""
    p = torch.nn.Parameter(torch.zeros(16, 16, device="cuda", dtype=torch.float16))
    opt = px.Muon([p], lr=0.001)
    grad = (torch.randn(16, 16, device="cuda", generator=torch.Generator(device="cuda").manual_seed(0)).sign() * 20000).half()
    for _ in range(60):
        p.grad = grad.clone()
        opt.step()
    assert bool(p.isfinite().all()) and float(opt.state[p]["momentum_buffer"].abs().max()) > 65504


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_a_checkpoint_goes_on_as_if_nothing_had_been(dtype):
    params = _parameters(dtype)
    opt = px.Muon([{"params": params[:2]}, {"params": params[2:], "lr": 0.05}], lr=0.1, weight_decay=0.1)
    for step in range(2):
        _give(params, step)
        opt.step()
    state = copy.deepcopy(opt.state_dict())
    others = [torch.nn.Parameter(p.detach().clone()) for p in params]
    again = px.Muon([{"params": others[:2]}, {"params": others[2:]}])
    again.load_state_dict(state)
    for p, q in zip(params, others):
        a, b = opt.state[p]["momentum_buffer"], again.state[q]["momentum_buffer"]
        assert b.dtype == torch.float32 and torch.equal(a, b)
    for step in range(2, 4):
        for o, ps in ((opt, params), (again, others)):
            _give(ps, step)
            o.step()
    assert all(torch.equal(p, q) for p, q in zip(params, others))


def test_a_checkpoint_with_a_momentum_in_16_bits():
    """What an older one holds is taken over into fp32."""
    p = torch.nn.Parameter(torch.randn(16, 8, device="cuda").bfloat16())
    opt = px.Muon([p])
    p.grad = torch.randn_like(p)
    opt.step()
    state = copy.deepcopy(opt.state_dict())
    state["state"][0]["momentum_buffer"] = state["state"][0]["momentum_buffer"].bfloat16()
    opt.load_state_dict(state)
    p.grad = torch.randn_like(p)
    opt.step()
    assert opt.state[p]["momentum_buffer"].dtype == torch.float32


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_captured_step(dtype):
    """Replays move the state and the weights as calls do."""
    params, others = _parameters(dtype), _parameters(dtype)
    opt, again = px.Muon(params, lr=0.1, weight_decay=0.1), px.Muon(others, lr=0.1, weight_decay=0.1)
    grads = [torch.zeros_like(p) for p in params]
    for p, g in zip(params, grads):
        p.grad = g
    for o, ps in ((opt, params), (again, others)):
        for p in ps:
            p.grad = torch.zeros_like(p) if ps is others else p.grad
        o.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for step in range(3):
        _give(others, step)
        for g, q in zip(grads, others):
            g.copy_(q.grad)
        graph.replay()
        again.step()
        assert all(torch.equal(p, q) for p, q in zip(params, others))
        assert all(torch.equal(opt.state[p]["momentum_buffer"], again.state[q]["momentum_buffer"]) for p, q in zip(params, others))
