"""The Muon optimiser, and the operators of a training step together: rotary positions, local attention, a head with its loss, the gradients, the update."""
import math

import pytest
import torch

import protenix_b200 as px
from window_reference import visible

pytestmark = pytest.mark.gpu


def _orthogonal(x):
    x = x / (torch.linalg.matrix_norm(x)[..., None, None] + 1e-7)
    for _ in range(5):
        s = x @ x.mT
        x = 3.4445 * x + (-4.7750 * s + 2.0315 * (s @ s)) @ x
    return x


@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_steps(nesterov, dtype):
    torch.manual_seed(3)
    shapes = [(40, 24), (24, 40), (40, 24), (3, 16, 16), (40, 24)]
    params = [torch.nn.Parameter(torch.randn(s, device="cuda").to(dtype)) for s in shapes]
    frozen = torch.nn.Parameter(torch.randn(8, 8, device="cuda").to(dtype))
    before = frozen.detach().clone()
    opt = px.Muon([*params, frozen], lr=0.1, momentum=0.9, nesterov=nesterov, weight_decay=0.01)
    want, held = [p.detach().double() for p in params], [torch.zeros(s, device="cuda", dtype=torch.float64) for s in shapes]
    u = torch.finfo(dtype).eps / 2
    for step in range(3):
        grads = [torch.randn(s, device="cuda").to(dtype) for s in shapes]
        for i, (p, g) in enumerate(zip(params, grads)):
            p.grad = g.clone()
            held[i] = 0.9 * held[i] + g.double()
            x = g.double() + 0.9 * held[i] if nesterov else held[i]
            want[i] = want[i] * (1 - 0.1 * 0.01) - 0.1 * math.sqrt(max(1.0, g.shape[-2] / g.shape[-1])) * _orthogonal(x)
        opt.step()
    # three steps of roundings: of the momentum (three products and sums, and the noise in small directions that the iteration multiplies), the update and the weight
    for p, w in zip(params, want):
        assert float((p.detach().double() - w).norm()) <= (60 * u + 1e-5) * float(w.norm())
    assert torch.equal(frozen.detach(), before)
    state = opt.state_dict()
    other = px.Muon([*params, frozen], lr=0.1)
    other.load_state_dict(state)
    assert torch.equal(other.state[params[0]]["momentum_buffer"], opt.state[params[0]]["momentum_buffer"])


def test_a_parameter_without_elements():
    for shape in ((3, 0), (0, 3), (2, 0, 0)):
        p = torch.nn.Parameter(torch.zeros(shape, device="cuda"))
        p.grad = torch.zeros_like(p)
        px.Muon([p]).step()
        assert p.shape == shape


def test_refusals():
    with pytest.raises(ValueError, match="two axes"):
        px.Muon([torch.nn.Parameter(torch.randn(5, device="cuda"))])
    for kw in ({"lr": -1.0}, {"momentum": 1.0}, {"weight_decay": -0.1}):
        with pytest.raises(ValueError):
            px.Muon([torch.nn.Parameter(torch.randn(5, 5, device="cuda"))], **kw)


N, C, H, HK, D, V = 200, 64, 4, 2, 32, 77
LEFT, RIGHT, SECTIONS = 40, 40, (8, 5, 3)


class Model(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.norm = px.LayerNorm(C)
        self.qkv = torch.nn.Linear(C, (H + 2 * HK) * D, bias=False)
        self.out = torch.nn.Linear(H * D, C, bias=False)
        self.head = torch.nn.Linear(C, V)

    def forward(self, s, positions, target):
        q, k, v = (t.transpose(0, 1)[None] for t in self.qkv(self.norm(s)).bfloat16().view(N, H + 2 * HK, D).split([H, HK, HK], 1))
        q, k = px.rotary_embedding(q, k, positions, sections=SECTIONS, per_axis=True)
        o = px.window_attention(q, k, v, (LEFT, RIGHT))
        x = s + self.out(o[0].transpose(0, 1).reshape(N, H * D).float())
        return px.linear_cross_entropy(x.bfloat16(), self.head.weight.bfloat16(), target, bias=self.head.bias)


def _in_64_bits(model, s, positions, target):
    """The same, with the roundings of inputs to 16 bits as the only ones (straight through)."""
    w = {k: v.detach().double().requires_grad_() for k, v in model.named_parameters()}
    short = lambda x: x + (x.to(torch.bfloat16).double() - x).detach()  # noqa: E731
    x = torch.nn.functional.layer_norm(s, (C,), w["norm.weight"], w["norm.bias"])
    q, k, v = (t.transpose(0, 1) for t in short(x @ w["qkv.weight"].t()).view(N, H + 2 * HK, D).split([H, HK, HK], 1))
    speed = torch.tensor([10000.0 ** -(i / n) for n in SECTIONS for i in range(n)], dtype=torch.float64, device="cuda")
    angle = positions.double()[:, [a for a, n in enumerate(SECTIONS) for _ in range(n)]] * speed
    cos, sin = angle.cos(), angle.sin()

    def turned(t):
        a, b = t[..., : D // 2], t[..., D // 2:]
        return short(torch.cat([a * cos - b * sin, b * cos + a * sin], -1))

    q, k = turned(q), turned(k)
    seen = visible(N, LEFT, RIGHT, 0, None, s.device)
    p = torch.softmax((q @ k.repeat_interleave(H // HK, 0).mT * D ** -0.5).masked_fill(~seen, -1e300), -1)
    o = (p @ v.repeat_interleave(H // HK, 0)).transpose(0, 1).reshape(N, H * D)
    x = short(s + o @ w["out.weight"].t())
    return torch.nn.functional.cross_entropy(x @ short(w["head.weight"]).t() + w["head.bias"], target), w


def test_a_training_step():
    torch.manual_seed(7)
    model = Model().cuda()
    s = torch.randn(N, C, device="cuda")
    positions = torch.stack([torch.arange(N), torch.arange(N) % 8, torch.arange(N) // 70], -1).cuda()
    target = torch.randint(0, V, (N,), device="cuda")
    target[::9] = -100
    loss = model(s, positions, target)
    loss.backward()
    ref, w = _in_64_bits(model, s.double(), positions, target)
    want = dict(zip(w, torch.autograd.grad(ref, list(w.values()))))
    # Half a step of bf16 enters at q, k, P, o, x, dl, dx, dW of the head, dO, dS, dq, dk and their turned forms: a path to a parameter meets at most ten.
    u = 2.0 ** -8
    assert abs(float(loss.detach()) - float(ref.detach())) <= 4 * u * float(ref.detach())
    for name, p in model.named_parameters():
        assert float((p.grad.double() - want[name]).norm()) <= 10 * u * float(want[name].norm()), name
    matrices = [p for p in model.parameters() if p.dim() == 2]
    before = [p.detach().double() for p in matrices]
    held = [p.grad.double() for p in matrices]
    px.Muon(matrices, lr=0.02).step()
    for p, b, g in zip(matrices, before, held):
        step = -0.02 * max(1.0, p.shape[0] / p.shape[1]) ** 0.5 * _orthogonal(1.95 * g)
        assert float((p.detach().double() - b - step).norm()) <= 1e-4 * float(step.norm()) + 2.0 ** -23 * float(b.norm())
