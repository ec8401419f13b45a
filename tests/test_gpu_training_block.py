"""The training operators together, as a sequence-local block uses them: relative positions start the pair stream, which goes through a row- and a
column-shared dropout; the single stream goes through LayerNorm, local attention with a learned bias by offset, and an element-wise
dropout into the residual.  Loss and gradients against the same block in 64 bits."""
import pytest
import torch

import protenix_b200 as px
from philox import keep
from window_reference import visible

pytestmark = pytest.mark.gpu
N, C, H, D, CZ, R = 150, 64, 4, 16, 32, 12
LEFT, RIGHT, SINKS, SEED, P = 30, 20, 2, 99, 0.25


class Block(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.relpos = px.RelativePositionEncoding(r_max=R, s_max=2, c_z=CZ)
        self.norm = px.LayerNorm(C)
        self.qkv = torch.nn.Linear(C, 3 * H * D, bias=False)
        self.out = torch.nn.Linear(H * D, C, bias=False)
        self.rel_bias = torch.nn.Parameter(torch.randn(H, 2 * R + 1) * 0.3)
        self.gate = torch.nn.Linear(CZ, CZ, bias=False)

    def forward(self, s, features, mask):
        z = self.relpos(features)
        z = px.dropout_add(z, self.gate(z), P, SEED, offset=0, shared_dim=-3)
        z = px.dropout_add(z, self.gate(z), P, SEED, offset=1, shared_dim=-2)
        q, k, v = (t.transpose(0, 1)[None] for t in self.qkv(self.norm(s)).to(torch.bfloat16).view(N, 3 * H, D).chunk(3, 1))
        o = px.window_attention(q, k, v, (LEFT, RIGHT), sinks=SINKS, rel_bias=self.rel_bias, mask=mask)
        update = self.out(o[0].transpose(0, 1).reshape(N, H * D).float())
        return px.dropout_add(s, update, P, SEED, offset=2), z


def _in_64_bits(block, s, features, mask):
    """The same, with the roundings of q, k and v to 16 bits as the only ones (straight through)."""
    w = {k: v.detach().double().requires_grad_() for k, v in block.named_parameters()}
    f = {k: v[:, None] - v[None, :] for k, v in features.items()}
    far = lambda d, r, ok: torch.where(ok, d.clamp(-r, r) + r, 2 * r + 1)
    chain, entity = f["asym_id"] == 0, f["entity_id"] == 0
    hot = torch.nn.functional.one_hot
    one = torch.cat([hot(far(f["residue_index"], R, chain), 2 * R + 2), hot(far(f["token_index"], R, chain & (f["residue_index"] == 0)), 2 * R + 2),
                     entity[..., None].long(), hot(far(f["sym_id"], 2, entity), 6)], -1).double()
    m = lambda shape, offset, dim=None: torch.from_numpy(keep(shape, P, SEED, offset, dim)).cuda().double() / (1 - P)
    z = one @ w["relpos.linear_no_bias.weight"].t()
    for offset, dim in ((0, -3), (1, -2)):
        z = z + (z @ w["gate.weight"].t()) * m(z.shape, offset, dim)
    x = torch.nn.functional.layer_norm(s, (C,), w["norm.weight"], w["norm.bias"])
    qkv = x @ w["qkv.weight"].t()
    qkv = qkv + (qkv.to(torch.bfloat16).double() - qkv).detach()
    q, k, v = (t.transpose(0, 1) for t in qkv.view(N, 3 * H, D).chunk(3, 1))
    at = (torch.arange(N, device="cuda")[None] - torch.arange(N, device="cuda")[:, None]).clamp(-R, R) + R
    seen = visible(N, LEFT, RIGHT, SINKS, mask, s.device)
    p = torch.softmax((q @ k.transpose(-1, -2) * D ** -0.5 + w["rel_bias"][:, at]).masked_fill(~seen, -1e300), -1) * seen.any(-1, keepdim=True)
    update = (p @ v).transpose(0, 1).reshape(N, H * D) @ w["out.weight"].t()
    return s + update * m(s.shape, 2), z, w


def test_a_training_step():
    torch.manual_seed(5)
    block = Block().cuda()
    s = torch.randn(N, C, device="cuda", requires_grad=True)
    asym = (torch.arange(N, device="cuda") >= 90).long()
    features = {"asym_id": asym, "residue_index": torch.arange(N, device="cuda") - 90 * asym, "entity_id": asym * 0,
                "token_index": torch.arange(N, device="cuda"), "sym_id": asym}
    mask = torch.arange(N, device="cuda")[None] < N - 11
    gs, gz = torch.randn(N, C, device="cuda"), torch.randn(N, N, CZ, device="cuda") / N
    s_out, z_out = block(s, features, mask)
    names, params = zip(*block.named_parameters())
    grads = torch.autograd.grad((s_out, z_out), (s, *params), (gs, gz))
    s64 = s.detach().double().requires_grad_()
    s_ref, z_ref, w = _in_64_bits(block, s64, features, mask)
    want = torch.autograd.grad((s_ref, z_ref), (s64, *[w[n] for n in names]), (gs.double(), gz.double()))
    # Half a step of bf16 enters at P, o, dO, dS and the results of the attention and of its gradient; a path from the loss to a parameter meets at most
    # six of these.  Library products are fp32.
    u = 2.0 ** -8
    for name, x, y in (("s", s_out, s_ref), ("z", z_out, z_ref), ("ds", grads[0], want[0]), *zip(names, grads[1:], want[1:])):
        assert float((x.detach().double() - y.detach()).norm()) <= 6 * u * float(y.detach().norm()), name
    # the pair stream has no 16-bit value
    assert float((z_out.detach().double() - z_ref.detach()).norm()) <= 1e-5 * float(z_ref.detach().norm())
    again = torch.autograd.grad(block(s, features, mask), (s, *params), (gs, gz))
    for name, a, b in zip(("s", *names), grads, again):
        if name != "norm.weight" and name != "norm.bias":      # sums of the LayerNorm op's own
            assert torch.equal(a, b), name
