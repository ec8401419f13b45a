"""Which outputs of rotary_embedding ask for a gradient."""
import pytest
import torch

import protenix_b200 as px

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(1, 2, 9, 16), (2, 9, 16), (2, 3, 2, 9, 16)])
@pytest.mark.parametrize("of_q,of_k", [(True, False), (False, True), (True, True), (False, False)])
def test_only_what_depends_on_a_leaf(of_q, of_k, shape):
    q, k = torch.randn(shape, device="cuda", requires_grad=of_q), torch.randn(shape, device="cuda", requires_grad=of_k)
    at = torch.arange(9, device="cuda")[:, None]
    yq, yk = px.rotary_embedding(q, k, at)
    assert yq.requires_grad == of_q and yk.requires_grad == of_k
    both = torch.randn(shape, device="cuda", requires_grad=True), torch.randn(shape, device="cuda", requires_grad=True)
    out = px.rotary_embedding(*both, at)
    for leaf, y, want_leaf, want in zip((q, k), (yq, yk), both, out):
        if leaf.requires_grad:
            up = torch.randn(shape, device="cuda", requires_grad=True)
            g = torch.autograd.grad(y, leaf, up, create_graph=True, retain_graph=True)[0]
            assert torch.equal(g, torch.autograd.grad(want, want_leaf, up, retain_graph=True)[0])
            assert torch.equal(torch.autograd.grad(g, up, leaf.detach())[0], px.rotary_embedding(leaf.detach(), None, at))
    assert px.rotary_embedding(q, None, at).requires_grad == of_q
