"""The trainable operators have no forward-mode derivative: a tensor with a tangent is refused, with and without gradients, and not taken for one without."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import protenix_b200 as px

BF16 = torch.bfloat16


def _calls():
    x = torch.randn(6, 4, 128, device="cuda")
    w = torch.randn(128, 139, device="cuda")
    f = {k: torch.arange(9, device="cuda") for k in ("asym_id", "residue_index", "entity_id", "token_index", "sym_id")}
    q, bias = torch.randn(1, 2, 20, 32, device="cuda").to(BF16), torch.randn(2, 5, device="cuda")
    win = lambda **kw: px.window_attention(**{"q": q, "k": q, "v": q, "window": 3, "rel_bias": bias, **kw})
    norm = px.LayerNorm(128).cuda()
    return {
        "dropout_x": (x, lambda t: px.dropout_add(x, t, 0.5, 3)),
        "dropout_residual": (x, lambda t: px.dropout_add(t, x, 0.5, 3)),
        "relpos_weight": (w, lambda t: px.relative_position_encoding(t, **f)),
        "window_q": (q, lambda t: win(q=t)),
        "window_k": (q, lambda t: win(k=t)),
        "window_v": (q, lambda t: win(v=t)),
        "window_rel_bias": (bias, lambda t: win(rel_bias=t)),
        "layer_norm": (x, norm),
        "dropout_rowwise_x": (x, lambda t: px.dropout_add_rowwise(x, t, 0.5, True)),
        "dropout_rowwise_residual": (x, lambda t: px.dropout_add_rowwise(t, x, 0.5, True)),
    }


NAMES = ["dropout_x", "dropout_residual", "relpos_weight", "window_q", "window_k", "window_v", "window_rel_bias", "layer_norm", "dropout_rowwise_x",
         "dropout_rowwise_residual"]


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("grad", [True, False])
def test_tangents_are_refused(name, grad):
    t, call = _calls()[name]
    with torch.set_grad_enabled(grad):
        call(t)
        with fwd.dual_level():
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(fwd.make_dual(t, torch.ones_like(t)))
            call(t)
        call(t)


@pytest.mark.gpu
def test_evaluation_carries_tangents():
    x = torch.randn(6, 128, device="cuda")
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.full_like(x, 2.0))
        assert bool((fwd.unpack_dual(px.dropout_add(x, dual, 0.5, 3, training=False)).tangent == 2).all())
        assert bool((fwd.unpack_dual(px.dropout_add(None, dual, 0.5, 3, training=False)).tangent == 2).all())
