"""RelativePositionEncoding against the one-hot form of the definition in 64 bits."""
import pytest
import torch

import protenix_b200 as px

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _features(n, seed, lead=(), wild=False):
    g = torch.Generator().manual_seed(seed)
    r = lambda lo, hi: torch.randint(lo, hi, (*lead, n), generator=g)
    if wild:
        return {"asym_id": r(0, 3), "residue_index": r(-50, 50), "entity_id": r(0, 2), "token_index": r(-40, 40), "sym_id": r(-5, 5)}
    asym = r(0, 2).cumsum(-1) // 9
    return {"asym_id": asym, "residue_index": torch.arange(n).expand(*lead, n) // 2 + 3, "entity_id": asym // 2,
            "token_index": torch.arange(n).expand(*lead, n).contiguous(), "sym_id": asym % 2}


def _one_hot(f, r, s):
    d = {k: v[..., :, None] - v[..., None, :] for k, v in f.items()}
    clip = lambda x, m, ok: torch.where(ok, x.clamp(-m, m) + m, 2 * m + 1)
    chain, entity = d["asym_id"] == 0, d["entity_id"] == 0
    hot = torch.nn.functional.one_hot
    return torch.cat([hot(clip(d["residue_index"], r, chain), 2 * r + 2), hot(clip(d["token_index"], r, chain & (d["residue_index"] == 0)), 2 * r + 2),
                      entity[..., None].long(), hot(clip(d["sym_id"], s, entity), 2 * s + 2)], -1).double()


def _check(f, c, r, s, dtype, seed=1):
    """z: four weights added up in fp32 (three roundings, each of half a step of a partial sum of at most their magnitudes) and rounded once.
    dW: a pair sum in fp32 in some order; its error is at most (terms in a chain) half steps of the sum of magnitudes, and the longest
    chain of a bucket here is its number of pairs."""
    one = _one_hot(f, r, s).cuda()
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(c, one.shape[-1], generator=g).cuda().requires_grad_()
    dz = torch.randn(*one.shape[:-1], c, generator=g).to(dtype).cuda()
    z = px.relative_position_encoding(w, **{k: v.cuda() for k, v in f.items()}, r_max=r, s_max=s, dtype=dtype)
    assert z.dtype == dtype and z.shape == dz.shape
    want, size = one @ w.detach().double().t(), one @ w.detach().double().abs().t()
    bound = HALF_STEP[dtype] * want.abs() + 3.01 * 2.0 ** -24 * size + torch.finfo(dtype).smallest_normal * HALF_STEP[dtype]
    assert bool(((z.detach().double() - want).abs() <= bound).all())
    dw, = torch.autograd.grad(z, w, dz)
    flat, onef = dz.double().reshape(-1, c), one.reshape(-1, one.shape[-1])
    want, size, terms = flat.t() @ onef, flat.abs().t() @ onef, onef.sum(0)
    assert bool(((dw.double() - want).abs() <= 2.0 ** -24 * terms * size + 1e-30).all())
    # far inside that bound: the errors of a sum's steps do not all point one way
    assert float((dw.double() - want).norm()) <= 1e-6 * max(1.0, float(want.norm()))
    return z.detach(), dw


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("n", [1, 2, 16, 31, 33, 97, 150])
def test_chains(n, dtype):
    _check(_features(n, n), 128, 32, 2, DTYPES[dtype])


@pytest.mark.gpu
@pytest.mark.parametrize("c,r,s,lead", [(128, 32, 2, (3,)), (8, 0, 0, ()), (136, 5, 1, (2, 2)), (384, 3, 7, ()), (256, 92, 2, ()), (24, 1, 180, (1,))])
def test_sizes_and_wild_features(c, r, s, lead):
    for dtype in (torch.float32, torch.bfloat16):
        _check(_features(45, c, lead, wild=True), c, r, s, dtype)


@pytest.mark.gpu
def test_same_bits_every_time_and_integer_types():
    f = {k: v.cuda() for k, v in _features(70, 3).items()}
    w = torch.randn(128, 139, device="cuda").requires_grad_()
    dz = torch.randn(70, 70, 128, device="cuda")
    a, b = [torch.autograd.grad(px.relative_position_encoding(w, **f), w, dz)[0] for _ in range(2)]
    assert torch.equal(a, b)
    z = px.relative_position_encoding(w, **f)
    short = {k: v.to(torch.int32) for k, v in f.items()}
    assert torch.equal(px.relative_position_encoding(w, **short), z)
    # a gradient that is one value for all pairs, and one whose channels do not lie side by side
    dw, = torch.autograd.grad(z.sum(), w)
    assert torch.equal(dw, torch.autograd.grad(px.relative_position_encoding(w, **f), w, torch.ones_like(z))[0])
    turned = dz.permute(2, 0, 1).contiguous().permute(1, 2, 0)
    assert torch.equal(torch.autograd.grad(px.relative_position_encoding(w, **f), w, turned)[0], a)


@pytest.mark.gpu
def test_module_and_its_state():
    m = px.RelativePositionEncoding(r_max=32, s_max=2, c_z=128).cuda()
    assert list(m.state_dict()) == ["linear_no_bias.weight"] and m.linear_no_bias.weight.shape == (128, 139)
    f = {k: v.cuda() for k, v in _features(20, 3).items()}
    z = m({**f, "something_else": torch.zeros(1)})
    assert z.shape == (20, 20, 128) and z.dtype == torch.float32
    z.sum().backward()
    assert m.linear_no_bias.weight.grad.shape == (128, 139)
    half = m.bfloat16()
    half.zero_grad(set_to_none=True)
    half(f).sum().backward()
    assert half.linear_no_bias.weight.grad.dtype == torch.bfloat16
    with pytest.raises(RuntimeError, match="sym_id"):
        m({k: v for k, v in f.items() if k != "sym_id"})


@pytest.mark.gpu
def test_features_may_change_before_the_backward_pass():
    f = {k: v.cuda() for k, v in _features(40, 8).items()}
    w = torch.randn(128, 139, device="cuda").requires_grad_()
    dz = torch.randn(40, 40, 128, device="cuda")
    want, = torch.autograd.grad(px.relative_position_encoding(w, **f), w, dz)
    z = px.relative_position_encoding(w, **f)
    for v in f.values():
        v.zero_()
    assert torch.equal(torch.autograd.grad(z, w, dz)[0], want)


@pytest.mark.gpu
def test_capture_and_empty():
    f = {k: v.cuda() for k, v in _features(50, 8).items()}
    w, dz = torch.randn(128, 139, device="cuda").requires_grad_(), torch.randn(50, 50, 128, device="cuda")
    step = lambda: torch.autograd.grad(px.relative_position_encoding(w, **f), w, dz)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    got.zero_()
    graph.replay()
    assert torch.equal(got, want)
    none = {k: v[:0] for k, v in f.items()}
    z = px.relative_position_encoding(w, **none)
    assert z.shape == (0, 0, 128) and not torch.autograd.grad(z.sum(), w)[0].any()


@pytest.mark.gpu
def test_refusals():
    f = {k: v.cuda() for k, v in _features(12, 1).items()}
    w = torch.randn(128, 139, device="cuda").requires_grad_()
    call = lambda weight=w, r_max=32, s_max=2, dtype=None, **kw: px.relative_position_encoding(weight, **{**f, **kw}, r_max=r_max, s_max=s_max, dtype=dtype)
    for match, kw in [("weight must be", {"r_max": 31}), ("weight must be", {"weight": w[:, :100]}), ("multiple of 8", {"weight": w[:100]}),
                      ("negative", {"s_max": -1}), ("integer tensor", {"sym_id": f["sym_id"].float()}), ("one shape", {"asym_id": f["asym_id"][:5]}),
                      ("CUDA tensor", {"token_index": f["token_index"].cpu()}), ("dtype", {"dtype": torch.float64}),
                      ("multiple of 8", {"weight": torch.zeros(8, 411, device="cuda"), "r_max": 100})]:
        with pytest.raises(RuntimeError, match=match):
            call(**kw)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(call().sum(), w, create_graph=True)


def test_cpu_tensors_are_refused():
    f = _features(12, 1)
    with pytest.raises(RuntimeError, match="no CPU path"):
        px.relative_position_encoding(torch.randn(128, 139), **f)
