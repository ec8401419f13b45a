"""window_attention against its formulas in 64 bits."""
import math

import pytest
import torch

import protenix_b200 as px
from protenix_b200 import ops
from window_reference import check, half_step, reference, visible

BF16, FP16 = torch.bfloat16, torch.float16
NAMES = ("dq", "dk", "dv", "drel_bias")


def _inputs(b, h, hk, n, d, dtype, r=None, seed=0, bias_dtype=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")
    q, k, v, grad = (rand(b, x, n, d).to(dtype) for x in (h, hk, hk, h))
    bias = None if r is None else rand(h, 2 * r + 1).to(bias_dtype or dtype)
    return q, k, v, grad, bias


def _mask(kind, b, n):
    """Samples of unlike length: padded behind, in front, or with holes."""
    if kind is None:
        return None
    at = torch.arange(n, device="cuda")[None].expand(b, n)
    pad = (torch.arange(b, device="cuda")[:, None] + 1) * n // (2 * b)
    if kind == "end":
        return at < n - pad
    if kind == "front":
        return at >= pad
    if kind == "none":
        return at < 0
    return (at * 7 + torch.arange(b, device="cuda")[:, None]) % 3 != 0


def _run(q, k, v, grad, bias, mask, left, right, sinks, scale=None):
    leaves = [t.detach().clone(memory_format=torch.preserve_format).requires_grad_() for t in (q, k, v)]
    if bias is not None:
        leaves.append(bias.detach().clone().requires_grad_())
    o = px.window_attention(*leaves[:3], (left, right), sinks=sinks, rel_bias=leaves[3] if bias is not None else None, mask=mask, scale=scale)
    grads = torch.autograd.grad(o, leaves, grad)
    plain = px.window_attention(q, k, v, (left, right), sinks=sinks, rel_bias=bias, mask=mask, scale=scale)
    ops.device_error_flags()
    assert torch.equal(plain, o.detach()) and all(x.dtype == y.dtype and x.shape == y.shape for x, y in zip(grads, leaves))
    return {"o": o.detach(), **dict(zip(NAMES, grads))}


def _case(b, h, hk, n, d, left, right, sinks, r, mask, dtype, seed=0, scale=None, bias_dtype=None):
    q, k, v, grad, bias = _inputs(b, h, hk, n, d, dtype, r, seed, bias_dtype)
    m = _mask(mask, b, n)
    got = _run(q, k, v, grad, bias, m, left, right, sinks, scale)
    check(got, reference(q, k, v, left, right, sinks, bias, m, scale, grad), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 127, 128, 129, 200, 333])
def test_lengths(n):
    _case(2, 4, 4, n, 32, 64, 63, 0, None, None, BF16, seed=n)
    _case(1, 2, 1, n, 24, 17, 0, 3, 8, "holes", FP16, seed=n)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [8, 16, 24, 32, 40, 64, 72, 80, 96, 128])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_head_sizes(d, dtype):
    _case(1, 2, 2, 150, d, 40, 30, 0, 16, None, dtype, seed=d)


@pytest.mark.gpu
@pytest.mark.parametrize("left,right", [(0, 0), (1, 0), (0, 1), (0, 500), (500, 0), (63, 64), (127, 128), (200, 7), (10 ** 12, 10 ** 12)])
@pytest.mark.parametrize("sinks", [0, 1, 64, 70])
def test_windows(left, right, sinks):
    _case(1, 2, 2, 300, 32, left, right, sinks, 20, "holes" if left % 2 else None, BF16, seed=left % 97 + sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("sinks", [1, 128, 129, 300, 5000])
@pytest.mark.parametrize("heads,kv_heads,d", [(4, 4, 32), (6, 2, 40), (4, 1, 128)])
def test_many_queries_of_a_sink(sinks, heads, kv_heads, d):
    """Long enough for the queries of the first keys to be cut into chunks."""
    n = 4300 if heads == kv_heads else 2200
    _case(1, heads, kv_heads, n, d, 33, 0, sinks, None, None, BF16, seed=sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("mask", ["end", "front", "holes", "none"])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_masks_and_rows_that_see_nothing(mask, dtype):
    _case(3, 4, 2, 261, 32, 20, 20, 2, 8, mask, dtype)
    _case(2, 2, 2, 261, 72, 20, 0, 0, None, mask, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("r", [0, 1, 31, 63, 64, 65, 200, 256])
def test_learned_bias(r):
    _case(2, 3, 3, 420, 32, 150, 90, 5, r, None, BF16, seed=r)
    _case(1, 4, 2, 260, 64, 300, 0, 0, r, "holes", FP16, seed=r, bias_dtype=torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1e-3, 1.0, 4.0])
def test_scales(scale):
    _case(1, 2, 2, 200, 32, 100, 100, 0, None, None, FP16, scale=scale)


@pytest.mark.gpu
def test_logits_that_grow_along_the_row():
    """The reference maximum has to move again and again, and the sums with it."""
    n, d = 700, 32
    q, k, v, grad, _ = _inputs(1, 2, 2, n, d, BF16)
    k = (k + torch.linspace(0, 12, n, device="cuda")[:, None] * q.mean(2, keepdim=True).sign()).to(BF16)
    q = (q.abs() * q.mean(2, keepdim=True).sign()).to(BF16)
    got = _run(q, k, v, grad, None, None, 600, 600, 0)
    check(got, reference(q, k, v, 600, 600, grad=grad), BF16)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [32, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), 65504.0])
def test_what_masked_places_hold_has_no_influence(bad, d):
    q, k, v, grad, bias = _inputs(2, 4, 2, 290, d, FP16, 16)
    for kind in ("front", "holes", "end"):
        m = _mask(kind, 2, 290)
        want = _run(q, k, v, grad, bias, m, 25, 10, 0)
        hidden = ~m[:, None, :, None]
        nothing = ~visible(290, 25, 10, 0, m, q.device).any(-1)[:, None, :, None]
        got = _run(torch.where(nothing, bad, q), torch.where(hidden, bad, k), torch.where(hidden, bad, v), torch.where(nothing, bad, grad), bias, m,
                   25, 10, 0)
        for name in want:
            assert torch.equal(got[name], want[name]), (kind, name)
        assert not got["dk"].masked_select(hidden).any() and not got["dv"].masked_select(hidden).any()
        assert not got["o"].masked_select(nothing).any() and not got["dq"].masked_select(nothing).any()


@pytest.mark.gpu
def test_bias_of_minus_infinity_hides():
    q, k, v, grad, bias = _inputs(1, 2, 2, 200, 32, BF16, 4)
    bias[:, 0] = -math.inf                     # everything four or more behind
    got = _run(q, k, v, grad, bias, None, 60, 20, 0)
    want = _run(q, k, v, grad, torch.where(bias == -math.inf, 0.0, bias).to(BF16), None, 3, 20, 0)
    for name in ("o", "dq", "dk", "dv"):
        assert float((got[name].float() - want[name].float()).norm()) <= 2 * half_step(BF16) * float(want[name].float().norm()), name


@pytest.mark.gpu
def test_layouts():
    """Heads inside the rows of one projection, three axes, five axes, broadcast k, rows off their 16 bytes: the same numbers."""
    b, h, n, d = 2, 4, 170, 32
    packed = torch.randn(b, n, 3 * h, d, device="cuda").to(BF16).requires_grad_()
    q, k, v = (t.transpose(1, 2) for t in packed.chunk(3, 2))
    grad = torch.randn(b, n, h, d, device="cuda").to(BF16).transpose(1, 2)
    o = px.window_attention(q, k, v, 40)
    assert o.stride() == grad.stride() and o.transpose(1, 2).is_contiguous()
    dp, = torch.autograd.grad(o, packed, grad)
    plain = _run(*(t.detach().contiguous() for t in (q, k, v)), grad.contiguous(), None, None, 40, 40, 0)
    assert torch.equal(o, plain["o"])
    assert torch.equal(dp, torch.cat([plain[x].transpose(1, 2) for x in NAMES[:3]], 2))
    q, k, v = (t.detach().contiguous() for t in (q, k, v))
    assert torch.equal(px.window_attention(q[0], k[0], v[0], 40), plain["o"][0])
    five = lambda t: t.reshape(2, 1, h, n, d).expand(2, 3, h, n, d)
    mask = torch.ones(2, 1, n, device="cuda")
    got = px.window_attention(five(q), five(k), five(v), 40, mask=mask)
    assert got.shape == (2, 3, h, n, d) and all(torch.equal(got[:, i], plain["o"]) for i in range(3))
    k1 = k[:1].clone().requires_grad_()
    o = px.window_attention(q, k1.expand(b, h, n, d), v, 40)
    want = _run(q, k[:1].expand(b, h, n, d).contiguous(), v, grad, None, None, 40, 40, 0)
    assert torch.equal(o, want["o"])
    dk1, = torch.autograd.grad(o, k1, grad)
    assert torch.equal(dk1, want["dk"].sum(0, keepdim=True))
    off = torch.empty(q.numel() + 4, dtype=BF16, device="cuda")[4:].view(q.shape).copy_(q)
    assert off.data_ptr() % 16 and torch.equal(px.window_attention(off, k, v, 40), plain["o"])
    wide = torch.zeros(b, h, n, d + 4, dtype=BF16, device="cuda")[..., :d].copy_(q)
    assert torch.equal(px.window_attention(wide, k, v, 40), plain["o"])
    turned = q.transpose(-1, -2).contiguous().transpose(-1, -2)
    assert torch.equal(px.window_attention(turned, k, v, 40), plain["o"])
    # a gradient that is one value everywhere
    qr = q.clone().requires_grad_()
    px.window_attention(qr, k, v, 40).sum().backward()
    assert torch.equal(qr.grad, _run(q, k, v, torch.ones_like(q), None, None, 40, 40, 0)["dq"])


@pytest.mark.gpu
def test_shapes_of_a_mask():
    """One row for all samples, one value for a sample, any type."""
    q, k, v, grad, _ = _inputs(3, 2, 2, 140, 32, BF16)
    at = torch.arange(140, device="cuda")
    row = (at % 3 != 0)
    want = px.window_attention(q, k, v, 20, mask=row[None].expand(3, 140).contiguous())
    for m in (row, row[None], row.float(), row.to(torch.int32) * 7, row[None].expand(3, 140)):
        assert torch.equal(px.window_attention(q, k, v, 20, mask=m), want)
    some = torch.tensor([[True], [False], [True]], device="cuda")
    got = px.window_attention(q, k, v, 20, mask=some)
    plain = px.window_attention(q, k, v, 20)
    assert torch.equal(got[0], plain[0]) and torch.equal(got[2], plain[2]) and not got[1].any()
    assert torch.equal(px.window_attention(q, k, v, 20, mask=torch.ones(1, device="cuda")), plain)


@pytest.mark.gpu
def test_some_gradients_only():
    q, k, v, grad, bias = _inputs(1, 4, 2, 200, 32, BF16, 8)
    want = _run(q, k, v, grad, bias, None, 50, 0, 3)
    for names in (("dq",), ("dk",), ("dv",), ("drel_bias",), ("dk", "drel_bias")):
        leaves = {"dq": q, "dk": k, "dv": v, "drel_bias": bias}
        leaves = {x: t.detach().clone().requires_grad_(x in names) for x, t in leaves.items()}
        o = px.window_attention(leaves["dq"], leaves["dk"], leaves["dv"], (50, 0), sinks=3, rel_bias=leaves["drel_bias"])
        for x, g in zip(names, torch.autograd.grad(o, [leaves[x] for x in names], grad)):
            assert torch.equal(g, want[x]), x


@pytest.mark.gpu
def test_gradients_against_differences():
    """Central differences of the kernel's own forward pass in one random direction per input.  The step h moves the loss by 2 h times the slope; its
    two values carry the rounding of o (half a step u of each |o|, and as much for P), with signs that do not add up: the root of the sum of
    squares, six times it for safety, is the tolerance."""
    q, k, v, grad, bias = _inputs(1, 2, 2, 300, 32, FP16, 16, bias_dtype=torch.float32)
    got = _run(q, k, v, grad, bias, None, 80, 40, 3)
    loss = lambda a, b, c, d: (px.window_attention(a, b, c, (80, 40), sinks=3, rel_bias=d).double() * grad.double()).sum()
    noise = float((grad.double() * got["o"].double()).norm()) * half_step(FP16) * 2
    for i, name in enumerate(NAMES):
        base = [q, k, v, bias]
        g = torch.Generator(device="cuda").manual_seed(i)
        step = torch.randn(base[i].shape, generator=g, device="cuda").sign() * 2.0 ** -4
        up, down = [list(base) for _ in range(2)]
        up[i], down[i] = (base[i] + step).to(base[i].dtype), (base[i] - step).to(base[i].dtype)
        moved = (up[i].double() - down[i].double())
        slope = float((moved * got[name].double()).sum())
        diff = float(loss(*up) - loss(*down))
        # third-order term: the logits move by about |step| * norm of the other side, at most a third here: h^2/6 of the change
        assert abs(diff - slope) <= 6 * noise + 0.05 * float((moved * got[name].double()).norm()), name


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv_heads,d", [(16, 4, 64), (8, 8, 32), (4, 2, 128)])
def test_what_follows_sees_all_gradients(heads, kv_heads, d):
    """The kernels of the backward pass run beside one another; whatever is launched behind it, by this package or another, waits for all of them."""
    q, k, v, grad, bias = _inputs(1, heads, kv_heads, 3000, d, BF16, 128)
    want = _run(q, k, v, grad, bias, None, 300, 0, 4)
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v, bias)]
    results = []
    for i in range(12):
        o = px.window_attention(*leaves[:3], (300, 0), sinks=4, rel_bias=leaves[3])
        dq, dk, dv, db = torch.autograd.grad(o, leaves, grad)
        if i % 2:
            results.append((dq + 0, dk + 0, dv + 0, db + 0, None))
        else:
            results.append((dq, dk, dv, db, ops.layer_norm(dq.reshape(-1, d), None, None)))
        del dq, dk, dv, db
    normed = ops.layer_norm(want["dq"].reshape(-1, d), None, None)
    ops.device_error_flags()
    for *grads, n in results:
        assert all(torch.equal(g, want[x]) for g, x in zip(grads, NAMES))
        assert n is None or torch.equal(n, normed)


@pytest.mark.gpu
def test_same_bits_on_other_streams_and_in_a_graph():
    q, k, v, grad, bias = _inputs(2, 8, 2, 900, 64, BF16, 32)
    m = _mask("end", 2, 900)
    want = _run(q, k, v, grad, bias, m, 200, 0, 4)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    results = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                leaves = [t.detach().clone().requires_grad_() for t in (q, k, v, bias)]
                o = px.window_attention(*leaves[:3], (200, 0), sinks=4, rel_bias=leaves[3], mask=m)
                results.append((o.detach(), *torch.autograd.grad(o, leaves, grad)))
    torch.cuda.synchronize()
    for got in results:
        assert all(torch.equal(a, b) for a, b in zip(got, want.values()))
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v, bias)]

    def step():
        o = px.window_attention(*leaves[:3], (200, 0), sinks=4, rel_bias=leaves[3], mask=m)
        return (o, *torch.autograd.grad(o, leaves, grad))

    with torch.cuda.stream(streams[0]):
        step()
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(step())
    with torch.no_grad():
        for t in leaves:
            t.mul_(0.5)
    for s, graph in zip(streams, graphs):
        with torch.cuda.stream(s):
            graph.replay()
    torch.cuda.synchronize()
    half = _run(*(t.detach() for t in leaves[:3]), grad, leaves[3].detach(), m, 200, 0, 4)
    for out in outs:
        assert all(torch.equal(a, b) for a, b in zip(out, half.values()))


@pytest.mark.gpu
def test_empty():
    for shape in ((0, 4, 8, 32), (2, 4, 0, 32)):
        q = torch.zeros(shape, dtype=BF16, device="cuda").requires_grad_()
        bias = torch.zeros(4, 5, device="cuda").requires_grad_()
        o = px.window_attention(q, q, q, 3, rel_bias=bias)
        dq, db = torch.autograd.grad(o.sum(), (q, bias))
        assert o.shape == shape and dq.shape == shape and not db.any()


@pytest.mark.gpu
def test_refusals():
    q, k, v, _, bias = _inputs(2, 4, 2, 20, 32, BF16, 3)
    call = lambda q=q, k=k, v=v, window=5, **kw: px.window_attention(q, k, v, window, **kw)
    for match, kw in [("bfloat16 or float16", {"q": q.float()}), ("type of q", {"k": k.half()}), ("divisor", {"k": k[:, :1].expand(2, 3, 20, 32), "v": v[:, :1].expand(2, 3, 20, 32)}),
                      ("divisor", {"v": v[:, :, :10]}), ("divisor", {"k": k[:1], "v": v[:1]}), ("H, N, D", {"q": q[0, 0]}),
                      ("head sizes", {"q": q[..., :12], "k": k[..., :12], "v": v[..., :12]}), ("negative", {"window": -1}), ("negative", {"window": (3, -2)}),
                      ("negative", {"sinks": -1}), ("positive", {"scale": 0.0}), ("positive", {"scale": -1.0}), ("positive", {"scale": float("nan")}),
                      ("positive", {"scale": float("inf")}), ("rel_bias must be", {"rel_bias": bias[:, :6]}), ("rel_bias must be", {"rel_bias": bias[:2]}),
                      ("rel_bias must be", {"rel_bias": torch.zeros(4, 515, device="cuda")}), ("float32 or", {"rel_bias": bias.half()}),
                      ("CUDA", {"rel_bias": bias.cpu()}), ("mask must be", {"mask": torch.ones(2, 19, device="cuda")}),
                      ("CUDA", {"mask": torch.ones(2, 20)}), ("CUDA", {"k": k.cpu()})]:
        with pytest.raises(RuntimeError, match=match):
            call(**kw)
    wide = torch.zeros(1, 1, 4, 136, dtype=BF16, device="cuda")
    with pytest.raises(RuntimeError, match="head sizes"):
        call(wide, wide, wide)
    leaf = q.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(call(leaf).sum(), leaf, create_graph=True)


def test_cpu_tensors_are_refused():
    q = torch.zeros(1, 2, 5, 32, dtype=BF16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        px.window_attention(q, q, q, 3)


def test_status_codes_of_the_c_interface():
    """Bad calls end with a status before anything is launched (no GPU needed)."""
    import ctypes

    from protenix_b200 import _lib

    class Rows(ctypes.Structure):
        _fields_ = [("data", ctypes.c_void_p), ("batch", ctypes.c_int64), ("head", ctypes.c_int64), ("row", ctypes.c_int64)]

    class Window(ctypes.Structure):
        _fields_ = [(x, ctypes.c_int64) for x in ("batch", "heads", "kv_heads", "n", "d", "left", "right", "sinks", "r_max")] + \
                   [("bias", ctypes.c_void_p), ("mask", ctypes.c_void_p), ("scale", ctypes.c_float), ("dtype", ctypes.c_int32), ("bias_dtype", ctypes.c_int32)]

    lib = _lib.load()
    buf = ctypes.create_string_buffer(256)
    at = (ctypes.addressof(buf) + 15) // 16 * 16
    good = dict(batch=1, heads=4, kv_heads=2, n=10, d=32, left=3, right=0, sinks=0, r_max=-1, scale=1.0, dtype=_lib.PX_BF16)
    ref = ctypes.byref

    def fwd(q=Rows(at, 1280, 320, 32), **kw):
        w, x = Window(**{**good, **kw}), Rows(at, 1280, 320, 32)
        return lib.px_window_fwd(ref(w), ref(q), ref(x), ref(x), ref(x), None, None, None)

    assert fwd(n=0) == 0 and fwd(batch=0) == 0
    for kw in ({"kv_heads": 3}, {"left": -1}, {"d": 0}, {"scale": 0.0}, {"scale": float("nan")}, {"r_max": 2}, {"heads": 0}):
        assert fwd(**kw) == -1, kw
    for kw in ({"d": 12}, {"d": 136}, {"dtype": _lib.PX_F32}, {"n": 1 << 25}, {"r_max": 257, "bias": at}, {"batch": 1 << 20}):
        assert fwd(**kw) == -2, kw
    for q in (Rows(None, 1280, 320, 32), Rows(at + 2, 1280, 320, 32), Rows(at, 1280, 320, 36), Rows(at, 1280, 0, 32), Rows(at, 1280, -320, 32)):
        assert fwd(q) == -1
    w, x = Window(**good), Rows(at, 1280, 320, 32)
    size = lib.px_window_workspace_bytes(ref(w), 0)
    assert size >= 4 * 128 * 4 and lib.px_window_workspace_bytes(ref(Window(**{**good, "d": 12})), 0) == 0
    work = at // 256 * 256 + 256      # never touched: only its alignment is looked at
    bwd = lambda bytes_, lse=at, dbias=None: lib.px_window_bwd(ref(w), ref(x), ref(x), ref(x), ref(x), None, ref(x), lse, ref(x), ref(x), ref(x), dbias, work, bytes_, None)
    assert bwd(size - 1) == -4 and bwd(size, lse=None) == -1 and bwd(size, dbias=at) == -1
