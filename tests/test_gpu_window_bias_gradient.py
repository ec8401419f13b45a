"""What the backward pass of windowed attention does for the learned bias's gradient: delta of an output with what its rounding has taken off, and
a row's left-over taken out of the sums over clipped offsets.  Few tokens a window, many sinks behind one entry of the bias."""
import ctypes
import math

import pytest
import torch

import protenix_b200 as px
from protenix_b200 import _lib, ops
from window_reference import check, reference, visible

BF16 = torch.bfloat16


class Rows(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("batch", ctypes.c_int64), ("head", ctypes.c_int64), ("row", ctypes.c_int64)]


class Window(ctypes.Structure):
    _fields_ = [(x, ctypes.c_int64) for x in ("batch", "heads", "kv_heads", "n", "d", "left", "right", "sinks", "r_max")] + \
               [("bias", ctypes.c_void_p), ("mask", ctypes.c_void_p), ("scale", ctypes.c_float), ("dtype", ctypes.c_int32), ("bias_dtype", ctypes.c_int32)]


def _inputs(n, h, d, r, seed):
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g).to(BF16).cuda()
    q, k, v, grad = (rand(1, h, n, d) for _ in range(4))
    return q, k, v, grad, torch.randn(h, 2 * r + 1, generator=g).cuda()


def _c_interface(q, k, v, grad, bias, left, right, sinks, keep_rest):
    """The same through the C functions, with or without the residue of o."""
    lib, (b, h, n, d) = _lib.load(), q.shape
    w = Window(b, h, k.shape[1], n, d, left, right, sinks, bias.shape[1] // 2, bias.data_ptr(), None, d ** -0.5, _lib.PX_BF16, _lib.PX_F32)
    rows = lambda t: ctypes.byref(Rows(t.data_ptr(), *t.stride()[:3]))
    out = {x: torch.empty_like(t) for x, t in (("o", q), ("dq", q), ("dk", k), ("dv", v), ("drel_bias", bias))}
    rest = torch.empty_like(q) if keep_rest else None
    lse = torch.empty(lib.px_window_lse_floats(b, h, n), device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    opt = rows(rest) if keep_rest else None
    assert lib.px_window_fwd(ctypes.byref(w), rows(q), rows(k), rows(v), rows(out["o"]), opt, lse.data_ptr(), st) == 0
    size = lib.px_window_workspace_bytes(ctypes.byref(w), 1)
    work = torch.empty(size, dtype=torch.uint8, device="cuda")
    assert lib.px_window_bwd(ctypes.byref(w), rows(q), rows(k), rows(v), rows(out["o"]), opt, rows(grad), lse.data_ptr(), rows(out["dq"]), rows(out["dk"]),
                             rows(out["dv"]), out["drel_bias"].data_ptr(), work.data_ptr(), size, st) == 0
    ops.device_error_flags()
    return out


def _model(q, k, v, grad, bias, left, right, sinks):
    """Relative errors of drel_bias from the roundings that the kernels cannot do without (weights and output to bf16, all else exact), played through in 64 bits:
    as built, with delta of the rounded output, and without the correction.  The kernel takes a row's left-over out of blocks of 32 queries and 32 keys
    whose offsets are all clipped to one side."""
    n, r, dtype = q.shape[2], bias.shape[1] // 2, q.dtype
    q, k, v, grad, bias = (t.double() for t in (q, k, v, grad, bias))
    at = torch.arange(n, device="cuda")
    far = at[None, :] - at[:, None]
    bucket, block = far.clamp(-r, r) + r, at // 32 * 32
    apart = ((block[None, :] + 31 - block[:, None]) <= -r) | ((block[None, :] - block[:, None] - 31) >= r)
    logits = (q.shape[3] ** -0.5 * q @ k.transpose(-1, -2) + bias[:, bucket]).masked_fill(~visible(n, left, right, sinks, None, "cuda")[:, None], -math.inf)
    weight = (logits - logits.amax(-1, keepdim=True)).exp()
    total = weight.sum(-1, keepdim=True)
    p, exact, o = weight / total, weight @ v / total, weight.to(dtype).double() @ v / total
    kept = o.to(dtype).double()
    rest = (o - kept).to(dtype).double()

    def gradient(o, correct):
        ds = p * (grad @ v.transpose(-1, -2) - (grad * o).sum(-1, keepdim=True))
        if correct:
            ds = ds - ds.sum(-1, keepdim=True) * p * apart
        return torch.zeros_like(bias).index_add_(1, bucket.flatten(), ds.sum(0).flatten(1))

    true = gradient(exact, False)
    return [float((gradient(*x) - true).norm() / true.norm()) for x in ((kept + rest, True), (kept, True), (kept + rest, False))]


@pytest.mark.gpu
@pytest.mark.parametrize("n,h,d,left,right,sinks,r", [(300, 8, 16, 1, 0, 37, 2), (600, 4, 32, 2, 0, 64, 2), (1500, 4, 32, 2, 0, 37, 2)])
def test_both_measures_are_at_work(n, h, d, left, right, sinks, r):
    """Geometric means over eight draws: the kernel's error lies below the middle (in the logarithm) between that of the model as built and of the model with either measure left
    out, whichever is nearer; the models lie a factor of two apart."""
    logs = torch.zeros(4, dtype=torch.float64)
    for seed in range(8):
        x = _inputs(n, h, d, r, seed)
        want = reference(*x[:3], left, right, sinks, x[4], grad=x[3])["drel_bias"][0]
        got = _c_interface(*x, left, right, sinks, True)["drel_bias"].double()
        logs += torch.tensor([float((got - want).norm() / want.norm()), *_model(*x, left, right, sinks)], dtype=torch.float64).log() / 8
    here, built, no_rest, uncorrected = logs.exp().tolist()
    print(f"kernel {here:.2e}, model {built:.2e}, without the residue {no_rest:.2e}, without the correction {uncorrected:.2e}")
    assert min(no_rest, uncorrected) > 1.7 * built
    assert here <= math.sqrt(built * min(no_rest, uncorrected))


@pytest.mark.gpu
@pytest.mark.parametrize("n,h,d,left,right,sinks,r", [(300, 8, 16, 1, 0, 37, 2), (333, 2, 72, 50, 9, 3, 16), (260, 4, 40, 0, 0, 1, 1)])
def test_without_the_residue(n, h, d, left, right, sinks, r):
    """o_rest NULL: the bounds of a delta made from the rounded o hold."""
    q, k, v, grad, bias = _inputs(n, h, d, r, 5)
    got = _c_interface(q, k, v, grad, bias, left, right, sinks, False)
    check(got, reference(q, k, v, left, right, sinks, bias, grad=grad), BF16)
    full = _c_interface(q, k, v, grad, bias, left, right, sinks, True)
    assert torch.equal(got["o"], full["o"]) and torch.equal(got["dv"], full["dv"])
    leaves = [t.clone().requires_grad_() for t in (q, k, v, bias)]
    o = px.window_attention(*leaves[:3], (left, right), sinks=sinks, rel_bias=leaves[3])
    for name, t in zip(("dq", "dk", "dv", "drel_bias"), torch.autograd.grad(o, leaves, grad)):
        assert torch.equal(t, full[name]), name
