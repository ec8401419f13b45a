"""Views whose rows overlap, as unfold makes them: windowed attention copies them, and the C functions refuse them."""
import ctypes

import pytest
import torch

import protenix_b200 as px

BF16 = torch.bfloat16


@pytest.mark.gpu
@pytest.mark.parametrize("step", [8, 16])
def test_overlapping_rows(step):
    n, d = 150, 32
    line = torch.randn(2, 3, step * (n - 1) + d, device="cuda").to(BF16)
    rows = lambda t: t.unfold(2, d, step)
    k, v = (torch.randn(2, 3, n, d, device="cuda").to(BF16) for _ in range(2))
    assert rows(line).shape == (2, 3, n, d) and rows(line).stride(2) == step
    for order in ((line, k, v), (k, line, v), (k, v, line)):
        views = [rows(t) if t is line else t for t in order]
        leaves = [t.contiguous().clone().requires_grad_() for t in views]
        want = px.window_attention(*leaves, 20)
        base = line.clone().requires_grad_()
        got = px.window_attention(*(rows(base) if t is line else t for t in order), 20)
        assert torch.equal(got, want)
        assert torch.equal(px.window_attention(*views, 20), want)
        grad = torch.randn(2, 3, n, d, device="cuda").to(BF16)
        dline, = torch.autograd.grad(got, base, grad)
        dview = torch.autograd.grad(want, leaves, grad)[[t is line for t in order].index(True)]
        again = line.clone().requires_grad_()
        assert torch.equal(dline, torch.autograd.grad(rows(again), again, dview)[0])


def test_the_c_functions_refuse_them():
    from protenix_b200 import _lib

    class Rows(ctypes.Structure):
        _fields_ = [("data", ctypes.c_void_p), ("batch", ctypes.c_int64), ("head", ctypes.c_int64), ("row", ctypes.c_int64)]

    class Window(ctypes.Structure):
        _fields_ = [(x, ctypes.c_int64) for x in ("batch", "heads", "kv_heads", "n", "d", "left", "right", "sinks", "r_max")] + \
                   [("bias", ctypes.c_void_p), ("mask", ctypes.c_void_p), ("scale", ctypes.c_float), ("dtype", ctypes.c_int32), ("bias_dtype", ctypes.c_int32)]

    buf = ctypes.create_string_buffer(256)
    at = (ctypes.addressof(buf) + 15) // 16 * 16
    w, good = Window(1, 4, 2, 10, 32, 3, 0, 0, -1, None, None, 1.0, _lib.PX_BF16, 0), Rows(at, 1280, 320, 32)
    for bad in (Rows(at, 1280, 320, 24), Rows(at, 1280, 8, 128)):
        for place in range(4):
            rows = [ctypes.byref(bad if i == place else good) for i in range(4)]
            assert _lib.load().px_window_fwd(ctypes.byref(w), *rows, None, None, None) == -1
