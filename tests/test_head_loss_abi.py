"""px_head_loss_* refuse what they cannot do by a status, before any launch."""
import ctypes

import pytest

from protenix_b200 import _lib


class Head(ctypes.Structure):
    _fields_ = [("x", ctypes.c_void_p), ("w", ctypes.c_void_p), ("bias", ctypes.c_void_p), ("target", ctypes.c_void_p), ("rows", ctypes.c_int64),
                ("c", ctypes.c_int64), ("classes", ctypes.c_int64), ("x_stride", ctypes.c_int64), ("w_stride", ctypes.c_int64), ("ignore", ctypes.c_int64),
                ("smoothing", ctypes.c_float), ("dtype", ctypes.c_int32), ("bias_dtype", ctypes.c_int32)]


BUFFER = ctypes.create_string_buffer(4096)
AT = (ctypes.addressof(BUFFER) + 1023) // 1024 * 1024


def _head(**changed):
    h = dict(x=AT, w=AT, bias=None, target=AT, rows=10, c=64, classes=20, x_stride=64, w_stride=64, ignore=-100, smoothing=0.0, dtype=_lib.PX_BF16, bias_dtype=_lib.PX_F32)
    h.update(changed)
    return Head(**h)


@pytest.mark.parametrize("changed,status", [
    (dict(rows=-1), -1), (dict(c=0), -1), (dict(classes=0), -1), (dict(x=None), -1), (dict(w=None), -1), (dict(target=None), -1), (dict(x_stride=56), -1),
    (dict(w_stride=68), -1), (dict(x=AT + 2), -1), (dict(w=AT + 8), -1), (dict(bias=AT + 4), -1), (dict(smoothing=1.5), -1), (dict(smoothing=float("nan")), -1),
    (dict(dtype=_lib.PX_F32), -2), (dict(bias_dtype=_lib.PX_F16), -2), (dict(c=60), -2), (dict(classes=(1 << 24) + 1), -2), (dict(rows=(1 << 26) + 1), -2), (dict(rows=1 << 26, classes=1 << 24), -2)])
def test_heads(changed, status):
    lib, h = _lib.load(), _head(**changed)
    assert lib.px_head_loss_fwd(ctypes.byref(h), AT, AT, AT, AT, 1, AT, 1 << 40, None) == status
    assert lib.px_head_loss_bwd(ctypes.byref(h), AT, AT, 0, AT, AT, AT, AT, AT, 1 << 40, None) == status


def test_other_arguments():
    lib, h = _lib.load(), _head()
    p = ctypes.byref(h)
    size = lib.px_head_loss_workspace_bytes(10, 20)
    assert size > 0 and lib.px_head_loss_workspace_bytes(0, 20) == 0
    assert lib.px_head_loss_fwd(None, AT, AT, AT, AT, 1, AT, size, None) == -1
    assert lib.px_head_loss_fwd(p, None, AT, AT, AT, 1, AT, size, None) == -1
    assert lib.px_head_loss_fwd(p, AT, None, None, AT, 1, AT, size, None) == -1
    assert lib.px_head_loss_fwd(p, AT, None, AT, None, 1, AT, size, None) == -1
    assert lib.px_head_loss_fwd(p, AT, AT, AT, AT, 1, None, size, None) == -1
    assert lib.px_head_loss_fwd(p, AT, AT, AT, AT, 1, AT + 16, size, None) == -1
    assert lib.px_head_loss_fwd(p, AT, AT, AT, AT, 1, AT, size - 1, None) == -4
    size = lib.px_head_loss_bwd_workspace_bytes(p, 1, 1, 1)
    assert size > 0 and lib.px_head_loss_bwd_workspace_bytes(None, 1, 1, 1) == 0
    assert lib.px_head_loss_bwd(p, None, AT, 0, AT, AT, AT, AT, AT, size, None) == -1
    assert lib.px_head_loss_bwd(p, AT, None, 0, AT, AT, AT, AT, AT, size, None) == -1
    assert lib.px_head_loss_bwd(p, AT, AT, 0, None, AT, AT, AT, AT, size, None) == -1
    assert lib.px_head_loss_bwd(p, AT, AT, 0, AT, AT + 2, AT, AT, AT, size, None) == -1
    assert lib.px_head_loss_bwd(p, AT, AT, 0, AT, AT, AT, AT, None, size, None) == -1
    assert lib.px_head_loss_bwd(p, AT, AT, 0, AT, AT, AT, AT, AT, size - 1, None) == -4


def test_pieces_bound_the_workspace():
    """16 bits a logit up to 512 MiB, however many classes there are."""
    lib = _lib.load()
    small = lib.px_head_loss_bwd_workspace_bytes(ctypes.byref(_head(rows=8192, classes=32768)), 0, 0, 0)
    large = lib.px_head_loss_bwd_workspace_bytes(ctypes.byref(_head(rows=8192, classes=1 << 20)), 0, 0, 0)
    assert 512 << 20 <= small <= large <= (512 << 20) + (1 << 20)
