"""px_rotary_turn refuses what it cannot do by a status, before any launch."""
import ctypes

import pytest

from protenix_b200 import _lib


class Rows(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("batch", ctypes.c_int64), ("head", ctypes.c_int64), ("row", ctypes.c_int64)]


class Rotary(ctypes.Structure):
    _fields_ = [("positions", ctypes.c_void_p), ("position_batch", ctypes.c_int64), ("position_row", ctypes.c_int64), ("position_axis", ctypes.c_int64),
                ("batch", ctypes.c_int64), ("heads", ctypes.c_int64), ("kv_heads", ctypes.c_int64), ("n", ctypes.c_int64), ("d", ctypes.c_int64),
                ("sections", ctypes.POINTER(ctypes.c_int32)), ("base", ctypes.c_double), ("axes", ctypes.c_int32), ("interleaved", ctypes.c_int32),
                ("per_axis", ctypes.c_int32), ("dtype", ctypes.c_int32)]


BUFFER = ctypes.create_string_buffer(4096)
AT = (ctypes.addressof(BUFFER) + 1023) // 1024 * 1024


def _call(sections=(8, 8), rows=None, k=True, **changed):
    held = (ctypes.c_int32 * len(sections))(*sections)
    f = dict(positions=AT, position_batch=0, position_row=2, position_axis=1, batch=2, heads=4, kv_heads=2 if k else 0, n=10, d=32, sections=held, base=1e4,
             axes=len(sections), interleaved=0, per_axis=0, dtype=_lib.PX_F32)
    f.update(changed)
    r, x = Rotary(**f), Rows(**{**dict(data=AT, batch=1280, head=320, row=32), **(rows or {})})
    p = ctypes.byref(x)
    return _lib.load().px_rotary_turn(ctypes.byref(r), p, p, p if k else None, p if k else None, 0, None)


@pytest.mark.parametrize("changed,status", [
    (dict(batch=-1), -1), (dict(heads=0), -1), (dict(kv_heads=-1), -1), (dict(kv_heads=0), -1), (dict(n=-1), -1), (dict(d=1), -1), (dict(sections=(8, -1)), -1),
    (dict(sections=(16, 1)), -1), (dict(sections=(0, 0)), -1), (dict(sections=(200, 100), d=1024), -2), (dict(base=0.9), -1), (dict(base=float("nan")), -1),
    (dict(base=1e31), -1), (dict(axes=0), -1), (dict(dtype=7), -2), (dict(positions=None), -1), (dict(rows=dict(data=None)), -1), (dict(rows=dict(data=AT + 1)), -1),
    (dict(batch=65536), -2), (dict(n=(1 << 30) + 1), -2), (dict(d=65537), -2), (dict(k=False, kv_heads=2), -1), (dict(batch=0), 0), (dict(n=0), 0)])
def test_statuses(changed, status):
    assert _call(**changed) == status


def test_null():
    assert _lib.load().px_rotary_turn(None, None, None, None, None, 0, None) == -1
