"""px_orthogonalize refuses what it cannot do by a status, before any launch."""
import ctypes

import pytest

from protenix_b200 import _lib

BUFFER = ctypes.create_string_buffer(4096)
AT = (ctypes.addressof(BUFFER) + 1023) // 1024 * 1024
ABC = (ctypes.c_float * 3)(3.4445, -4.7750, 2.0315)


@pytest.mark.parametrize("changed,status", [
    (dict(g=None), -1), (dict(out=None), -1), (dict(batch=-1), -1), (dict(m=-1), -1), (dict(n=-1), -1), (dict(abc=None), -1), (dict(steps=0), -1), (dict(steps=1001), -2),
    (dict(eps=-1.0), -1), (dict(eps=float("nan")), -1), (dict(dtype=5), -2), (dict(batch=65536), -2), (dict(m=(1 << 20) + 1), -2), (dict(n=(1 << 20) + 1), -2),
    (dict(ws=None), -1), (dict(ws=AT + 16), -1), (dict(g=AT + 2), -1), (dict(size=100), -4), (dict(batch=0), 0), (dict(m=0), 0), (dict(n=0), 0)])
def test_statuses(changed, status):
    lib = _lib.load()
    a = dict(g=AT, out=AT, batch=2, m=10, n=20, abc=ABC, steps=1, eps=1e-7, dtype=_lib.PX_F32, ws=AT, size=1 << 40)
    a.update(changed)
    assert lib.px_orthogonalize(a["g"], a["out"], a["batch"], a["m"], a["n"], a["abc"], a["steps"], a["eps"], a["dtype"], a["ws"], a["size"], None) == status


def test_workspace():
    size = _lib.load().px_orthogonalize_workspace_bytes
    assert size(0, 4, 4) == size(1, 0, 4) == size(1, 4, 0) == 0
    assert size(3, 128, 512) >= 3 * 2 * 2 * (2 * 128 * 512 + 2 * 128 * 128)
