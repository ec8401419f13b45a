"""The workspace of px_orthogonalize."""
import ctypes

import pytest

from protenix_b200 import _lib


@pytest.mark.parametrize("batch,m,n", [(65535, 8, 8), (65535, 16, 16), (1, 4096, 4096), (24, 384, 1536), (1, 300, 300), (500, 200, 300), (3, 1, 1)])
def test_planes_and_a_few_sums(batch, m, n):
    """Two iterates, A and the polynomial in two fp16 planes with rows of whole 16 bytes; beside them a sum for each 2048 elements at most, and no part of A in more
    places than there are SMs."""
    up = lambda x: (x + 7) // 8 * 8  # noqa: E731
    s = min(m, n)
    planes = batch * 2 * 2 * (2 * m * up(n) + 2 * s * up(s))
    size = _lib.load().px_orthogonalize_workspace_bytes(batch, m, n)
    assert planes <= size <= planes + 8 * batch * ((m * n + 2047) // 2048) + 148 * 4 * 128 * 136 + 8 * 1024


@pytest.mark.parametrize("batch,m,n", [(48, 128, 128), (48, 512, 128), (148, 64, 64), (1, 1, 1)])
def test_one_launch_takes_none(batch, m, n):
    """Short sides of up to 128 keep everything on the chip, up to 32 steps; the query without steps is for any number of them."""
    lib = _lib.load()
    most = lib.px_orthogonalize_workspace_bytes(batch, m, n)
    assert lib.px_orthogonalize_steps_workspace_bytes(batch, m, n, 5) == 1024
    assert lib.px_orthogonalize_steps_workspace_bytes(batch, m, n, 33) == most
    assert lib.px_orthogonalize_steps_workspace_bytes(batch, 200, 300, 5) == lib.px_orthogonalize_workspace_bytes(batch, 200, 300)
    assert lib.px_orthogonalize_steps_workspace_bytes(0, m, n, 5) == lib.px_orthogonalize_steps_workspace_bytes(batch, 0, n, 5) == 0


def test_too_small():
    buffer = ctypes.create_string_buffer(4096)
    at = (ctypes.addressof(buffer) + 1023) // 1024 * 1024
    abc = (ctypes.c_float * (3 * 33))(*[1.5, -0.5, 0.0] * 33)
    lib = _lib.load()
    for steps in (5, 33):
        for m, n in ((10, 20), (200, 300)):
            size = lib.px_orthogonalize_steps_workspace_bytes(2, m, n, steps)
            assert lib.px_orthogonalize(at, at, 2, m, n, abc, steps, 1e-7, _lib.PX_F32, at, size - 1, None) == -4
