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
