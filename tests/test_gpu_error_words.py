"""px_device_error_detail writes as many words as it always has, whatever families have come since; px_device_error_words as many as it is asked for."""
import ctypes

import pytest
import torch

from protenix_b200 import _lib, ops


@pytest.mark.gpu
def test_words_beyond_the_sixteen_are_left_alone():
    torch.zeros(1, device="cuda")
    flags, detail = ctypes.c_uint32(7), (ctypes.c_uint32 * 32)(*[0xABCD] * 32)
    assert _lib.load().px_device_error_detail(ctypes.byref(flags), detail) == 0
    assert flags.value == 0 and not any(detail[:16]) and all(v == 0xABCD for v in detail[16:])


@pytest.mark.gpu
@pytest.mark.parametrize("count", [0, 1, 16, len(ops.KERNEL_FAMILIES), 32])
def test_words_by_count(count):
    torch.zeros(1, device="cuda")
    flags, detail = ctypes.c_uint32(7), (ctypes.c_uint32 * 40)(*[0xABCD] * 40)
    assert _lib.load().px_device_error_words(ctypes.byref(flags), detail, count) == 0
    n = min(count, len(ops.KERNEL_FAMILIES))
    assert flags.value == 0 and not any(detail[:n]) and all(v == 0xABCD for v in detail[n:])


def test_bad_arguments():
    lib = _lib.load()
    flags, detail = ctypes.c_uint32(0), (ctypes.c_uint32 * 4)()
    assert lib.px_device_error_words(None, detail, 4) == -1
    assert lib.px_device_error_words(ctypes.byref(flags), detail, -1) == -1
    assert lib.px_device_error_words(ctypes.byref(flags), None, 4) == -1
    assert lib.px_version() >= 101
