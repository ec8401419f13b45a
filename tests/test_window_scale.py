"""Scales that windowed attention refuses."""


def test_a_scale_that_is_infinite_in_base_two_is_refused():
    """The kernels multiply by scale * log2(e) (no GPU needed)."""
    import ctypes

    from protenix_b200 import _lib

    class Window(ctypes.Structure):
        _fields_ = [(x, ctypes.c_int64) for x in ("batch", "heads", "kv_heads", "n", "d", "left", "right", "sinks", "r_max")] + \
                   [("bias", ctypes.c_void_p), ("mask", ctypes.c_void_p), ("scale", ctypes.c_float), ("dtype", ctypes.c_int32), ("bias_dtype", ctypes.c_int32)]

    size = lambda scale: _lib.load().px_window_workspace_bytes(ctypes.byref(Window(1, 2, 2, 10, 32, 3, 0, 0, -1, None, None, scale, _lib.PX_BF16, 0)), 0)
    assert size(1.0) > 0 and size(2.3e38) > 0
    assert size(2.4e38) == 0 and size(2.9e38) == 0
