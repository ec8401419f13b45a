"""What a backward pass of the loss takes beside its gradients."""
import ctypes

from protenix_b200 import _lib
from test_head_loss_abi import _head


def _bytes(h, *wanted):
    return _lib.load().px_head_loss_bwd_workspace_bytes(ctypes.byref(h), *wanted)


def test_no_copy_of_x():
    """Rows without what is not finite lie where dx will be; a call without dx has no such place."""
    h = _head(rows=1 << 20, c=512, x_stride=512, w_stride=512, classes=256)
    assert _bytes(h, 1, 1, 0) < 1 << 30 <= _bytes(h, 0, 1, 0)
    assert _bytes(h, 1, 0, 0) < 1 << 30
