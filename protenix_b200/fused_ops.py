"""``dropout_add_rowwise``: residual + dropout(x) with the dropout mask shared along axis -3.

Mirror of protenix/model/modules/fused_ops.py:190-224.  In eval mode (or p = 0) the op is ``residual + x`` (:213-214);
the fused kernels of this package fold that add into their epilogues, and this function exists for API compatibility.
In training mode the mask of shape [..., 1, C, D] is drawn exactly as the reference's own fallback draws it
(``dropout`` of a tensor of ones, :219-223), so the same seed gives the same mask, and the scaled product and the add
run in one kernel (``px_scale_add_rowwise``), forward and backward.  CUDA tensors only.

``dropout_add`` draws its mask inside the kernel, from a counter-based generator, and stores it nowhere; it shares it along any
one axis or none (the reference's ``Dropout`` modules, protenix/model/triangular/layers.py, with or without ``batch_dim``).
"""
from typing import Optional, Union

import torch

from . import native


def dropout_add_rowwise(residual: torch.Tensor, x: torch.Tensor, p_drop: float, training: bool) -> torch.Tensor:
    if not training or p_drop == 0.0:
        return residual + x
    if not x.is_cuda:
        raise RuntimeError("dropout_add_rowwise (training): CUDA tensors only, this package has no CPU path")
    return native.load().dropout_add(residual, x, p_drop)


def dropout_add(residual: Optional[torch.Tensor], x: torch.Tensor, p_drop: float, seed: Union[int, torch.Tensor], offset: int = 0,
                shared_dim: Optional[int] = None, training: bool = True) -> torch.Tensor:
    """residual + dropout(x), with a mask that is a function of (seed, offset, place) and is stored nowhere; ``residual`` None:
    the dropped x alone.

    Which elements drop is decided by Philox4x32-10 with key ``seed`` and counter (place // 4, ``offset``): a call with the same
    two drops the same places, on any device and in any split over streams, and the backward pass draws them again.  Calls of one
    step that are to differ (layers, samples) take different offsets.  ``shared_dim``: the axis along which one decision
    holds for all (-3 for the row-wise, -2 for the column-wise dropout of a pair update).  ``seed`` as an int64 CUDA tensor (seed,
    offset) is read on the device (``offset`` is then not given), so that the replays of a captured graph drop anew when the
    tensor changes; the backward pass uses what its forward pass read.

    Kept elements are scaled by 1 / (1 - p_drop); product and sum are fp32 and are rounded once.  A dropped element contributes
    nothing whatever x holds there.  p_drop = 1 drops everything.  fp32, bf16 and fp16 CUDA tensors of any shape.
    ``training`` False: residual + x (a copy of x), after the same checks of the arguments.
    """
    if not x.is_cuda:
        raise RuntimeError("dropout_add: CUDA tensors only, this package has no CPU path")
    state = seed if isinstance(seed, torch.Tensor) else None
    if state is not None and offset != 0:
        raise RuntimeError("dropout_add: a seed tensor holds the offset, too")
    for name, v in (("seed", 0 if state is not None else seed), ("offset", offset)):
        if not isinstance(v, int) or not 0 <= v < 1 << 63:
            raise RuntimeError(f"dropout_add: {name} must be an integer in [0, 2^63), got {v!r}")
    return native.load().counter_dropout_add(residual, x, p_drop, 0 if state is not None else seed, offset, state, shared_dim, training)
