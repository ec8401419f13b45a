"""``linear_cross_entropy``: the loss of a classifying head, and its gradient, without the logits.

The reference's heads (protenix/model/modules/head.py: distances, residues, confidences) are a linear layer whose logits go to torch; over all
pairs of tokens, or over a large vocabulary, these are the largest tensor of a training step.  Here the layer and the loss are one operator:
the forward pass (``px_head_loss_fwd``) keeps two numbers of each row and tile of classes, the backward pass (``px_head_loss_bwd``) forms the
logits again, a piece of the classes at a time.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import native


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, bias: Optional[torch.Tensor] = None, ignore_index: int = -100,
                         label_smoothing: float = 0.0, reduction: str = "mean") -> torch.Tensor:
    """Softmax cross entropy of the logits x weight^T + bias with the classes ``target``; fp32, a number or (``reduction`` "none") [...] like target.

    ``x`` [..., C], bf16 or fp16, C a multiple of 8; ``weight`` [V, C] of x's type; ``bias`` [V], fp32 or of x's type; ``target`` [...], integers in
    [0, V), or ``ignore_index``: such rows have loss 0, do not count in the mean, get no gradient, and what they hold, NaN included, has no
    influence.  Any other target makes its row's loss, and the gradients that it enters, NaN.  ``label_smoothing`` e: the
    class counts 1 - e, and each class e / V more.  ``reduction``: "mean" (over the rows that count; of none NaN, with gradients of zero), "sum" or "none".

    Logits, exponentials and their sums are fp32, the sum of the losses fp64.  Sums of dx and of dW are fp32, in parts of at most 131072 (bf16) or 16384 (fp16) terms:
    what a part loses to the tensor core's cuts is below a quarter of the result's rounding.  The gradient of the logits is rounded to x's type where the
    products for x and weight take it, before the scale of the loss is applied (of losses by row, relative to the largest of their gradients); in fp16 what is
    below 2^-38 of that vanishes.  That of bias is not rounded before its sum.  Differentiable once in x, weight and bias; the gradients have their types and are the same to the bit on each call.
    """
    if not x.is_cuda:
        raise RuntimeError("linear_cross_entropy: CUDA tensors only, this package has no CPU path")
    return native.load().linear_cross_entropy(x, weight, target, bias, ignore_index, label_smoothing, reduction)
