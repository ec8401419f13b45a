"""``orthogonalize``: matrices with their singular values driven towards one, and ``Muon``, the optimiser that takes such updates.

The weights of a Pairformer stack are matrices, many of one shape (128 x 128, 512 x 128 and 128 x 512 in the pair path of each block, 384 x 384 to 1536 x
384 in the single one).  A momentum whose singular values are made alike moves all directions of a weight by the same amount.  The
polynomial iteration (Newton-Schulz) needs products only; ``px_orthogonalize`` runs it for all matrices of a shape at once.
"""
from __future__ import annotations

from typing import Iterable, Optional, Sequence, Tuple, Union

import torch

from . import native

Coefficients = Union[Tuple[float, float, float], Sequence[Tuple[float, float, float]]]
DEFAULT = (3.4445, -4.7750, 2.0315)


def orthogonalize(g: torch.Tensor, steps: int = 5, coefficients: Coefficients = DEFAULT, eps: float = 1e-7) -> torch.Tensor:
    """Each matrix of ``g`` [..., M, N] with its singular values near one; a new tensor of g's shape and type (fp32, bf16 or fp16).

    X = g / (|g| + eps), |g| the root of the sum of squares, then ``steps`` times X <- a X + b (X X^T) X + c (X X^T)^2 X with (a, b, c) =
    ``coefficients``, or one triple for each step (``steps`` is then their number).  The default triple takes singular values above 0.01 |g| to
    between 0.7 and 1.2 in five steps.

    Products take operands of 22 bits and add in fp32 whatever the type: 16-bit iterates lose up to a third of the result where singular values differ
    much.  Iterates and polynomials of up to 60 are held; an overflow comes out infinite or NaN.  A matrix that is not finite gives NaN, a zero one zero (eps > 0).
    Not differentiable: g is detached or no_grad is in force.
    """
    if not g.is_cuda:
        raise RuntimeError("orthogonalize: CUDA tensors only, this package has no CPU path")
    triples = [tuple(c) for c in coefficients] if not isinstance(coefficients[0], (int, float)) else [tuple(coefficients)] * int(steps)
    if any(len(c) != 3 for c in triples):
        raise RuntimeError("orthogonalize: coefficients are triples (a, b, c)")
    return native.load().orthogonalize(g, [float(x) for c in triples for x in c], eps)
