"""``rotary_embedding``: positions of queries and keys as rotations of their channels, on one axis or several.

The reference's attention takes positions as a bias of pairs (protenix/model/modules/embedders.py); where no pair tensor exists, as in local
attention over atoms or long chains (``window_attention``), queries and keys that are turned by their positions give logits that depend on the
offsets alone.  Residue, atom and chain number (or time, height and width) are axes, each with its share of a head's channels.  One kernel
(``px_rotary_turn``) turns q and k, forward and, by the negated angles, backward.
"""
from __future__ import annotations

from typing import Optional, Sequence, Tuple, Union

import torch

from . import native


def rotary_embedding(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, sections: Optional[Sequence[int]] = None, base: float = 10000.0,
                     interleaved: bool = False, per_axis: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """(q, k) turned by their positions; ``k`` None: q alone.

    ``q`` [..., H, N, D] and ``k`` [..., H_kv, N, D], fp32, bf16 or fp16 (views are taken as they are; the outputs lie in memory like
    them: heads inside the rows where theirs are); ``positions`` [..., N, A], integers that int64 holds, over the batch axes of q or broadcast
    along them.  ``sections``: how many pairs of channels each of the A axes turns, in the order of the pairs (default, for one axis:
    all D // 2).  P = sum(sections) pairs are (j, j + P), or with ``interleaved`` (2 j, 2 j + 1); the channels from 2 P on stay as they are.

    Pair j turns by positions[axis] * base ** -(j / P): one ladder of speeds through all axes.  ``per_axis``: each axis has the whole ladder,
    base ** -(i / S) for the i-th of its S pairs.  Far positions keep their angles: they are off by 2^-31 of a turn up to 2^57, by 2^-25 up to 2^63.  Products are
    fp32, rounded once.  Differentiable any number of times in q and k (the operator is linear).
    """
    if not q.is_cuda:
        raise RuntimeError("rotary_embedding: CUDA tensors only, this package has no CPU path")
    if sections is None:
        if positions.dim() < 1 or positions.shape[-1] != 1:
            raise RuntimeError("rotary_embedding: positions of several axes need sections")
        sections = (q.shape[-1] // 2,)
    return native.load().rotary_embedding(q, k, positions, [int(s) for s in sections], base, interleaved, per_axis)
