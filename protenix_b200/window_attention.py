"""``window_attention``: attention in which a token sees its neighbours in the sequence and a few first tokens.

The reference's local attention (protenix/model/modules/primitives.py, ``n_queries`` / ``n_keys``; atoms in the encoder and decoder) gives
blocks of queries blocks of keys; here the window moves with the query.  Forward and backward are tcgen05 kernels
(``px_window_fwd``, ``px_window_bwd``) that only touch the tiles that a window reaches; neither a mask nor a bias matrix exists.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import native


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: Union[int, Tuple[int, int]], sinks: int = 0,
                     rel_bias: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """softmax(scale q k^T + bias) v over the keys that a query sees; [..., H, N, D] like q.

    ``q`` [..., H, N, D], ``k`` and ``v`` [..., H_kv, N, D] (H_kv divides H: query head h reads head h // (H / H_kv)), bf16 or fp16, D a multiple
    of 8 up to 128.  Views are taken as they are (heads inside the rows of one projection, say); what the kernels cannot
    address (broadcast axes, rows that overlap or do not begin on 16 bytes) is copied.  The output lies in memory like q: heads inside the rows where q's are.

    Query i sees key j when j <= i + right and (j >= i - left or j < sinks), ``window`` = (left, right) or one number for both, and
    ``mask`` [..., N] (any type, nonzero = there) holds at j.  right = 0 is causal.  A query that sees nothing gives zeros and no gradient,
    and what masked keys and such queries hold, NaN included, has no influence.  (A NaN or an infinity elsewhere may reach
    all queries, and in the backward pass all keys, of its tile of 128.)

    ``rel_bias`` [H, 2 r + 1], fp32 or of q's type, r up to 256: learned, added to the logits by the clipped offset, entry
    clip(j - i, -r, r) + r; an entry of minus infinity, or one that is times log2(e) (fp32 below -2.35e38), hides its offset like a mask.  ``scale``: positive,
    default D ** -0.5.

    Logits, softmax and sums are fp32; the weights, and their gradients, are rounded to q's type where a product takes them.  A gradient that
    fp16 cannot hold, on the way to the result or as such, comes out infinite or NaN, so that a loss scaler finds it.  Differentiable
    once in q, k, v and rel_bias; the gradients are the same to the bit on each call.
    """
    left, right = (window, window) if isinstance(window, int) else window
    if not q.is_cuda:
        raise RuntimeError("window_attention: CUDA tensors only, this package has no CPU path")
    return native.load().window_attention(q, k, v, left, right, sinks, rel_bias, mask, scale)
