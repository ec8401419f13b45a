"""``RelativePositionEncoding``: what the pair representation starts from, a learned bias by buckets of relative position.

AlphaFold 3's algorithm 3 under the name and parameters of the reference's module (protenix/model/modules/embedders.py): for each
pair of tokens the clipped differences of residue number (within a chain), of token number (within a residue) and of copy number
(between copies of an entity) and the flag "same entity" pick rows of one weight, which are added up.  Neither the one-hot
vectors nor their product exist: ``px_relpos_fwd`` writes the sum of two table rows a pair, ``px_relpos_bwd`` adds the gradient up
by buckets, in a fixed order.
"""
from __future__ import annotations

from typing import Dict, Optional

import torch
import torch.nn as nn

from . import native
from .primitives import LinearNoBias

FEATURES = ("asym_id", "residue_index", "entity_id", "token_index", "sym_id")


def relative_position_encoding(weight: torch.Tensor, asym_id: torch.Tensor, residue_index: torch.Tensor, entity_id: torch.Tensor,
                               token_index: torch.Tensor, sym_id: torch.Tensor, r_max: int = 32, s_max: int = 2,
                               dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """z [..., N, N, c] of ``dtype`` (default: the weight's) for features [..., N] (integer tensors).

    ``weight``: [c, 4 r_max + 2 s_max + 7], columns in the reference's order: residue offsets -r_max .. r_max and "another chain",
    token offsets likewise, "same entity", copy offsets -s_max .. s_max and "another entity".  c is a multiple of 8.  Sums are
    fp32 whatever the types; the gradient of ``weight`` is the same to the bit on each call.  A gradient of z that is infinite or NaN makes its channel of
    ``weight``'s gradient so: the columns of its pair for an fp32 z, all of them for a 16-bit one.
    """
    return native.load().relative_position_encoding(weight, [asym_id, residue_index, entity_id, token_index, sym_id], r_max, s_max, dtype)


class RelativePositionEncoding(nn.Module):
    def __init__(self, r_max: int = 32, s_max: int = 2, c_z: int = 128) -> None:
        super().__init__()
        self.r_max = r_max
        self.s_max = s_max
        self.c_z = c_z
        self.linear_no_bias = LinearNoBias(in_features=4 * r_max + 2 * s_max + 7, out_features=c_z)

    def forward(self, input_feature_dict: Dict[str, torch.Tensor], dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        """``input_feature_dict``: at least the five features, [..., N_token].  Returns [..., N_token, N_token, c_z]."""
        missing = [k for k in FEATURES if k not in input_feature_dict]
        if missing:
            raise RuntimeError(f"RelativePositionEncoding needs the features {', '.join(missing)}")
        return relative_position_encoding(self.linear_no_bias.weight, **{k: input_feature_dict[k] for k in FEATURES},
                                          r_max=self.r_max, s_max=self.s_max, dtype=dtype)
