"""The tests' generator against the published known answers of Philox4x32-10."""
import numpy as np
import pytest

from philox import keep, philox

KNOWN = [
    ([0] * 4, [0] * 2, [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]),
    ([0xffffffff] * 4, [0xffffffff] * 2, [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]),
    ([0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344], [0xa4093822, 0x299f31d0], [0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1]),
]


@pytest.mark.parametrize("counter,key,want", KNOWN)
def test_known_answers(counter, key, want):
    assert [int(w) for w in philox(counter, key)] == want


def test_rate_of_kept_elements():
    k = keep((1 << 20,), 0.1, 7, 3)
    assert abs(k.mean() - 0.9) < 5 * np.sqrt(0.09 / k.size)      # five standard deviations
    assert keep((5, 3), 0.0, 1, 0).all() and not keep((5, 3), 1.0, 1, 0).any()
