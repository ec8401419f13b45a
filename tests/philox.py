"""Philox4x32-10 (Salmon, Moraes, Dror, Shaw, 2011) in numpy, for the tests of the dropout that draws from it."""
import numpy as np

LOW, SHIFT = np.uint64(0xFFFFFFFF), np.uint64(32)


def philox(counter, key):
    """counter: four arrays or ints, key: two ints, all of 32 bits; the four output words."""
    x = [np.asarray(c, dtype=np.uint64) for c in counter]
    for r in range(10):
        k = [np.uint64((key[0] + r * 0x9E3779B9) & 0xFFFFFFFF), np.uint64((key[1] + r * 0xBB67AE85) & 0xFFFFFFFF)]
        a, b = np.uint64(0xD2511F53) * x[0], np.uint64(0xCD9E8D57) * x[2]
        x = [(b >> SHIFT) ^ x[1] ^ k[0], b & LOW, (a >> SHIFT) ^ x[3] ^ k[1], a & LOW]
    return x


def keep(shape, p, seed, offset, shared_dim=None):
    """Truth values of ``shape`` (the shared axis of length one): which elements a dropout of probability p keeps."""
    shape = list(shape)
    if shared_dim is not None:
        shape[shared_dim] = 1
    n = int(np.prod(shape))
    block = np.arange(-(-n // 4), dtype=np.uint64)
    words = philox([block & LOW, block >> SHIFT, np.full_like(block, offset & 0xFFFFFFFF), np.full_like(block, offset >> 32)],
                   (seed & 0xFFFFFFFF, seed >> 32))
    u = np.stack(words, -1).reshape(-1)[:n]
    return (u >= np.uint64(round(p * 2 ** 32))).reshape(shape)
