"""Dropout's mask from the definition, in plain Python and numpy (no torch, nothing of the package)."""

import numpy as np

M = 0xFFFFFFFF


def philox(counter, key):
    """Philox 4x32 with ten rounds of one counter of four words, in Python's whole numbers."""
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & M, (a >> 32) ^ c[3] ^ k[1], a & M]
        k = [(k[0] + 0x9E3779B9) & M, (k[1] + 0xBB67AE85) & M]
    return c


def kept(rows, cols, thresholds, seed, offset):
    """Truth values [rows, cols]; thresholds: one whole number a row."""
    out = np.empty((rows, cols), dtype=bool)
    for t in range(rows):
        for g in range(-(-cols // 8)):
            words = philox((g, t, offset & M, offset >> 32), (seed & M, seed >> 32))
            for i in range(min(8, cols - 8 * g)):
                out[t, 8 * g + i] = (words[i // 2] >> (16 * (i % 2)) & 0xFFFF) >= thresholds[t]
    return out
