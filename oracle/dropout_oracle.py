"""Dropout's mask from the definition, in plain Python and numpy (no torch, nothing of the package).

No counterpart in the reference: the generator is Philox 4x32 with ten rounds (Salmon et al., 2011), pinned by the numbers its
authors published (``tests/test_quant_dropout_cpu.py``).
"""

import numpy as np

M = 0xFFFFFFFF


def philox(counter, key):
    """Ten rounds of one counter of four words, in Python's whole numbers."""
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & M, (a >> 32) ^ c[3] ^ k[1], a & M]
        k = [(k[0] + 0x9E3779B9) & M, (k[1] + 0xBB67AE85) & M]
    return c


def kept(rows, cols, thresholds, seed, offset):
    """Truth values [rows, cols], which elements dropout keeps; thresholds: one whole number a row."""
    groups = -(-cols // 8)
    shape = (rows, groups)
    c = [np.broadcast_to(np.arange(groups, dtype=np.uint64), shape),
         np.broadcast_to(np.arange(rows, dtype=np.uint64)[:, None], shape),
         np.full(shape, offset & M, dtype=np.uint64), np.full(shape, offset >> 32, dtype=np.uint64)]
    low, half = np.uint64(M), np.uint64(32)
    k = [seed & M, seed >> 32]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> half) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> half) ^ c[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & M, (k[1] + 0xBB67AE85) & M]
    numbers = np.empty((*shape, 8), dtype=np.uint32)
    for i, word in enumerate(c):
        numbers[:, :, 2 * i], numbers[:, :, 2 * i + 1] = word & np.uint64(0xFFFF), word >> np.uint64(16)
    return numbers.reshape(rows, -1)[:, :cols] >= np.asarray(thresholds, dtype=np.uint32)[:, None]
