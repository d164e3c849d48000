"""Philox4x32-10 (Salmon, Moraes, Dror, Shaw 2011) in whole numbers on the host, and the dropout's rule on it."""
import math

import numpy as np

WORD = 0xFFFFFFFF


def philox(counter, key):
    """Four words of 32 bits (arrays or numbers) under a key of two."""
    c = [np.asarray(v, dtype=np.uint64) for v in counter]
    k = [int(v) for v in key]
    low, half = np.uint64(WORD), np.uint64(32)
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [b >> half ^ c[1] ^ np.uint64(k[0]), b & low, a >> half ^ c[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & WORD, (k[1] + 0xBB67AE85) & WORD]
    return c


def keep_mask(rows, width, p, seed, offset):
    """Which values of a matrix the dropout keeps."""
    groups = (width + 3) // 4
    seed, offset = seed & (1 << 64) - 1, offset & (1 << 64) - 1
    col, row = np.meshgrid(np.arange(groups), np.arange(rows))
    words = philox([col, row, np.full_like(col, offset & WORD), np.full_like(col, offset >> 32)], [seed & WORD, seed >> 32])
    return np.stack(words, axis=2).reshape(rows, groups * 4)[:, :width] >= math.floor(p * 2 ** 32)
