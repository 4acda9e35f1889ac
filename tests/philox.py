"""Dropout's numbers for the tests: Philox4x32-10 (Salmon, Moraes, Dror, Shaw 2011) on the host."""
import numpy as np


def philox4x32(counter, key):
    """counter: whole numbers [n] (the low 64 bits of the 128), key: a 64-bit number -> uint32 [n, 4]."""
    m = np.uint64(0xFFFFFFFF)
    counter = np.asarray(counter, dtype=np.uint64)
    a, b = counter & m, counter >> np.uint64(32)
    c, d = np.zeros_like(a), np.zeros_like(a)
    for r in range(10):
        k = [np.uint64((key + r * 0x9E3779B9) & 0xFFFFFFFF), np.uint64(((key >> 32) + r * 0xBB67AE85) & 0xFFFFFFFF)]
        x, y = np.uint64(0xD2511F53) * a, np.uint64(0xCD9E8D57) * c
        a, b, c, d = (y >> np.uint64(32)) ^ b ^ k[0], y & m, (x >> np.uint64(32)) ^ d ^ k[1], x & m
    return np.stack([a, b, c, d], -1).astype(np.uint32)


def kept(n, p, seed):
    """Which of n elements (a multiple of 8) are kept, and the factor of those."""
    draws = philox4x32(np.arange(n // 8), seed & (2 ** 64 - 1)).astype("<u4").view("<u2").reshape(-1)
    cut = int(p * 65536 + 0.5)
    return draws >= cut, 65536 / (65536 - cut)
