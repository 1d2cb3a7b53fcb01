"""Philox-4x32-10 (Salmon, Moraes, Dror, Shaw, 2011) in numpy, for the dropout tests."""
import numpy as np


def philox(counter, key):
    """counter: uint64 [n, 2] (block, offset); key: int.  uint32 [n, 4]."""
    m = np.uint64(0xFFFFFFFF)
    s = np.uint64(32)
    c = [counter[:, 0] & m, counter[:, 0] >> s, counter[:, 1] & m, counter[:, 1] >> s]
    k0, k1 = key & 0xFFFFFFFF, key >> 32
    for _ in range(10):
        p, q = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(q >> s) ^ c[1] ^ np.uint64(k0), q & m, (p >> s) ^ c[3] ^ np.uint64(k1), p & m]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack(c, 1).astype(np.uint32)


def keep_mask(first, n, p, seed, offset):
    """bool [n]: whether elements first .. first + n - 1 are kept."""
    e = np.arange(first, first + n, dtype=np.uint64)
    blocks = np.unique(e >> np.uint64(3))
    w = philox(np.stack([blocks, np.full_like(blocks, np.uint64(offset))], 1), seed)
    halves = np.stack([w & np.uint32(0xFFFF), w >> np.uint32(16)], -1).reshape(-1)
    base = int(blocks[0]) * 8
    return halves[first - base:first - base + n] >= int(p * 65536.0 + 0.5)
