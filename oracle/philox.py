"""The counter-based dropout masks in NumPy (TEST INFRASTRUCTURE): Philox-4x32 with ten rounds
(Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011) and the
counter layout that include/talm.h documents."""

import numpy as np

_LOW = np.uint64(0xffffffff)
_WORD = np.uint64(32)


def philox4x32(counter, key, rounds=10):
    """counter: four uint64 arrays holding 32-bit words; key: two 32-bit ints. Four uint64 arrays
    holding the block's words."""
    c = [np.asarray(w, np.uint64) & _LOW for w in counter]
    k0, k1 = int(key[0]), int(key[1])
    for _ in range(rounds):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> _WORD) ^ c[1] ^ np.uint64(k0), b & _LOW,
             (a >> _WORD) ^ c[3] ^ np.uint64(k1), a & _LOW]
        k0, k1 = (k0 + 0x9E3779B9) % 2 ** 32, (k1 + 0xBB67AE85) % 2 ** 32
    return c


def threshold(p):
    return min(int(np.floor(np.float64(np.float32(p)) * 65536 + 0.5)), 65535)


def factor(p):
    """What a kept element is multiplied by (float32, as the kernels hold it)."""
    return np.float32(65536) / np.float32(65536 - threshold(p))


def keep(key, rows, cols, p, site=0):
    """bool [rows, cols]: the elements a dropout with this key (two ints) and site keeps."""
    key = [int(k) % 2 ** 64 for k in key]
    block = np.arange(rows * -(-cols // 8), dtype=np.uint64)
    words = philox4x32((block, block >> _WORD, np.full_like(block, site),
                        np.full_like(block, key[1] % 2 ** 32)),
                       (key[0] % 2 ** 32, key[0] >> 32))
    bits = np.stack(words, 1).astype("<u4").view("<u2").reshape(rows, -1)[:, :cols]
    return bits.astype(np.int64) >= threshold(p)
