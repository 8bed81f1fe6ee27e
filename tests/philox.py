"""Philox 4x32-10 in numpy, the generator of the dropout's masks (Salmon et al.,
SC 2011): word i % 4 of the counter (i / 4, offset) under the key ``seed``."""

from __future__ import annotations

import numpy as np

LOW = np.uint64(0xFFFFFFFF)


def block(counter, key, rounds: int = 10):
    """The four words of each counter, a (4, ...) array of 32-bit values."""
    c = [np.asarray(x, np.uint64) for x in counter]
    k = [int(x) for x in key]
    for _ in range(rounds):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & LOW, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & LOW]
        k = [(k[0] + 0x9E3779B9) % 2**32, (k[1] + 0xBB67AE85) % 2**32]
    return np.stack(c)


def words(n: int, seed: int, offset: int) -> np.ndarray:
    i = np.arange((n + 3) // 4, dtype=np.uint64)
    full = lambda v: np.full_like(i, v)  # noqa: E731
    c = (i & LOW, i >> np.uint64(32), full(offset % 2**32), full(offset // 2**32))
    return block(c, (seed % 2**32, seed // 2**32)).T.reshape(-1)[:n]
