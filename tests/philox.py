"""Philox4x32-10 in numpy, from its definition (Salmon, Moraes, Dror and Shaw,
"Parallel random numbers: as easy as 1, 2, 3", SC 2011)."""
import numpy as np

LOW, HALF = np.uint64(0xFFFFFFFF), np.uint64(32)


def blocks(counter, key, rounds=10):
    """counter: four uint64 arrays of 32-bit words; key: two 32-bit ints."""
    c = [np.asarray(x, np.uint64) for x in counter]
    for r in range(rounds):
        k0 = np.uint64((key[0] + r * 0x9E3779B9) & 0xFFFFFFFF)
        k1 = np.uint64((key[1] + r * 0xBB67AE85) & 0xFFFFFFFF)
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> HALF) ^ c[1] ^ k0, b & LOW, (a >> HALF) ^ c[3] ^ k1, a & LOW]
    return np.stack(c, axis=-1)


def words(n, seed, call, first=0):
    """The words of elements first .. first + n - 1 of a dropout call."""
    i = np.arange(first // 4, (first + n + 3) // 4, dtype=np.uint64)
    call &= 0xFFFFFFFFFFFFFFFF
    c = blocks([i & LOW, i >> HALF, np.full_like(i, call & 0xFFFFFFFF), np.full_like(i, call >> 32)],
               (seed & 0xFFFFFFFF, seed >> 32))
    return c.reshape(-1)[first % 4:][:n]
