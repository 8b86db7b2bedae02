"""The dropout draw restated: Philox-4x32-10 (Salmon, Moraes, Dror, Shaw, SC 2011) in numpy's unsigned integers."""
import numpy as np


def philox(c, key):
    """c: four uint64 arrays of 32-bit words -> four of the same"""
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    k = [int(key[0]), int(key[1])]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> half) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> half) ^ c[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    return c


def numbers(first_group, groups, seed, offset, step=0):
    """[groups, 8] 16-bit numbers of the elements of groups first_group, first_group + 1, ..."""
    g = np.arange(first_group, first_group + groups, dtype=np.uint64)
    full = lambda v: np.full(groups, v, dtype=np.uint64)  # noqa: E731
    words = philox([g & np.uint64(0xFFFFFFFF), g >> np.uint64(32), full(offset), full(step)], (seed % 2 ** 32, seed >> 32))
    return np.stack([(w >> np.uint64(s)) & np.uint64(0xFFFF) for w in words for s in (0, 16)], 1)


def factor(shape, threshold, seed, offset, step=0, first_group=0):
    """What each element of a tensor is multiplied by, in fp64."""
    n = int(np.prod(shape)) // 8
    kept = numbers(first_group, n, seed, offset, step) >= threshold
    return np.where(kept, 65536 / (65536 - threshold) if threshold < 65536 else 0.0, 0.0).reshape(shape)
