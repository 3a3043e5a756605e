"""The dropout's mask and its sums in float64 on the CPU (numpy), from the definition of the generator (J. Salmon et al.,
Parallel random numbers: as easy as 1, 2, 3, 2011)."""
from __future__ import annotations

import numpy as np

__all__ = ["philox", "keep_ref", "dropout_ref", "dropout_grad_ref"]


def philox(counter, key, rounds=7):
    """Philox4x32: four words of arrays ``counter`` (4) and two of ``key``, uint32 values in uint64."""
    c = [np.asarray(x, dtype=np.uint64) for x in counter]
    k = [int(x) for x in key]
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    for _ in range(rounds):
        p0, p1 = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(p1 >> half) ^ c[1] ^ np.uint64(k[0]), p1 & low, (p0 >> half) ^ c[3] ^ np.uint64(k[1]), p0 & low]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    return c


def keep_ref(n, c, p, seed, offset, row0=0):
    """(which values of rows row0 .. row0 + n - 1 stay, their scale)."""
    seed, offset = seed % 2 ** 64, offset % 2 ** 64
    group, row = np.arange(-(-c // 8), dtype=np.uint64)[None, :], np.arange(row0, row0 + n, dtype=np.uint64)[:, None]
    zero = np.zeros_like(group + row)
    w = philox((group + zero, row + zero, zero + np.uint64(offset % 2 ** 32), zero + np.uint64(offset >> 32)),
               (seed % 2 ** 32, seed >> 32))
    u = np.stack([h for x in w for h in (x % np.uint64(65536), x >> np.uint64(16))], axis=-1).reshape(n, -1)[:, :c]
    cut = int(round(65536 * p))
    return u >= cut, 65536 / (65536 - cut) if cut < 65536 else 0.0


def dropout_ref(x, p, seed, offset, residual=None, row0=0):
    """(rows, C) float64."""
    keep, up = keep_ref(*x.shape, p, seed, offset, row0)
    y = np.where(keep, x * up, 0.0)
    return y if residual is None else y + residual


def dropout_grad_ref(gy, p, seed, offset):
    return dropout_ref(gy, p, seed, offset)
