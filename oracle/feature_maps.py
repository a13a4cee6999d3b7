"""64-bit CPU oracle of the feature-map operators (group norm with activation, dropout).

Written from the definitions with numpy and torch float64; shares no code with
the package. Philox4x32-10 is the generator of Salmon, Moraes, Dror and Shaw,
"Parallel random numbers: as easy as 1, 2, 3" (SC 2011).
"""

import numpy as np
import torch


def philox4x32_10(counter, key):
    """counter: four uint64 arrays below 2**32; key: two ints below 2**32. Four words."""
    mask = np.uint64(0xFFFFFFFF)
    c = [np.asarray(v, dtype=np.uint64) for v in counter]
    k = [int(key[0]), int(key[1])]
    for _ in range(10):
        p0 = c[0] * np.uint64(0xD2511F53)
        p1 = c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), p1 & mask,
             (p0 >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), p0 & mask]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    return c


def draws(seed, offset, start, count):
    """16-bit draws start .. start + count - 1 of the stream (seed, offset)."""
    e = np.arange(start, start + count, dtype=np.uint64)
    block = e >> np.uint64(3)
    low = np.uint64(0xFFFFFFFF)
    words = philox4x32_10(
        [block & low, block >> np.uint64(32), np.full_like(block, offset % 2 ** 32),
         np.full_like(block, offset >> 32)], (seed % 2 ** 32, seed >> 32))
    piece = (e & np.uint64(7)).astype(np.int64)
    word = np.choose(piece // 2, words)
    return ((word >> (np.uint64(16) * (piece % 2).astype(np.uint64)))
            & np.uint64(0xFFFF)).astype(np.int64)


def drop_factors(shape, p, seed, offset, channel=False):
    """Factor of every element of a channels-last map (float64, broadcastable to shape)."""
    t = int(p * 65536 + 0.5)
    if channel:
        shape = (shape[0],) + (1,) * (len(shape) - 2) + (shape[-1],)
    count = int(np.prod(shape))
    kept = torch.from_numpy(draws(seed, offset, 0, count) >= t).view(shape)
    return kept.double() * (65536 / (65536 - t) if t < 65536 else 0.0)


def normalised(x, groups, eps):
    """(x - mean) / sqrt(var + eps) of a channels-last float64 map, and 1 / sqrt(var + eps)
    per element."""
    b, c = x.shape[0], x.shape[-1]
    v = x.reshape(b, -1, groups, c // groups)
    mean = v.mean((1, 3), keepdim=True)
    var = ((v - mean) ** 2).mean((1, 3), keepdim=True)
    rstd = 1.0 / torch.sqrt(var + eps)
    return ((v - mean) * rstd).reshape(x.shape), rstd.expand(v.shape).reshape(x.shape)


def activated(z, activation, slope=0.01):
    if activation == "relu":
        return torch.relu(z)
    if activation == "silu":
        return z * torch.sigmoid(z)
    if activation == "leaky_relu":
        return torch.where(z > 0, z, slope * z)
    assert activation == "none"
    return z
