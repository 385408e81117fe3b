"""Counter-based dropout and the LoRA down projections under it, in 64 bits on the host.

The generator is Philox4x32 with 7 rounds (Salmon et al., SC 2011); the mask of (seed, offset + stream)
at index i of a row-major tensor is lane i % 8 (16 bits, low half of a word first) of the words of
counter (i // 8, offset + stream) under the key seed, kept iff >= floor(p * 65536 + 1/2)."""

import math

import numpy as np

_M32 = np.uint64(0xFFFFFFFF)


def philox(counter, key, rounds=7):
    """Words uint64 [n, 4] (32-bit values) of counters [n, 4] under key (k0, k1)."""
    c = [np.asarray(counter[:, j], dtype=np.uint64) for j in range(4)]
    k0, k1 = int(key[0]), int(key[1])
    for _ in range(rounds):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), p1 & _M32,
             (p0 >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), p0 & _M32]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack(c, 1)


def cut_scale(p):
    cut = math.floor(p * 65536 + 0.5)
    return cut, (65536.0 / (65536 - cut) if cut < 65536 else 0.0)


def keep(n, p, seed, offset, stream=0, start=0):
    """bool [n]: the mask of the values start .. start + n - 1 (start a multiple of 8)."""
    group = np.arange(start // 8, (start + n + 7) // 8, dtype=np.uint64)
    seed, off = int(seed) % 2 ** 64, (int(offset) + int(stream)) % 2 ** 64
    counter = np.stack([group & _M32, group >> np.uint64(32), np.full_like(group, off & 0xFFFFFFFF),
                        np.full_like(group, off >> 32)], 1)
    lanes = philox(counter, (seed & 0xFFFFFFFF, seed >> 32)).astype("<u4").view("<u2").reshape(-1)
    return lanes[:n] >= cut_scale(p)[0]


def dropout(x, p, seed, offset, stream=0, residual=None):
    k = keep(x.size, p, seed, offset, stream).reshape(x.shape)
    y = np.where(k, x.astype(np.float64) * cut_scale(p)[1], 0.0)
    return y if residual is None else residual.astype(np.float64) + y


def lora_down(x16, a, p, seed, offset, stream=0):
    """u [T, branches * rank] and the sum of its terms' magnitudes, from the 16-bit x and a's values."""
    x16, nb = x16.astype(np.float64), len(p)
    r = a.shape[0] // nb
    us, mags = [], []
    for b in range(nb):
        k = keep(x16.size, p[b], seed, offset, stream + b).reshape(x16.shape)
        s, ab = cut_scale(p[b])[1], a[b * r:(b + 1) * r].astype(np.float64)
        xm = np.where(k, x16, 0.0)
        us.append(s * (xm @ ab.T))
        mags.append(s * (np.abs(xm) @ np.abs(ab).T))
    return np.concatenate(us, 1), np.concatenate(mags, 1)


def lora_down_bwd(du, x16, a, p, seed, offset, stream=0, addend=None):
    """(dx, da) and the sums of their terms' magnitudes."""
    du, x16, nb = du.astype(np.float64), x16.astype(np.float64), len(p)
    r = a.shape[0] // nb
    dx = np.zeros_like(x16) if addend is None else addend.astype(np.float64)
    mdx, das, mdas = np.abs(dx), [], []
    for b in range(nb):
        k = keep(x16.size, p[b], seed, offset, stream + b).reshape(x16.shape)
        s, ab, g = cut_scale(p[b])[1], a[b * r:(b + 1) * r].astype(np.float64), du[:, b * r:(b + 1) * r]
        dx = dx + np.where(k, s * (g @ ab), 0.0)
        mdx = mdx + np.where(k, s * (np.abs(g) @ np.abs(ab)), 0.0)
        xm = np.where(k, x16, 0.0)
        das.append(s * (g.T @ xm))
        mdas.append(s * (np.abs(g).T @ np.abs(xm)))
    return dx, np.concatenate(das), mdx, np.concatenate(mdas)
