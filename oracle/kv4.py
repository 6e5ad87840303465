"""CPU restatement of the paged 4-bit KV cache in 64 bits: the bytes of a
written token, the values that they stand for, attention over them, and the
error that an implementation in 32-bit sums and 16-bit weights may show."""

from __future__ import annotations

import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def encode(x):
    """x (..., D) -> (nibbles (..., D) uint8, codes (..., D // 32) uint8)."""
    x = np.asarray(x, np.float64)
    b = x.reshape(*x.shape[:-1], -1, 32)
    amax = np.abs(b).max(-1)
    bad = ~np.isfinite(amax)
    e = np.full(amax.shape, -99, np.int64)
    safe = np.where(bad, 0.0, amax)
    for step in (128, 64, 32, 16, 8, 4, 2, 1):  # smallest e >= -99 with 6 * 2^e >= amax
        e = np.where(np.ldexp(6.0, e + step - 1) < safe, e + step, e)
    with np.errstate(invalid="ignore"):
        y = np.where(bad[..., None], 0.0, np.ldexp(b, -e[..., None]))
    d = np.abs(np.abs(y)[..., None] - GRID)
    mag = 7 - np.argmin(d[..., ::-1], axis=-1)   # ties to the larger
    nib = (mag + 8 * (y < 0)).astype(np.uint8).reshape(x.shape)
    return nib, np.where(bad, 255, e + 127).astype(np.uint8)


def decode(nib, codes):
    """Inverse of ``encode``: float64 values."""
    codes = np.asarray(codes).astype(np.int64)
    s = np.where(codes == 255, np.nan, np.ldexp(1.0, codes - 127))
    v = GRID[nib & 7] * np.where(nib & 8, -1.0, 1.0)
    return (v.reshape(*v.shape[:-1], v.shape[-1] // 32, 32) * s[..., None]).reshape(v.shape)


def _at(D, piece):
    """Byte of each element of a row whose blocks are interleaved by pieces of
    ``piece`` elements."""
    el = np.arange(D)
    blk, i = el // 32, el % 32
    return ((i // piece) * (D // 32) + blk) * (piece // 2) + (i % piece) // 2


def write(pool, k, v, slots):
    """Write tokens into the pool (a numpy uint8 array, changed in place)."""
    D = pool.shape[3] // 17
    page, nb = pool.shape[2] * 16, D // 32
    el = np.arange(D)
    for t, s in enumerate(slots):
        if s < 0 or s >= pool.shape[0] * page:
            continue
        p, tile, r = s // page, s % page // 16, s % 16
        for h in range(pool.shape[1]):
            b = pool[p, h, tile]
            for x, row, code, piece in ((k, r * D // 2, 16 * D + r * nb, 8),
                                        (v, 8 * D + r * D // 2, 16 * D + D // 2 + r * nb, 4)):
                nib, c = encode(x[t, h])
                at = row + _at(D, piece)
                b[row:row + D // 2] = 0
                np.bitwise_or.at(b, at, (nib << (4 * (el % 2))).astype(np.uint8))
                b[code:code + nb] = c


def read(pool, slots):
    """Tokens of the pool as float64 (T, Hkv, D) keys and values; zeros for
    slots outside it."""
    D = pool.shape[3] // 17
    page, nb = pool.shape[2] * 16, D // 32
    slots = np.asarray(slots)
    live = (slots >= 0) & (slots < pool.shape[0] * page)
    s = np.where(live, slots, 0)
    tiles = pool[s // page, :, s % page // 16]            # (T, Hkv, 17 D)
    r = (s % 16)[:, None, None]
    el = np.arange(D)
    out = []
    for row, code, piece in ((0, 16 * D, 8), (8 * D, 16 * D + D // 2, 4)):
        byte = np.take_along_axis(tiles, row + r * (D // 2) + _at(D, piece) +
                                  np.zeros((1, tiles.shape[1], 1), np.int64), 2)
        nib = np.where(el % 2, byte >> 4, byte & 15).astype(np.uint8)
        c = np.take_along_axis(tiles, code + r * nb + np.arange(nb) +
                               np.zeros((1, tiles.shape[1], 1), np.int64), 2)
        out.append(np.where(live[:, None, None], decode(nib, c), 0.0))
    return out


def attention(q, pool, table, lens, rows, scale=None):
    """q (T, Hq, D) -> (out, bound): attention in 64 bits, and for every output
    the error that comes of 32-bit scores and 16-bit weights (not of the
    rounding of the output).

    A score is a sum of D products, each exact, in 32 bits: off by at most
    D 2^-24 sum|q k| scale, times two for the blocks' sums and the scale.  Off by ds,
    all weights are off by a factor within e^(2 ds).  A weight rounded to 11
    bits is off by 2^-12; an exp2 and a running rescale by some 2^-20 in all.
    So |error| <= (2^-12 + 2 ds + 2^-18) max|v|, the maximum over the tokens
    that the row sees."""
    q = np.asarray(q, np.float64)
    T, Hq, D = q.shape
    Hkv, page = pool.shape[1], pool.shape[2] * 16
    G = Hq // Hkv
    scale = D ** -0.5 if scale is None else scale
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    t = 0
    for i, (R, L) in enumerate(zip(rows, lens)):
        pos = np.arange(L)
        k, v = read(pool, np.asarray(table[i])[pos // page].astype(np.int64) * page + pos % page)
        for r in range(R):
            see = L - R + r + 1
            if see > 0:
                for h in range(Hq):
                    kk, vv = k[:see, h // G], v[:see, h // G]
                    s = kk @ q[t, h] * scale
                    p = np.exp(s - s.max())
                    out[t, h] = p @ vv / p.sum()
                    ds = 2 * D * 2.0 ** -24 * (np.abs(kk) @ np.abs(q[t, h])).max() * abs(scale)
                    bound[t, h] = (2.0 ** -12 + 2 * ds + 2.0 ** -18) * np.abs(vv).max()
            t += 1
    return out, bound
