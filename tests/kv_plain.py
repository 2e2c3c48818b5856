"""The token cache's operators from their definition, in 64 bits (numpy), for the tests."""
import numpy as np

CODES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantise(x):
    """float64 [..., D] -> (codes 0..15 [..., D], scale bytes [..., D / 32])."""
    g = x.reshape(x.shape[:-1] + (x.shape[-1] // 32, 32))
    amax = np.abs(g).max(-1)
    bad = ~np.isfinite(amax)
    a = np.where(bad, 1.0, amax)
    # the smallest e with amax < 7 * 2^e: amax / 7 = f * 2^e, f in [.5, 1)
    e = np.clip(np.frexp(a / 7.0)[1], -125, 125)
    y = np.abs(np.where(bad[..., None], 0.0, g)) / np.exp2(e.astype(np.float64))[..., None]
    mids = (CODES[1:] + CODES[:-1]) / 2
    code = np.searchsorted(mids, y, side="left")  # ties: the lower code
    tie = (code < 7) & (y == mids[np.minimum(code, 6)]) & (code % 2 == 1)
    code = code + tie
    code = np.where(np.signbit(g) & ~bad[..., None], code + 8, code)
    return code.reshape(x.shape).astype(np.uint8), np.where(bad, 255, e + 127).astype(np.uint8)


def values(codes, scales):
    v = np.where(codes >= 8, -1.0, 1.0) * CODES[codes % 8]
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return (v.reshape(v.shape[:-1] + (v.shape[-1] // 32, 32)) * s[..., None]).reshape(v.shape)


def stored(x):
    return values(*quantise(np.asarray(x, np.float64)))


def tile_values(tile, D):
    """One tile's bytes [34 D] -> (keys, values) [32, D], byte by byte as include/gvdb.h lays them out."""
    k = np.zeros((32, D // 2), np.uint8)
    v = np.zeros((32, D // 2), np.uint8)
    for t in range(32):
        for b in range(D // 2):
            u = (t % 2) * (D // 8) + b % (D // 8)
            k[t, b] = tile[((u // 16) * 64 + b // (D // 8) * 16 + t // 2) * 16 + u % 16]
            u = (t % 8) * (D // 32) + b % (D // 32)
            v[t, b] = tile[17 * D + ((u // 16) * 64 + t // 8 * 16 + b // (D // 32)) * 16 + u % 16]
    ks = tile[16 * D:17 * D].reshape(D // 32, 32).T
    vs = tile[33 * D:34 * D].reshape(D // 32, 32).T
    wide = lambda c: np.stack([c & 15, c >> 4], -1).reshape(32, D)  # noqa: E731
    return values(wide(k), ks), values(wide(v), vs)


def power(amax):
    """The smallest e with amax <= 127 * 2^e, at least 7 - 133."""
    f, e = np.frexp(amax / 127.0)
    return np.maximum(np.where(f == 0.5, e - 1, e), 7 - 133)


def bounds(k):
    """Stored keys [n, D] of a page -> (int8 [2, D], byte)."""
    if not np.isfinite(k).all():
        return np.zeros((2, k.shape[1]), np.int8), 255
    hi, lo = k.max(0), k.min(0)
    e = int(power(max(np.abs(hi).max(), np.abs(lo).max())))
    return np.stack([np.ceil(hi / 2.0 ** e), np.floor(lo / 2.0 ** e)]).astype(np.int8), e + 133


def attend(q, k, v, scale, sees):
    """q [D], k and v [n, D], sees [n] -> (o, lse, largest sum of |v| p / l, sum_d |q k| scale at most)."""
    k, v = k[sees], v[sees]
    if not len(k):
        z = np.zeros(q.shape)
        return z, -np.inf, z, 0.0
    s = (k @ q) * scale
    m = s.max()
    p = np.exp(s - m)
    return (p @ v) / p.sum(), m + np.log(p.sum()), (p @ np.abs(v)) / p.sum(), float((np.abs(k) @ np.abs(q)).max() * abs(scale))


def choose(q, page_bounds, seen, top, first, recent):
    """q [group, D], page_bounds: list of (int8 [2, D], byte) or None for a page that is not there -> positions, in order."""
    score = np.zeros(seen)
    for j in range(seen):
        b8, e = page_bounds[j] if page_bounds[j] is not None else (None, 255)
        if e == 255:
            score[j] = 3.402823466e38
            continue
        best = -np.inf
        for row in q:
            a = float(power(np.abs(row).max())) if np.isfinite(row).all() else 0.0
            q8 = np.rint(row / 2.0 ** a) if np.isfinite(row).all() else np.zeros(row.shape)
            best = max(best, float((np.maximum(q8, 0) @ b8[0] + np.minimum(q8, 0) @ b8[1]) * 2.0 ** a))
        score[j] = best * 2.0 ** (e - 133)
    score[:min(first, seen)] = np.inf
    if recent:
        score[max(0, seen - recent):] = np.inf
    return sorted(np.argsort(-score, kind="stable")[:top].tolist())
