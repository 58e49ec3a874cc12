"""Plain NumPy statement (float64 and whole numbers) of the 4-bit dictionary and of the 8-bit columns: the formats
of include/onmf_hip.h entry by entry, and the products from the values they stand for."""
import math

import numpy as np

GROUP8 = 128


def bf16_up(v):
    """The smallest bfloat16 that is not below v >= 0, as a float."""
    if v == 0.0:
        return 0.0
    m, e = math.frexp(v)                       # v = m 2^e, 0.5 <= m < 1
    e = max(e, -125)                           # below 2^-126 the spacing stays that of the smallest normal number
    return math.ceil(math.ldexp(v, 8 - e)) * math.ldexp(1.0, e - 8)


def pack4_group(w):
    """One group -> (q, z, s); s is NaN for a group with a NaN or an infinity."""
    w = np.asarray(w, dtype=np.float64)
    if not np.isfinite(w).all():
        return np.zeros(len(w), dtype=int), 0, math.nan
    lo, hi = w.min(), w.max()
    floor = max(abs(lo), abs(hi)) / 255
    s = bf16_up(max((hi - lo) / 15, floor))
    if s > 0 and np.rint(hi / s) - np.rint(lo / s) > 15:
        s = bf16_up(max((hi - lo) / 14, floor))
    if s < 2.0 ** -126:
        return np.zeros(len(w), dtype=int), 0, 0.0
    z = int(np.rint(lo / s))
    return np.rint(w / s).astype(int) - z, z, s


def pack4(W, group):
    """W (d x r) -> q (r, padded d), z (r, groups), s (r, groups)."""
    W = np.asarray(W, dtype=np.float64)
    d, r = W.shape
    groups = -(-d // group)
    q = np.zeros((r, groups * group), dtype=int)
    z = np.zeros((r, groups), dtype=int)
    s = np.zeros((r, groups))
    for k in range(r):
        for g in range(groups):
            part = W[g * group:min(d, (g + 1) * group), k]
            qq, z[k, g], s[k, g] = pack4_group(part)
            q[k, g * group:g * group + len(part)] = qq
    return q, z, s


def to_codes4(q, z, s):
    """The bytes and words of the format."""
    r, n = q.shape
    words = np.zeros((r, n // 8), dtype=np.uint32)
    for j in range(8):
        words |= q[:, j::8].astype(np.uint32) << np.uint32(4 * ((j >> 1) + 4 * (j & 1)))
    with np.errstate(invalid="ignore"):
        bits = s.astype(np.float32).view(np.uint32)
    return words.view(np.uint8), (bits | (z.astype(np.int64) & 0xFFFF).astype(np.uint32)).view(np.int32)


def values4(q, z, s, d):
    """The d x r matrix that q, z, s stand for."""
    r, n = q.shape
    groups = z.shape[1]
    v = (q.reshape(r, groups, -1) + z[:, :, None]) * s[:, :, None]
    return v.reshape(r, n)[:, :d].T


def reach4(q, z, s, d):
    """s (q + |z|): what the terms that are added up can be as large as."""
    return values4(q, np.abs(z), np.abs(s), d)


def keep8(X):
    """X (d x n) -> q (d, padded n), s (d, groups)."""
    X = np.asarray(X, dtype=np.float64)
    d, n = X.shape
    groups = -(-n // GROUP8)
    q = np.zeros((d, groups * GROUP8), dtype=int)
    s = np.zeros((d, groups))
    for i in range(d):
        for g in range(groups):
            part = X[i, g * GROUP8:min(n, (g + 1) * GROUP8)]
            if not np.isfinite(part).all():
                s[i, g] = math.nan
                continue
            step = float(np.float32(np.abs(part).max()) * np.float32(1 / 127))
            if step < 2.0 ** -126:
                continue
            s[i, g] = step
            q[i, g * GROUP8:g * GROUP8 + len(part)] = np.rint(part / step).astype(int)
    return q, s


def values8(q, s, n):
    return (q * np.repeat(s, GROUP8, axis=1))[:, :n]


def aggregate(X, H, w, A, B):
    return (1 - w) * A + w * (H @ H.T), (1 - w) * B + w * (H @ X.T)


def gradient(W, X, H):
    """The gradient of 1/2 |X - W H|^2 to W."""
    return (W @ H - X) @ H.T


def loss(W, X, H):
    return 0.5 * float(((X - W @ H) ** 2).sum())
