"""Plain 64-bit forms of the paged-cache operators, sequence by sequence (numpy).

Beside its result each gives what an output's error is measured against: the
magnitudes that enter the sums.
"""
from __future__ import annotations

import numpy as np


def rotate(x, pos, inv_freq, interleaved):
    """x [T, h, D] turned by pos [T] * inv_freq [n] -> (y, |x1| + |x2| of each pair)."""
    y, mag = x.copy(), np.abs(x)
    n = len(inv_freq)
    i0 = np.arange(n) * 2 if interleaved else np.arange(n)
    i1 = i0 + 1 if interleaved else i0 + n
    angle = pos.astype(np.float64)[:, None] * inv_freq.astype(np.float64)
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    y[..., i0] = x[..., i0] * c - x[..., i1] * s
    y[..., i1] = x[..., i1] * c + x[..., i0] * s
    mag[..., i0] = mag[..., i1] = np.abs(x[..., i0]) + np.abs(x[..., i1])
    return y, mag


def place(table, n_pages, page, b, pos):
    """(page, slot) of a sequence's token, or None where there is none."""
    if pos < 0 or pos // page >= table.shape[1]:
        return None
    p = int(table[b, pos // page])
    return (p, pos % page) if 0 <= p < n_pages else None


def append(k, v, k_cache, v_cache, table, lens, cu, q, inv_freq, interleaved):
    """-> (q rotated or None, k_cache, v_cache, magnitudes of q and of k_cache)."""
    T, (n_pages, page) = len(k), k_cache.shape[:2]
    cu = np.arange(len(lens) + 1) if cu is None else cu
    pos, seq = np.zeros(T, np.int64), np.full(T, -1)
    for b in range(len(lens)):
        t = np.arange(cu[b], cu[b + 1])
        pos[t], seq[t] = lens[b] + t - cu[b], b
    inv_freq = np.zeros(0) if inv_freq is None else inv_freq
    kr, kmag = rotate(k, pos, inv_freq, interleaved)
    kc, vc, kcm = k_cache.copy(), v_cache.copy(), np.abs(k_cache)
    for t in range(T):
        at = place(table, n_pages, page, seq[t], pos[t]) if seq[t] >= 0 else None
        if at is not None:
            kc[at], vc[at], kcm[at] = kr[t], v[t], kmag[t]
    if q is None:
        return None, kc, vc, None, kcm
    qr, qmag = rotate(q, pos, inv_freq, interleaved)
    gone = (seq < 0) | (pos < 0)
    qr[gone] = 0.0
    return qr, kc, vc, qmag, kcm


def decode(q, k_cache, v_cache, table, lens, scale, softcap=None, window=None, slopes=None):
    """-> (out [n, H, D], sum of P |v|, sum of |v| / sum of exp(score - max))."""
    n, H, D = q.shape
    n_pages, page, Hk = k_cache.shape[:3]
    out, mag, flat = np.zeros((3, n, H, D))
    for b in range(n):
        length = min(max(int(lens[b]), 0), table.shape[1] * page)
        first = max(0, length - window) if window else 0
        at = [(j, place(table, n_pages, page, b, j)) for j in range(first, length)]
        at = [(j, a) for j, a in at if a is not None]
        if not at:
            continue
        j = np.array([x[0] for x in at])
        pages, slots = np.array([x[1][0] for x in at]), np.array([x[1][1] for x in at])
        for h in range(H):
            hk = h // (H // Hk)
            k, v = k_cache[pages, slots, hk], v_cache[pages, slots, hk]
            z = scale * (k @ q[b, h])
            if softcap:
                z = softcap * np.tanh(z / softcap)
            if slopes is not None:
                z = z - float(slopes[h]) * (length - 1 - j)
            e = np.exp(z - z.max())
            P = e / e.sum()
            out[b, h], mag[b, h] = P @ v, P @ np.abs(v)
            flat[b, h] = np.abs(v).sum(0) / e.sum()
    return out, mag, flat
