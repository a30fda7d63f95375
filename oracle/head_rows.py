"""Plain 64-bit forms of the norms with the position rotation, forward and backward, and of
rows in 8 bits (numpy).

Beside its results each gives the magnitudes that enter the sums, against which an output's
error is measured.
"""
from __future__ import annotations

import numpy as np

from .paged import place, rotate

TOP = {"bf16": 120, "fp16": 8}  # a row's largest exponent


def normed(x, weight, eps):
    """x [T, h, D] -> (x r w, x r, r); weight None: x itself."""
    if weight is None:
        return x.copy(), x, np.ones(x.shape[:-1] + (1,))
    r = 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    return x * r * weight, x * r, r


def scaled_turn(y, pos, inv_freq, interleaved, rot_scale):
    """y turned and its turned features scaled -> (result, |y1| + |y2| times the scale)."""
    if inv_freq is None or not len(inv_freq):
        return y.copy(), np.abs(y)
    z, mag = rotate(y, pos, inv_freq, interleaved)
    n = 2 * len(inv_freq)
    z[..., :n] *= rot_scale
    mag[..., :n] *= abs(rot_scale)
    return z, mag


def forward(x, pos, inv_freq, interleaved, weight, eps, rot_scale=1.0):
    """-> (y, magnitudes)."""
    return scaled_turn(normed(x, weight, eps)[0], pos, inv_freq, interleaved, rot_scale)


def backward(x, dy, pos, inv_freq, interleaved, weight, eps, rot_scale=1.0):
    """-> (dx, magnitudes of dx, dweight or None, magnitudes of dweight)."""
    back = None if inv_freq is None else -np.asarray(inv_freq, dtype=np.float64)
    g, mag = scaled_turn(dy, pos, back, interleaved, rot_scale)
    if weight is None:
        return g, mag, None, None
    _, u, r = normed(x, weight, eps)
    dx = r * (g * weight - u * (g * weight * u).mean(-1, keepdims=True))
    dx_mag = r * (mag * np.abs(weight)
                  + np.abs(u) * (mag * np.abs(weight * u)).mean(-1, keepdims=True))
    return dx, dx_mag, (g * u).sum((0, 1)), (mag * np.abs(u)).sum((0, 1))


def exponent(amax, kind):
    """The least e with amax <= 448 * 2^e (-126 to the type's largest), 0 for amax = 0."""
    m, e = np.frexp(amax)  # amax = m 2^e, 0.5 <= m < 1; 448 = 0.875 * 2^9
    e = np.where(m > 0.875, e - 8, e - 9)
    return np.where(amax == 0, 0, np.clip(e, -126, TOP[kind]))


def to_code(x, e, kind):
    """x under 2^e as the value that its code stands for; infinities and NaN give NaN."""
    limit = np.where(e == TOP[kind], 240.0, 448.0)
    with np.errstate(invalid="ignore"):
        y = np.clip(np.ldexp(x, -e), -limit, limit)
        step = np.ldexp(1.0, np.frexp(np.maximum(np.abs(y), 2.0 ** -6))[1] - 4)
        out = np.ldexp(np.round(y / step) * step, e)  # (halves go to even)
    return np.where(np.isfinite(x), out, np.nan)


def row_exponents(x, kind):
    """[..., D] -> the rows' exponents, by their finite values."""
    return exponent(np.where(np.isfinite(x), np.abs(x), 0.0).max(-1), kind)


def gather(k, v, table, cu, starts, total):
    """Rows of k, v [n_pages, page, Hk, D] (as values) -> packed k and v, zeros where there is
    no token."""
    n_pages, page = k.shape[:2]
    out = np.zeros((2, total) + k.shape[2:])
    for b in range(len(table)):
        for t in range(max(int(cu[b]), 0), min(int(cu[b + 1]), total)):
            at = place(table, n_pages, page, b, int(starts[b]) + t - int(cu[b]))
            if at is not None:
                out[0, t], out[1, t] = k[at], v[at]
    return out[0], out[1]
