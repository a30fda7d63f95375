"""Plain 64-bit form of packed attention under a mask, segment by segment and head by head
(numpy), with the magnitudes that the errors of a 16-bit kernel are measured against.
"""
from __future__ import annotations

import numpy as np


def visible(nq, nk, causal=True, window=None, prefix=0):
    """[nq, nk] truth values."""
    p = np.arange(nq)[:, None] + nk - nq
    j = np.arange(nk)[None, :]
    if not causal:
        return np.ones((nq, nk), bool)
    see = j <= p
    if window:
        see &= j > p - window
    return see | (j < prefix)


def _head(q, k, scale, causal, window, prefix, softcap, slope):
    """(P, derivative of a score by scale q.k, sum of exp(score - max)) of one head."""
    nq, nk = len(q), len(k)
    z = scale * (q @ k.T)
    grad = np.ones_like(z)
    if softcap:
        t = np.tanh(z / softcap)
        z, grad = softcap * t, 1.0 - t * t
    if slope is not None:
        z = z - slope * np.abs(np.arange(nq)[:, None] + nk - nq - np.arange(nk)[None, :])
    see = visible(nq, nk, causal, window, prefix)
    z = np.where(see, z, -np.inf)
    m = z.max(axis=1, initial=-np.inf, keepdims=True)
    e = np.where(see, np.exp(z - np.where(np.isfinite(m), m, 0.0)), 0.0)
    l = e.sum(1, keepdims=True)
    return np.divide(e, l, out=np.zeros_like(e), where=l > 0), grad, l


def attention(q, k, v, do, cu_q, cu_k, scale, causal=True, window=None, prefix=None, softcap=None,
              slopes=None, u=0.0, a=0.0):
    """-> {name: (value, bound)} of o and, with an upstream gradient, dq, dk and dv.

    ``u`` is half a step of the type relative to a value, ``a`` half its smallest step.
    The bounds count, element by element: the rounding of P and of dS for the products
    (u each, and a), the sum of the rounded P (u, in o and through the LSE in P), the fp32
    sums behind the scores (2^-12 of P and of P (|dP| + |delta|)), and the output's own
    rounding (u, a).  delta = o.dO meets the rounding of P in o, u sum P |dP - delta| (the
    denominator is the sum of the same rounded P, so v enters as v - o); o itself comes with
    eight more bits than the type holds, off by at most one of their steps, 2^-7 u |o|, or
    by a below fp16's smallest normal value; it and dP are fp32 sums of D products.

    P, dS and a bf16 output below 2^-126, fp32's smallest normal value, may come out as 0:
    each is then off by less than that, so P by f = 2^-126 in what it multiplies, |v|, |dO|
    and |dP - delta|, dS by f |scale| and the output by f.  (Keys whose distance bias is above
    87 hold nothing else.)
    """
    H, Hk, eps = q.shape[1], k.shape[1], 2.0 ** -12
    f = 2.0 ** -126 if u else 0.0
    G = H // Hk
    names = ["o"] if do is None else ["o", "dq", "dk", "dv"]
    shapes = [q.shape] if do is None else [q.shape, q.shape, k.shape, v.shape]
    val = {n: np.zeros(s) for n, s in zip(names, shapes)}
    err = {n: np.zeros(s) for n, s in zip(names, shapes)}
    for s in range(len(cu_q) - 1):
        sq, sk = slice(cu_q[s], cu_q[s + 1]), slice(cu_k[s], cu_k[s + 1])
        for h in range(H):
            g = h // G
            qh, kh, vh = q[sq, h], k[sk, g], v[sk, g]
            P, grad, l = _head(qh, kh, scale, causal, window, 0 if prefix is None else prefix[s],
                               softcap, None if slopes is None else float(slopes[h]))
            see = P > 0
            o = P @ vh
            val["o"][sq, h] = o
            flat = np.divide(2 * a, l, out=np.zeros_like(l), where=l > 0)
            err["o"][sq, h] = (2 * u + eps) * (P @ np.abs(vh)) + (flat + f) * (see @ np.abs(vh))
            if do is None:
                continue
            d = do[sq, h]
            dP, delta = d @ vh.T, (d * o).sum(1, keepdims=True)
            dS = P * (dP - delta) * grad * scale
            # error of dS: its factors', delta's, its own rounding
            c, sums = abs(scale), (q.shape[2] + 1) * 2.0 ** -24 if u else 0.0
            e_delta = u * (P * np.abs(dP - delta)).sum(1, keepdims=True) \
                + (2.0 ** -7 * u + sums) * (np.abs(o) * np.abs(d)).sum(1, keepdims=True) \
                + a * np.abs(d).sum(1, keepdims=True)
            E = (3 * u + eps) * np.abs(dS) \
                + c * P * grad * (e_delta + sums * (np.abs(d) @ np.abs(vh).T)) \
                + c * eps * P * (np.abs(dP) + np.abs(delta)) \
                + c * (a + f + f * np.abs(dP - delta) * grad) * see
            val["dq"][sq, h] = dS @ kh
            err["dq"][sq, h] = E @ np.abs(kh)
            val["dk"][sk, g] += dS.T @ qh
            err["dk"][sk, g] += E.T @ np.abs(qh)
            val["dv"][sk, g] += P.T @ d
            err["dv"][sk, g] += (2 * u + eps) * (P.T @ np.abs(d)) + (a + f) * (see.T @ np.abs(d))
    return {n: (val[n], err[n] + u * np.abs(val[n]) + a + f * (val[n] != 0)) for n in names}
