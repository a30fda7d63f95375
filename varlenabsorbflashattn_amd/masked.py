"""Packed attention of a language model: causal, windowed and prefix masks on packed
sequences, grouped key heads, scores capped by a tanh, distance biases; forward and
backward.  There is no counterpart in the reference, whose packed attention sees every
key of a segment (:func:`packed_varlen_attn`).

A host plan built from the lengths (cached by content, as for the other packed
operators) names for every tile of queries the keys that some of its rows see, and for
every tile of keys the queries that see it; tiles outside the mask are never read.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _lib, varlen
from .varlen import _check_tokens, _seqinfo_to_cu_seqlens


def _host(t, name):
    """An integer tensor (arrays and lists too) as a contiguous one on the host."""
    t = torch.as_tensor(t).detach()
    if t.is_floating_point() or t.is_complex() or t.dtype == torch.bool:
        raise AssertionError(f"{name} must be integers, got {t.dtype}")
    return (t if t.device.type == "cpu" else t.cpu()).contiguous()


def _host_pair(a, b):
    """Both cu_seqlens on the host, with one copy for two of one shape on the GPU."""
    if a is b:
        h = _host(a, "cu_seqlens_q")
        return h, h
    if a.is_cuda and b.is_cuda and a.device == b.device and a.dtype == b.dtype \
            and a.shape == b.shape and a.dim() == 1:
        h = _host(torch.stack((a.detach(), b.detach())), "cu_seqlens")
        return h[0], h[1]
    return _host(a, "cu_seqlens_q"), _host(b, "cu_seqlens_k")


def _plan_of(q, k, cu_seqlens_q, cu_seqlens_k, causal, window, prefix_lens):
    """Validation and the device plan.  As for packed_varlen_attn, a cached plan of the
    same content that covers exactly these tokens passed the checks when it was built."""
    T_q, H, D = q.shape
    T_k, H_k = k.shape[:2]
    cu_q, cu_k = _host_pair(cu_seqlens_q, cu_seqlens_k)
    content = _lib.ops().cu_key
    prefix = None if prefix_lens is None else _host(prefix_lens, "prefix_lens").to(torch.int64)
    if prefix is not None and prefix.shape != (cu_q.numel() - 1,):  # (the key holds content alone)
        raise AssertionError(f"prefix_lens must be [{cu_q.numel() - 1}], got {tuple(prefix.shape)}")
    key = ("masked", content(cu_q), content(cu_k), None if prefix is None else content(prefix),
           H, H_k, D, causal, window, q.device)
    plan = _lib.cached_plan(key) if cu_q.dim() == 1 and cu_k.dim() == 1 else None
    if plan is not None and plan.T_q == T_q and plan.T_k == T_k:
        return plan
    cu_q_h, cu_k_h = _lib.as_host_i64(cu_q), _lib.as_host_i64(cu_k)
    varlen._validate_cu_seqlens(cu_q_h, cu_q.shape, T_q, "cu_seqlens_q")
    varlen._validate_cu_seqlens(cu_k_h, cu_k.shape, T_k, "cu_seqlens_k")
    if cu_q_h.ndim != 1 or cu_q_h.size < 2:
        raise ValueError("cu_seqlens_q: must be 1-D with at least 2 elements")
    if plan is None:
        host = _lib.plan_masked(cu_q_h, cu_k_h, H, H_k, D, causal, window,
                                None if prefix is None else prefix.numpy())
        plan = _lib.cache_plan(key, host, q.device)
    _check_tokens(plan.info, T_q, T_k)
    return plan


def _check_options(D, cu_seqlens_q, cu_seqlens_k, q_seqinfo, k_seqinfo, causal, window,
                   prefix_lens, softcap, scale):
    """cu_seqlens and the options as the kernels take them (window and softcap 0: none)."""
    if cu_seqlens_q is None:
        if q_seqinfo is None:
            raise ValueError("must provide either cu_seqlens_q or q_seqinfo")
        cu_seqlens_q = _seqinfo_to_cu_seqlens(q_seqinfo)
    if cu_seqlens_k is None:
        if k_seqinfo is None:
            raise ValueError("must provide either cu_seqlens_k or k_seqinfo")
        cu_seqlens_k = _seqinfo_to_cu_seqlens(k_seqinfo)
    n_seg = cu_seqlens_q.numel() - 1
    assert cu_seqlens_k.numel() - 1 == n_seg, \
        f"segment count mismatch: q has {n_seg}, k has {cu_seqlens_k.numel() - 1}"

    if window is not None and (window < 1 or window != int(window)):
        raise ValueError(f"window must be positive and whole, got {window}")
    if softcap is not None and not 1e-6 <= softcap <= 1e4:
        raise ValueError(f"softcap must be positive, from 1e-6 to 1e4, got {softcap}")
    if not causal and (window is not None or prefix_lens is not None):
        raise ValueError("window and prefix_lens belong to the causal mask")
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite, got {scale}")
    return (cu_seqlens_q, cu_seqlens_k, bool(causal), min(int(window or 0), 1 << 31),
            float(softcap or 0.0),
            float(scale))


def packed_masked_attn(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    *,
    cu_seqlens_q: Optional[torch.Tensor] = None,
    cu_seqlens_k: Optional[torch.Tensor] = None,
    q_seqinfo: Optional[torch.Tensor] = None,
    k_seqinfo: Optional[torch.Tensor] = None,
    causal: bool = True,
    window: Optional[int] = None,
    prefix_lens: Optional[torch.Tensor] = None,
    softcap: Optional[float] = None,
    alibi_slopes: Optional[torch.Tensor] = None,
    scale: Optional[float] = None,
) -> torch.Tensor:
    """Packed attention under a mask, within each segment.

    ``q`` is ``[T_q, H, D]`` (or ``[1, T_q, H, D]``), ``k`` and ``v`` ``[T_k, H_k, D]``:
    ``H / H_k`` query heads share a key head; bf16 or fp16, D 64, 128 or 256.  Segments
    are given as for :func:`packed_varlen_attn`.  The queries of a segment are its last
    positions: query i of n_q against n_k keys has position ``p = i + n_k - n_q`` and sees
    key j where ``j <= p``, with ``window`` also ``j > p - window``, or where
    ``j < prefix_lens[segment]`` (``[n_seg]``); every key with ``causal=False``, which
    takes neither.  Scores are ``scale * q.k`` (default 1/sqrt(D)), then
    ``softcap * tanh(. / softcap)`` (1e-6 to 1e4), then minus ``alibi_slopes[h]`` (float32
    ``[H]``, no gradient) times ``|p - j|``.  A row that sees no key gets zeros and no
    gradient.  The backward is deterministic; a second derivative raises.  At most 2^30 tokens
    and 4096 heads.

    Keys that no query sees, and queries that see no key, may hold anything: zeros come
    out for them.  A key that some query sees must be finite in ``k`` and ``v``: rows that
    do not see it may weigh it with 0, and 0 times an infinity is NaN, as in
    ``softmax(.) @ v``; the same holds for rows of ``q`` and of the gradient in the
    backward.  Lengths on the GPU are read back, which waits for
    the GPU and which no graph capture allows: pass them on the host there.
    """
    ops = _lib.ops()
    q3, k3, v3 = ops.masked_operands(q, k, v, alibi_slopes)

    cu_seqlens_q, cu_seqlens_k, causal, window, softcap, scale = _check_options(
        q3.shape[2], cu_seqlens_q, cu_seqlens_k, q_seqinfo, k_seqinfo, causal, window, prefix_lens,
        softcap, scale)
    plan = _plan_of(q3, k3, cu_seqlens_q, cu_seqlens_k, causal, window, prefix_lens)
    o3 = ops.masked_attn(q3, k3, v3, plan.native, scale, softcap, window, alibi_slopes)
    return o3.unsqueeze(0) if q.dim() == 4 else o3
