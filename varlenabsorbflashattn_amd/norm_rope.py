"""Norms of queries and keys with the position rotation, in one pass over the rows between a
projection and :func:`packed_masked_attn`; forward and backward.  :func:`paged_kv_append`
does the same on the way into a cache.  There is no counterpart in the reference.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib


def packed_qk_norm_rope(
    q: torch.Tensor,
    k: torch.Tensor,
    positions: Optional[torch.Tensor] = None,
    *,
    inv_freq: Optional[torch.Tensor] = None,
    interleaved: bool = False,
    q_weight: Optional[torch.Tensor] = None,
    k_weight: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    rot_scale: float = 1.0,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Each row (one token's head) of ``q [T, H, D]`` and ``k [T, H_k, D]`` (or ``[1, T, H, D]``)
    normed and rotated.

    With ``q_weight`` / ``k_weight`` (``[D]``, float32 or the rows' type, both alike) a row x
    becomes ``x * weight / sqrt(mean(x^2) + eps)``; without, it stays.  With ``inv_freq``
    (float32, half of the rotated features, a multiple of 8) the pairs ``(i, i + n)``, n =
    len(inv_freq), turn by ``positions[t] * inv_freq[i]`` (``positions`` int32 ``[T]``), or the
    pairs ``(2i, 2i + 1)`` if ``interleaved``, and are multiplied by ``rot_scale`` (which
    rotations scaled for long contexts carry beside their own frequencies); further features
    stay.  bf16 or fp16, D 64, 128 or 256; all in 32 bits, rounded once, whatever the size of a
    finite row (with ``eps`` 0 a row of zeros gives NaN).  ``q`` and ``k`` may be parts of one
    projection's output.

    Gradients for q, k and the weights; the backward is deterministic, a second derivative
    raises.  At most 2^30 tokens and 4096 heads, strides below 2^32 elements.  Forward and
    backward can be captured into a graph together; no eager graph of the same leaves may be
    alive then.  An infinity in a normed row gives NaN where it stands and at the other
    of its pair, and zeros else; a NaN gives NaN to the whole row.  Either gives NaN to the row's
    gradient and to the weights' gradients (an infinity at its feature alone), and neither
    touches another row.  Rows without a weight keep both where they stand.
    """
    yq, yk = _lib.ops().qk_norm_rope(q, k, positions, inv_freq, bool(interleaved), q_weight,
                                     k_weight, eps, rot_scale)
    return (yq.unsqueeze(0) if q.dim() == 4 else yq), (yk.unsqueeze(0) if k.dim() == 4 else yk)
