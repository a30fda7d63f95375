"""A paged key-value cache: appending tokens with the position rotation, and the
attention of one new token per sequence over the cache.

The caches are ``[n_pages, page_size, H_k, D]`` (bf16 or fp16), features contiguous and
other strides any multiple of 8 elements, so views of a joint or head-major allocation
serve too.  Token ``p`` of sequence ``b`` lies in page ``page_table[b, p // page_size]``
at ``p % page_size``.  ``page_table`` and the lengths are int32 tensors on the GPU and
stay there: no call waits for the GPU, all of them can be captured into a graph and
replayed with other lengths and pages in the same tensors.  As the host never sees them,
a position outside the table or a page outside the cache is no error: such a token is
neither stored nor read.  There is no counterpart in the reference, which has no cache.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _lib


def paged_kv_append(
    k: torch.Tensor,
    v: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    page_table: torch.Tensor,
    cache_lens: torch.Tensor,
    *,
    cu_seqlens: Optional[torch.Tensor] = None,
    q: Optional[torch.Tensor] = None,
    inv_freq: Optional[torch.Tensor] = None,
    interleaved: bool = False,
) -> Optional[torch.Tensor]:
    """Appends packed keys and values ``[T, H_k, D]`` to the caches, in place.

    Token ``t`` of sequence ``b`` goes to position ``cache_lens[b] + t - cu_seqlens[b]``
    (``cache_lens``: the lengths before the call, which it does not change); without
    ``cu_seqlens`` there is one token per sequence.  With ``inv_freq`` (float32, half of
    the rotated features) the pairs ``(i, i + n)``, n = len(inv_freq), of the keys and of
    ``q`` ``[T, H, D]`` turn by position * inv_freq[i] on the way, or the pairs
    ``(2i, 2i + 1)`` if ``interleaved``; further features stay.  Returns ``q`` rotated, or
    None without it.  Tokens behind the last sequence are not stored and their rows of
    the result are zeros.  Of two tokens that share a place in the cache, each 16 bytes
    there are of either.  D: multiples of 8 up to 1024.
    Forward only.
    """
    return _lib.ops().paged_append(k, v, k_cache, v_cache, page_table, cache_lens, cu_seqlens, q,
                                   inv_freq, bool(interleaved))


def paged_decode_attn(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    page_table: torch.Tensor,
    cache_lens: torch.Tensor,
    *,
    scale: Optional[float] = None,
    softcap: Optional[float] = None,
    window: Optional[int] = None,
    alibi_slopes: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Attention of the last token of each sequence, ``q [n_seq, H, D]``, over the first
    ``cache_lens[b]`` tokens of its pages (its own among them).

    ``H / H_k`` query heads share a key head; D is 64, 128 or 256.  Scores are
    ``scale * q.k`` (default 1/sqrt(D)), then ``softcap * tanh(. / softcap)`` (1e-6 to 1e4), then
    minus ``alibi_slopes[h]`` (float32 ``[H]``) times the key's distance; ``window`` keeps
    the last that many keys.  :func:`packed_masked_attn` applies the same to whole sequences.
    A sequence without keys gets zeros.  Forward only.
    """
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1])
    return _lib.ops().paged_decode(q, k_cache, v_cache, page_table, cache_lens, scale, softcap,
                                   window, alibi_slopes)
