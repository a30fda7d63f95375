"""A paged key-value cache: appending tokens with the position rotation, reading them
back, and the attention of one or several new tokens per sequence over the cache.

The caches are ``[n_pages, page_size, H_k, D]`` (bf16 or fp16), features contiguous and
other strides any multiple of 8 elements, so views of a joint or head-major allocation
serve too.  In 8 bits they are ``float8_e4m3fn`` (strides multiples of 16) beside
``k_scale`` and ``v_scale`` ``[n_pages, page_size, H_k]`` of ``float8_e8m0fnu``: a row (one
token and key head) is its codes times its power of two (page and token strides of the codes
below 2^36, strides of the powers below 2^32).  Token ``p`` of sequence ``b`` lies
in page ``page_table[b, p // page_size]`` at ``p % page_size``.  ``page_table`` and the
lengths are int32 tensors on the GPU and stay there: no call waits for the GPU, all of them
can be captured into a graph and replayed with other lengths and pages in the same tensors.
As the host never sees them, a position outside the table or a page outside the cache is no
error: such a token is neither stored nor read.  There is no counterpart in the reference,
which has no cache.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

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
    k_scale: Optional[torch.Tensor] = None,
    v_scale: Optional[torch.Tensor] = None,
    q_weight: Optional[torch.Tensor] = None,
    k_weight: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    rot_scale: float = 1.0,
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

    With ``k_scale`` and ``v_scale`` the rows are stored in 8 bits: a row's power of two is
    the least 2^e with max |x| <= 448 * 2^e (0 for a row of zeros), and x becomes the e4m3
    number nearest to x / 2^e, halves to even.  Keys are rounded once, from 32 bits.  In the
    last binade of the type of k and v, where a code would stand for more than the type
    holds, values end at 240 * 2^8 (fp16) or 240 * 2^120 (bf16); infinities and NaN become NaN.
    With ``q_weight`` and ``k_weight`` rows of q and k are normed before they turn, and with
    ``rot_scale`` turned features are scaled, as by :func:`packed_qk_norm_rope`.  These options
    take D 64, 128 or 256, a multiple of 16 rotated features, and rows with strides below 2^32
    elements.  Of two tokens that share a
    place in an 8-bit cache, codes and power of two may then not belong together.
    """
    return _lib.ops().paged_append(k, v, k_cache, v_cache, page_table, cache_lens, cu_seqlens, q,
                                   inv_freq, bool(interleaved), k_scale, v_scale, q_weight,
                                   k_weight, eps, rot_scale)


def paged_kv_gather(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    page_table: torch.Tensor,
    cu_seqlens: torch.Tensor,
    total: int,
    *,
    starts: Optional[torch.Tensor] = None,
    k_scale: Optional[torch.Tensor] = None,
    v_scale: Optional[torch.Tensor] = None,
    dtype: Optional[torch.dtype] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Keys and values of the caches as packed rows ``[total, H_k, D]``, for instance for
    :func:`packed_masked_attn`.

    Row ``t`` of sequence ``b`` (``cu_seqlens[b] <= t < cu_seqlens[b + 1]``, int32 on the GPU)
    is its token ``starts[b] + t - cu_seqlens[b]`` (``starts``: int32, default 0); rows of no
    sequence and tokens without a page are zeros.  An 8-bit cache takes its scales and the
    ``dtype`` of the result, bf16 or fp16 (fp16 where the rows came from fp16: it rounds
    values below its smallest step and overflows beyond its largest).  D: multiples of 16
    up to 1024.  Forward only.
    """
    return _lib.ops().paged_gather(k_cache, v_cache, page_table, cu_seqlens, int(total), starts,
                                   k_scale, v_scale, dtype)


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
    k_scale: Optional[torch.Tensor] = None,
    v_scale: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Attention of the last token of each sequence, ``q [n_seq, H, D]``, over the first
    ``cache_lens[b]`` tokens of its pages (its own among them).

    ``H / H_k`` query heads share a key head; D is 64, 128 or 256.  Scores are
    ``scale * q.k`` (default 1/sqrt(D)), then ``softcap * tanh(. / softcap)`` (1e-6 to 1e4), then
    minus ``alibi_slopes[h]`` (float32 ``[H]``) times the key's distance; ``window`` keeps
    the last that many keys.  :func:`packed_masked_attn` applies the same to whole sequences.
    A sequence without keys gets zeros.  ``k_scale`` and ``v_scale`` belong to an 8-bit cache,
    whose rows become ``q``'s type (bf16 or fp16).  Forward only.
    """
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1])
    return _lib.ops().paged_decode(q, k_cache, v_cache, page_table, cache_lens, scale, softcap,
                                   window, alibi_slopes, k_scale, v_scale)


def paged_chunk_attn(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    page_table: torch.Tensor,
    cache_lens: torch.Tensor,
    cu_seqlens: torch.Tensor,
    *,
    scale: Optional[float] = None,
    softcap: Optional[float] = None,
    window: Optional[int] = None,
    alibi_slopes: Optional[torch.Tensor] = None,
    k_scale: Optional[torch.Tensor] = None,
    v_scale: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Attention of several new tokens per sequence, packed ``q [T, H, D]``, over the caches:
    a chunk of a prompt, a turn behind a cached prefix, drafted tokens, or any mixture with
    sequences of one new token.

    Tokens ``cu_seqlens[b] .. cu_seqlens[b + 1] - 1`` (int32 on the GPU, not decreasing) are
    the last of the ``cache_lens[b]`` tokens of sequence ``b`` (their keys and values are in
    the cache), and each sees the keys up to its own, with ``window`` the last that many of
    them.  Scores, heads and 8-bit caches are those of :func:`paged_decode_attn`, the result
    is what :func:`packed_masked_attn` gives on the gathered keys.  Tokens in front of the
    first key (more new tokens than the cache holds) and rows of no sequence get zeros.  A key
    that some token of its sequence sees must be finite, also for the tokens that do not see
    it: they may weigh it with 0.  Query heads that share a key head read it together by the
    largest power of two in their number; other numbers read the cache several times.  At
    most 2^30 tokens and 4096 heads; strides of pages and tokens below 2^35 elements (2^36
    codes).  Forward only.
    """
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1])
    return _lib.ops().paged_chunk(q, k_cache, v_cache, page_table, cache_lens, cu_seqlens, scale,
                                  softcap, window, alibi_slopes, k_scale, v_scale)
