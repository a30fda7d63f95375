"""MI355X (gfx950) packed varlen FlashAttention and absorbed target attention.

Drop-in replacements for the reference packages' public APIs:

* ``triton_fa_varlen_v2``: :func:`packed_varlen_attn`, :func:`set_validate_cu_seqlens`
* ``triton_target_attn_absorb``: :func:`packed_target_attn`,
  :func:`target_attn_inner`, :func:`prepare_target_attn_indices`

Beside them, for language models: :func:`packed_masked_attn` (causal, windowed and prefix
masks, capped scores, distance biases, grouped key heads), :func:`packed_qk_norm_rope` (norms
of queries and keys with the position rotation), :func:`paged_kv_append`,
:func:`paged_kv_gather`, :func:`paged_decode_attn` and :func:`paged_chunk_attn` (a paged
key-value cache, in 16 or 8 bits, and the attention of one or several new tokens over it).

All compute runs in the in-tree HIP library ``libvafa.so`` (C ABI in
``include/vafa.h``); it is loaded on the first call.
"""
from .varlen import packed_varlen_attn, set_validate_cu_seqlens
from .absorb import packed_target_attn, prepare_target_attn_indices, target_attn_inner
from .masked import packed_masked_attn
from .norm_rope import packed_qk_norm_rope
from .paged import paged_chunk_attn, paged_decode_attn, paged_kv_append, paged_kv_gather

__all__ = [
    "packed_varlen_attn",
    "set_validate_cu_seqlens",
    "packed_target_attn",
    "prepare_target_attn_indices",
    "target_attn_inner",
    "packed_masked_attn",
    "packed_qk_norm_rope",
    "paged_kv_append",
    "paged_kv_gather",
    "paged_chunk_attn",
    "paged_decode_attn",
]
__version__ = "0.1.0"
