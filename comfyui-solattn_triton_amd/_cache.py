"""A paged key-value cache of 8 bits (``solattn_cache_append``, ``solattn_cache_read``),
half the memory and half the reads of a 16-bit one. No counterpart in the reference.

k_cache, v_cache: codes [pages, page_size, Hkv, D] of ``torch.int8`` or
``torch.float8_e4m3fn``; k_scale, v_scale: ``torch.float8_e8m0fnu`` [pages, Hkv,
page_size], a power of two for each row. A cached value is ``code * scale``, which bf16
holds exactly, and fp16 within its range: a read in fp16, and a call with fp16 queries over
keys that sequences share, may round values below 2^-14; a read makes those from 65520 on
infinities, a call takes them as they are. Of a written row the scale is the smallest power
of two that keeps its largest magnitude within 127 (int8) or 448 (e4m3) codes, the codes are
the nearest (ties to even): int8 is off by at most 1/127 of the row's largest value, e4m3 by
1/16 of each value or 2^-17 of the row's largest. Rows below 2^-110 become zeros; a row with
a NaN or an infinity reads as NaN throughout.

Written here or, with norms and rotation in the same pass, by
``_qk_rope.qk_norm_rope_append``; attended by ``_paged.paged_attn``, or read back for
``_window.window_attn`` where a prompt comes in pieces.
"""

from __future__ import annotations

import torch

from ._ops import native

__all__ = ["cache_append", "cache_read"]


def cache_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                 page_table: torch.Tensor, lengths: torch.Tensor, k_scale: torch.Tensor,
                 v_scale: torch.Tensor) -> None:
    """Writes k and v [B, T, Hkv, D] (bf16, fp16 or fp32; D a multiple of 16 up to 128), the
    newest T tokens of B sequences, to their places in the cache.

    ``lengths`` (int32 [B]) counts them too: token t is at position lengths[b] - T + t, slot
    position % page_size of page ``page_table[b, position // page_size]``. A token before
    position 0, past the page table or on a page id that the cache does not have writes
    nothing. No two tokens of a call may have the same slot of the same page: what it holds
    then is a mixture of both. Has no gradient.
    """
    native.cache_append(k, v, k_cache, v_cache, page_table, lengths, k_scale, v_scale)


def cache_read(k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor,
               k_scale: torch.Tensor, v_scale: torch.Tensor, *, tokens: int, start: torch.Tensor | None = None,
               dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
    """(k, v) [B, tokens, Hkv, D] of ``dtype`` (bf16 or fp16): row t is key start[b] + t
    (int32 [B]; None: t) of sequence b, zeros where the sequence of ``lengths[b]`` tokens has
    no such key or its page is none of the cache's. Has no gradient.
    """
    return native.cache_read(k_cache, v_cache, page_table, lengths, k_scale, v_scale, tokens, start, dtype)
