"""Attention of one new token of each sequence over a paged key-value cache
(``solattn_paged_attn``), the single-token form of ``_window.window_attn``. The pages
are written by ``_qk_rope.qk_norm_rope_append``. No counterpart in the reference.
"""

from __future__ import annotations

import torch

from ._ops import native

__all__ = ["paged_attn"]


def paged_attn(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
               page_table: torch.Tensor, lengths: torch.Tensor, *, window: int | None = None,
               sinks: int = 0, scale: float | None = None) -> torch.Tensor:
    """Attention of q [B, 1, H, D] (bf16 or fp16), the last token of sequences of
    ``lengths`` (int32 [B]) tokens, over their keys in k_cache, v_cache [pages,
    page_size, Hkv, D] (H a multiple of Hkv, page_size of 8); returns [B, 1, H, D].

    Key j of sequence b is slot j % page_size of page ``page_table[b, j //
    page_size]`` (int32 [B, pages of a sequence]). With ``window`` the token sees its
    last ``window`` keys and the first ``sinks``. A sequence of length 0 gives zeros;
    lengths are clamped to what the table holds, and keys on page ids that the cache
    does not have are not visible. Has no gradient.
    """
    return native.paged_attn(q, k_cache, v_cache, page_table, lengths, window, sinks, scale)
