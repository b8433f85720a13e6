"""Norms of queries and keys per head with the position rotation, in one pass
(``solattn_qk_norm_rope``): what runs in front of the attention of models that norm each
head's queries and keys.

``qk_norm_rope`` is differentiable in q, k and the weights;
``qk_norm_rope_append`` is its form for new tokens, writing k and v into the pages
that ``_paged.paged_attn`` reads. No counterpart in the reference.
"""

from __future__ import annotations

import torch

from ._ops import native

__all__ = ["qk_norm_rope", "qk_norm_rope_append"]


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor | None = None,
                 k_weight: torch.Tensor | None = None, cos: torch.Tensor | None = None,
                 sin: torch.Tensor | None = None, *, eps: float = 1e-6,
                 positions: torch.Tensor | None = None, interleaved: bool = False):
    """(q', k'): every head's row of q [B, T, H, D] and k [B, T, Hkv, D] divided by
    its root mean square, times the weight [D] (None: 1; the row is divided all the
    same), its first channels turned by the token's angles; fresh BTHD tensors of the
    inputs' type (bf16, fp16 or fp32).

    ``cos``, ``sin``: float32 [positions, pairs] (both None: no rotation); the pairs
    are channels (i, i + pairs), or (2i, 2i + 1) with ``interleaved``. Token t is at
    position t, or at ``positions`` ([T] or [B, T], clamped to the table).
    Differentiable (once) in q, k and the weights.
    """
    return native.qk_norm_rope(q, k, q_weight, k_weight, cos, sin, eps, positions, interleaved)


def qk_norm_rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor,
                        v_cache: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor,
                        q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None,
                        cos: torch.Tensor | None = None, sin: torch.Tensor | None = None, *,
                        eps: float = 1e-6, interleaved: bool = False, k_scale: torch.Tensor | None = None,
                        v_scale: torch.Tensor | None = None) -> torch.Tensor:
    """``qk_norm_rope`` of the newest T tokens of B sequences: returns q', and writes
    k' and v to the tokens' places in the cache.

    ``lengths`` (int32 [B]) counts the new tokens too, as ``paged_attn`` then reads
    it: token t is at position lengths[b] - T + t, slot position % page_size of page
    ``page_table[b, position // page_size]``. k_cache, v_cache: [pages, page_size,
    Hkv, D]. A token before position 0 (an idle slot's length 0), past the page table
    or on a page id that the cache does not have writes nothing, and its q' means
    nothing. No two tokens of a call may have the same slot of the same page: what it
    holds then is a mixture of both. Positions past the end of ``cos`` turn by its last
    row: it has to cover the sequences. Has no gradient.

    With ``k_scale`` and ``v_scale`` the caches are of 8 bits (``_cache``): k' and v are
    rounded to codes, k' once, from 32 bits.
    """
    return native.qk_norm_rope_append(q, k, v, k_cache, v_cache, page_table, lengths, q_weight, k_weight, cos, sin,
                                      eps, interleaved, k_scale, v_scale)
