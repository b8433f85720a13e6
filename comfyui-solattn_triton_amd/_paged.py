"""Attention of one new token of each sequence over a paged key-value cache
(``solattn_paged_attn``), the single-token form of ``_window.window_attn``. The pages
are written by ``_qk_rope.qk_norm_rope_append``. No counterpart in the reference.
"""

from __future__ import annotations

import torch

from ._capi import LIB, call, ptr, stream
from ._operands import (DTYPES, as_rows, check_cache, check_kv_heads, check_rows, check_window,
                        refuse_grad, strides, workspace)

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
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    refuse_grad("paged_attn", q, k_cache, v_cache)
    check_rows(q, (("k_cache", k_cache), ("v_cache", v_cache)))
    check_window(window, sinks, scale)
    B, T, H, D = q.shape
    if T != 1:
        raise ValueError(f"q holds {T} tokens of a sequence; one")
    Hkv = k_cache.shape[2]
    check_kv_heads(H, Hkv)
    check_cache(k_cache, v_cache, page_table, lengths, q)
    out = torch.empty((B, 1, H, D), device=q.device, dtype=q.dtype)
    pages, page_size = k_cache.shape[:2]
    if B == 0:
        return out
    if pages == 0 or page_table.shape[1] == 0:
        return out.zero_()
    q = as_rows(q)
    if page_table.stride(1) != 1:
        page_table = page_table.contiguous()
    lengths = lengths.contiguous()
    window = 0 if window is None else min(int(window), (1 << 31) - 1)
    sinks = min(int(sinks), (1 << 31) - 1)
    max_pages = page_table.shape[1]
    with torch.cuda.device(q.device):
        need = LIB.solattn_paged_attn_workspace_bytes(B, H, Hkv, D, max_pages, page_size, window, sinks)
        ws = workspace(need, q.device)
        call("solattn_paged_attn", ptr(q), q.stride(0), q.stride(2), ptr(k_cache), *strides(k_cache), ptr(v_cache),
             *strides(v_cache), pages, page_size, ptr(page_table), page_table.stride(0), max_pages, ptr(lengths), B, H,
             Hkv, D, DTYPES[q.dtype], window, sinks, scale, ptr(ws), need, ptr(out), out.stride(0), out.stride(2),
             stream(q.device))
    return out
