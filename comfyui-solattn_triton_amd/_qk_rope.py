"""Norms of queries and keys per head with the position rotation, in one pass
(``solattn_qk_norm_rope``): what runs in front of every attention call.

``qk_norm_rope`` is differentiable in q, k and the weights;
``qk_norm_rope_append`` is its form for new tokens, writing k and v into the pages
that ``_paged.paged_attn`` reads. No counterpart in the reference.
"""

from __future__ import annotations

import torch

from ._capi import LIB, call, ptr, stream
from ._operands import (DTYPES, as_rows, check_cache, check_kv_heads, check_rows, refuse_grad,
                        strides, workspace)

__all__ = ["qk_norm_rope", "qk_norm_rope_append"]


def _weight(w, name, q):
    if w is None:
        return None
    if tuple(w.shape) != (q.shape[-1],) or w.device != q.device or not w.is_floating_point():
        raise ValueError(f"{name} must be a float tensor of shape ({q.shape[-1]},) on {q.device}, "
                         f"got {w.dtype} {tuple(w.shape)} on {w.device}")
    w = w.float().contiguous()
    return w if w.data_ptr() % 16 == 0 else w.clone()


def _table(cos, sin, q, interleaved):
    """(cos, sin, positions, rotated channels)"""
    if cos is None and sin is None:
        return None, None, 0, 0
    if cos is None or sin is None:
        raise ValueError("cos and sin go together")
    if cos.dim() != 2 or cos.shape != sin.shape or cos.shape[0] == 0:
        raise ValueError(f"cos and sin must be [positions, pairs], got {tuple(cos.shape)} {tuple(sin.shape)}")
    for name, t in (("cos", cos), ("sin", sin)):
        if t.dtype != torch.float32 or t.device != q.device:
            raise ValueError(f"{name} must be float32 on {q.device}, got {t.dtype} on {t.device}")
    rotated, whole = 2 * cos.shape[1], 8 if interleaved else 16
    if rotated > q.shape[-1] or rotated % whole:
        raise ValueError(f"{rotated} rotated channels of {q.shape[-1]}; a multiple of {whole}")
    ready = [t if t.is_contiguous() and t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)
             for t in (cos, sin)]
    return ready[0], ready[1], cos.shape[0], rotated


def _positions(positions, q, table_rows, rotated):
    """(int32 positions or None, batch stride)"""
    B, T = q.shape[:2]
    if positions is None:
        if rotated and T > table_rows:
            raise ValueError(f"{T} tokens, a table of {table_rows} positions")
        return None, 0
    if positions.dtype not in (torch.int32, torch.int64) or positions.device != q.device:
        raise ValueError(f"positions must be int32 or int64 on {q.device}, got {positions.dtype} on {positions.device}")
    if tuple(positions.shape) not in ((T,), (B, T)):
        raise ValueError(f"positions must be [{T}] or [{B}, {T}], got {tuple(positions.shape)}")
    positions = positions.to(torch.int32).contiguous()
    return positions, T if positions.dim() == 2 else 0


def _forward(q, k, qw, kw, cos, sin, positions, plan):
    B, T, H, D = q.shape
    P, R, interleaved, pos_b, eps = plan
    qo = torch.empty((B, T, H, D), device=q.device, dtype=q.dtype)
    ko = torch.empty(k.shape, device=q.device, dtype=q.dtype)
    if q.numel():
        with torch.cuda.device(q.device):
            call("solattn_qk_norm_rope", ptr(q), *strides(q), ptr(k), *strides(k), B, T, H, k.shape[2], D,
                 DTYPES[q.dtype], ptr(qw), ptr(kw), ptr(cos), ptr(sin), P, R, interleaved, ptr(positions), pos_b, eps,
                 ptr(qo), *strides(qo), ptr(ko), *strides(ko), stream(q.device))
    return qo, ko


class _NormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, qw, kw, cos, sin, positions, plan):
        ctx.save_for_backward(q, k, qw, kw, cos, sin, positions)
        ctx.plan = plan
        return _forward(q, k, qw, kw, cos, sin, positions, plan)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dqo, dko):
        q, k, qw, kw, cos, sin, positions = ctx.saved_tensors
        P, R, interleaved, pos_b, eps = ctx.plan
        B, T, H, D = q.shape
        dq = torch.empty(q.shape, device=q.device, dtype=q.dtype)
        dk = torch.empty(k.shape, device=q.device, dtype=q.dtype)
        dqw = torch.empty(D, device=q.device, dtype=torch.float32) if ctx.needs_input_grad[2] else None
        dkw = torch.empty(D, device=q.device, dtype=torch.float32) if ctx.needs_input_grad[3] else None
        if q.numel():
            dqo, dko = as_rows(dqo), as_rows(dko)
            with torch.cuda.device(q.device):
                weights = dqw is not None or dkw is not None
                ws = workspace(LIB.solattn_qk_norm_rope_bwd_workspace_bytes(D) if weights else 0, q.device)
                call("solattn_qk_norm_rope_bwd", ptr(q), *strides(q), ptr(k), *strides(k), ptr(dqo), *strides(dqo),
                     ptr(dko), *strides(dko), B, T, H, k.shape[2], D, DTYPES[q.dtype], ptr(qw), ptr(kw), ptr(cos),
                     ptr(sin), P, R, interleaved, ptr(positions), pos_b, eps, ptr(dq), *strides(dq), ptr(dk),
                     *strides(dk), ptr(dqw), ptr(dkw), ptr(ws), ws.numel() if weights else 0, stream(q.device))
        else:
            for g in (dqw, dkw):
                if g is not None:
                    g.zero_()
        return dq, dk, dqw, dkw, None, None, None, None


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor | None = None,
                 k_weight: torch.Tensor | None = None, cos: torch.Tensor | None = None,
                 sin: torch.Tensor | None = None, *, eps: float = 1e-6,
                 positions: torch.Tensor | None = None, interleaved: bool = False):
    """(q', k'): every head's row of q [B, T, H, D] and k [B, T, Hkv, D] divided by
    its root mean square, times the weight [D] (None: 1), its first channels turned
    by the token's angles; fresh BTHD tensors of the inputs' type (bf16, fp16 or
    fp32).

    ``cos``, ``sin``: float32 [positions, pairs] (both None: no rotation); the pairs
    are channels (i, i + pairs), or (2i, 2i + 1) with ``interleaved``. Token t is at
    position t, or at ``positions`` ([T] or [B, T], clamped to the table).
    Differentiable in q, k and the weights.
    """
    check_rows(q, (("k", k),), types=tuple(DTYPES))
    if k.shape[:2] != q.shape[:2]:
        raise ValueError(f"q and k hold different tokens: {tuple(q.shape)} {tuple(k.shape)}")
    if k.shape[2] < 1 or q.shape[2] < 1:
        raise ValueError(f"no heads: {tuple(q.shape)} {tuple(k.shape)}")
    qw, kw = _weight(q_weight, "q_weight", q), _weight(k_weight, "k_weight", q)
    cos, sin, P, R = _table(cos, sin, q, interleaved)
    positions, pos_b = _positions(positions, q, P, R)
    q, k = as_rows(q), as_rows(k)
    plan = (P, R, int(interleaved), pos_b, float(eps))
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, qw, kw)):
        return _NormRope.apply(q, k, qw, kw, cos, sin, positions, plan)
    return _forward(q, k, qw, kw, cos, sin, positions, plan)


def qk_norm_rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor,
                        v_cache: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor,
                        q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None,
                        cos: torch.Tensor | None = None, sin: torch.Tensor | None = None, *,
                        eps: float = 1e-6, interleaved: bool = False) -> torch.Tensor:
    """``qk_norm_rope`` of the newest T tokens of B sequences: returns q', and writes
    k' and v to the tokens' places in the cache.

    ``lengths`` (int32 [B]) counts the new tokens too, as ``paged_attn`` then reads
    it: token t is at position lengths[b] - T + t, slot position % page_size of page
    ``page_table[b, position // page_size]``. k_cache, v_cache: [pages, page_size,
    Hkv, D]. A token before position 0 (an idle slot's length 0), past the table or
    on a page id that the cache does not have writes nothing, and its q' means
    nothing. Has no gradient.
    """
    refuse_grad("qk_norm_rope_append", q, k, v)
    check_rows(q, (("k", k), ("v", v), ("k_cache", k_cache), ("v_cache", v_cache)), types=tuple(DTYPES))
    if k.shape[:2] != q.shape[:2] or k.shape != v.shape or k.shape[2] != k_cache.shape[2]:
        raise ValueError(f"shapes do not match: q {tuple(q.shape)} k {tuple(k.shape)} v {tuple(v.shape)} "
                         f"cache {tuple(k_cache.shape)}")
    check_kv_heads(q.shape[2], k.shape[2])
    check_cache(k_cache, v_cache, page_table, lengths, q)
    qw, kw = _weight(q_weight, "q_weight", q), _weight(k_weight, "k_weight", q)
    cos, sin, P, R = _table(cos, sin, q, interleaved)
    q, k, v = as_rows(q), as_rows(k), as_rows(v)
    page_table, lengths = page_table.contiguous(), lengths.contiguous()
    B, T, H, D = q.shape
    qo = torch.empty((B, T, H, D), device=q.device, dtype=q.dtype)
    if k_cache.numel() == 0:  # a cache without pages holds nothing, but its address must not be null
        k_cache = v_cache = k
    if q.numel():
        with torch.cuda.device(q.device):
            call("solattn_qk_norm_rope_append", ptr(q), *strides(q), ptr(k), *strides(k), ptr(v), *strides(v), B, T, H,
                 k.shape[2], D, DTYPES[q.dtype], ptr(qw), ptr(kw), ptr(cos), ptr(sin), P, R, int(interleaved),
                 float(eps), ptr(qo), *strides(qo), ptr(k_cache), *strides(k_cache), ptr(v_cache), *strides(v_cache),
                 0 if k_cache is k else k_cache.shape[0], k_cache.shape[1], ptr(page_table), page_table.stride(0),
                 page_table.shape[1], ptr(lengths), stream(q.device))
    return qo
