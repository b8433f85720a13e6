"""Sliding-window attention with sinks (``solattn_window_attn``): a fixed pattern
beside ``sol_attn``'s routed one, with gradients. No counterpart in the reference.
"""

from __future__ import annotations

import torch

from ._capi import LIB, call, ptr, stream
from ._operands import (DTYPES, as_rows, check_int32, check_kv_heads, check_rows, check_window,
                        strides, workspace)

__all__ = ["window_attn"]


def _run(q, k, v, lengths, plan, lse):
    B, Tq, H, D = q.shape
    Tk, Hkv = k.shape[1:3]
    window, sinks, causal, scale, q_start = plan
    out = torch.empty((B, Tq, H, D), device=q.device, dtype=q.dtype)
    with torch.cuda.device(q.device):
        need = LIB.solattn_window_attn_workspace_bytes(B, Tq, Tk, H, Hkv, D, q_start, window, sinks, causal,
                                                       lse is not None)
        ws = workspace(need, q.device)
        call("solattn_window_attn", ptr(q), *strides(q), ptr(k), *strides(k), ptr(v), *strides(v), B, Tq, Tk, H, Hkv,
             D, DTYPES[q.dtype], q_start, ptr(lengths), window, sinks, causal, scale, ptr(out), *strides(out),
             ptr(lse), ptr(ws), need, stream(q.device))
    return out


class _WindowAttn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lengths, plan):
        B, Tq, H, _ = q.shape
        lse = torch.empty((B, H, Tq), device=q.device, dtype=torch.float32)
        out = _run(q, k, v, lengths, plan, lse)
        ctx.save_for_backward(q, k, v, out, lse, lengths)
        ctx.plan = plan
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        q, k, v, out, lse, lengths = ctx.saved_tensors
        window, sinks, causal, scale, q_start = ctx.plan
        B, Tq, H, D = q.shape
        Tk, Hkv = k.shape[1:3]
        grad = as_rows(grad)
        dq = torch.empty(q.shape, device=q.device, dtype=q.dtype)
        dk = torch.empty(k.shape, device=q.device, dtype=q.dtype)
        dv = torch.empty(k.shape, device=q.device, dtype=q.dtype)
        with torch.cuda.device(q.device):
            ws = workspace(LIB.solattn_window_attn_bwd_workspace_bytes(B, Tq, Tk, H, Hkv, D, window, sinks, causal), q.device)
            call("solattn_window_attn_bwd", ptr(q), *strides(q), ptr(k), *strides(k), ptr(v), *strides(v), ptr(out),
                 *strides(out), ptr(grad), *strides(grad), ptr(lse), B, Tq, Tk, H, Hkv, D, DTYPES[q.dtype], q_start,
                 ptr(lengths), window, sinks, causal, scale, ptr(dq), *strides(dq), ptr(dk), *strides(dk), ptr(dv),
                 *strides(dv), ptr(ws), ws.numel(), stream(q.device))
        return dq, dk, dv, None, None


def window_attn(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, window: int | None,
                sinks: int = 0, causal: bool = True, scale: float | None = None,
                lengths: torch.Tensor | None = None, q_start: int | None = None) -> torch.Tensor:
    """Attention of q [B, Tq, H, D] over k, v [B, Tk, Hkv, D] (bf16 or fp16, H a
    multiple of Hkv) within a window, the first ``sinks`` keys staying visible;
    returns a fresh [B, Tq, H, D] tensor.

    Row t sits at position p = q_start + t (default: the last Tq of the Tk) and sees
    the keys j with p - j < window or j < sinks, and j <= p; with ``causal=False``
    those with |p - j| < window or j < sinks. ``window=None``: no limit.
    ``lengths`` (int32 [B]): sequence b holds lengths[b] keys; later keys are not
    read and rows at later positions are zeros. Differentiable in q, k and v.
    """
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    check_rows(q, (("k", k), ("v", v)))
    check_window(window, sinks, scale)
    if k.shape != v.shape or k.shape[0] != q.shape[0]:
        raise ValueError(f"q/k/v shapes do not match: {tuple(q.shape)} {tuple(k.shape)} {tuple(v.shape)}")
    B, Tq, H, D = q.shape
    Tk = k.shape[1]
    check_kv_heads(H, k.shape[2])
    q_start = Tk - Tq if q_start is None else int(q_start)
    if q_start < 0 or q_start + Tq > Tk:
        raise ValueError(f"rows {q_start} to {q_start + Tq} of {Tk} keys")
    if lengths is not None:
        check_int32(lengths, "lengths", (B,), q.device)
        lengths = lengths.contiguous()
    plan = (Tk if window is None else min(int(window), Tk), min(int(sinks), Tk), int(causal), scale, q_start)
    grad = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
    if q.numel() == 0:  # no rows: nothing to run, gradients of zeros
        return q * 1 + 0 * (k[:0].sum() + v[:0].sum()) if grad else torch.empty_like(q)
    if D not in (64, 128) and (grad or Tq > 1 or not causal):
        # zero channels add exact zeros to every product; the pad's gradient is a slice
        wide = [torch.nn.functional.pad(t, (0, (64 if D < 64 else 128) - D)) for t in (q, k, v)]
        out = _WindowAttn.apply(*wide, lengths, plan) if grad else _run(*wide, lengths, plan, None)
        return out[..., :D].contiguous()
    q, k, v = as_rows(q), as_rows(k), as_rows(v)
    return _WindowAttn.apply(q, k, v, lengths, plan) if grad else _run(q, k, v, lengths, plan, None)
