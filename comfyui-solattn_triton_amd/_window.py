"""Sliding-window attention with sinks (``solattn_window_attn``): a fixed pattern
beside ``sol_attn``'s routed one, with gradients. No counterpart in the reference.
"""

from __future__ import annotations

import torch

from ._ops import native

__all__ = ["window_attn"]


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
    read and rows at later positions are zeros. Differentiable (once) in q, k and v.
    """
    return native.window_attn(q, k, v, window, sinks, causal, scale, lengths, q_start)
