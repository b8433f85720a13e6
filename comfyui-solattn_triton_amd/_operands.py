"""Checks and strides shared by the operators around attention (norms with
rotation, windowed and paged attention)."""

from __future__ import annotations

import torch

from ._preprocess import HEAD_DIM, head_dim_ok

# dtype arguments of the C entries (SOLATTN_BF16, SOLATTN_FP16, SOLATTN_FP32)
DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
HALF_TYPES = (torch.bfloat16, torch.float16)


def strides(t: torch.Tensor):
    return t.stride(0), t.stride(1), t.stride(2)


def row_ready(t: torch.Tensor) -> bool:
    """Whether the kernels can read ``t`` in place: a contiguous last dim and every
    row 16-byte aligned."""
    whole = 16 // t.element_size()
    return (t.stride(-1) == 1 and t.data_ptr() % 16 == 0
            and t.stride(0) % whole == 0 and t.stride(1) % whole == 0 and t.stride(2) % whole == 0
            and t.stride(1) < 1 << 24)


def as_rows(t: torch.Tensor) -> torch.Tensor:
    # (a contiguous tensor may be misaligned, so .contiguous() alone is not enough)
    return t if row_ready(t) else t.clone(memory_format=torch.contiguous_format)


def check_rows(q: torch.Tensor, named, types=HALF_TYPES):
    """q and the ``named`` tensors: 4-dimensional, of q's dtype and device, a
    supported head dim."""
    if not q.is_cuda:
        raise ValueError("q is not a GPU tensor")
    if q.dtype not in types:
        raise ValueError(f"q dtype {q.dtype}; one of {[str(t) for t in types]}")
    for name, t in (("q", q), *named):
        if t.dim() != 4:
            raise ValueError(f"{name} must have 4 dimensions, got shape {tuple(t.shape)}")
        if t.dtype != q.dtype:
            raise ValueError(f"{name} dtype {t.dtype} differs from q's {q.dtype}")
        if t.device != q.device:
            raise ValueError(f"{name} is on {t.device}, q on {q.device}")
        if t.shape[-1] != q.shape[-1]:
            raise ValueError(f"{name} has head_dim {t.shape[-1]}, q {q.shape[-1]}")
    if not head_dim_ok(q.shape[-1]):
        raise ValueError(f"head_dim {q.shape[-1]} not supported (multiples of 8 up to {HEAD_DIM})")


def check_kv_heads(heads: int, kv_heads: int):
    if kv_heads < 1 or heads % kv_heads:
        raise ValueError(f"{heads} query heads cannot share {kv_heads} kv heads")


def check_int32(t, name: str, shape, device):
    if t.dtype != torch.int32 or tuple(t.shape) != tuple(shape) or t.device != device:
        raise ValueError(f"{name} must be an int32 tensor of shape {tuple(shape)} on {device}, "
                         f"got {t.dtype} {tuple(t.shape)} on {t.device}")


def check_window(window, sinks, scale):
    if window is not None and window < 1:
        raise ValueError(f"window {window}; at least 1, or None")
    if sinks < 0:
        raise ValueError(f"sinks {sinks}")
    if not scale > 0.0:
        raise ValueError(f"scale {scale} is not positive")


def check_cache(k_cache, v_cache, page_table, lengths, q):
    """A paged cache: k_cache and v_cache [pages, page_size, Hkv, D] of q's type,
    page_table int32 [B, max_pages], lengths int32 [B]."""
    B = q.shape[0]
    if k_cache.shape != v_cache.shape:
        raise ValueError(f"cache shapes differ: {tuple(k_cache.shape)} {tuple(v_cache.shape)}")
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        if not row_ready(t):  # written or read in place: a copy would not be the cache
            raise ValueError(f"{name} rows must be contiguous and 16-byte aligned, strides {t.stride()}")
    if k_cache.shape[1] % 8 or k_cache.shape[1] == 0:
        raise ValueError(f"page size {k_cache.shape[1]} is not a multiple of 8")
    if page_table.dim() != 2 or page_table.shape[0] != B:
        raise ValueError(f"page_table must be [{B}, pages of a sequence], got {tuple(page_table.shape)}")
    check_int32(page_table, "page_table", page_table.shape, q.device)
    check_int32(lengths, "lengths", (B,), q.device)


def workspace(nbytes: int, device) -> torch.Tensor | None:
    return torch.empty(nbytes, device=device, dtype=torch.uint8) if nbytes else None


def refuse_grad(what: str, *tensors):
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise ValueError(f"{what} has no gradient; call it under torch.no_grad()")
