"""Plain reference of the 8-bit cache: its codes and powers of two, and the bounds of
attention over them, in 64 bits."""

import torch

import _operators as ref

MOST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
KINDS = [torch.int8, torch.float8_e4m3fn]
E8 = torch.float8_e8m0fnu


def encode(x, kind):
    """(codes, exponent bytes uint8) of the rows of x (the last dim)."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    bad, none = ~torch.isfinite(x).all(-1, keepdim=True), top < 2.0 ** -110
    x, top = x.masked_fill(bad | none, 0.0), top.masked_fill(bad | none, 1.0)
    m, e = torch.frexp(top / MOST[kind])
    e = e - (m == 0.5).int()  # 2^(e - 1) <= top / most < 2^e before: the smallest power that is no less
    y = torch.ldexp(x, -e)
    codes = y.round().to(torch.int8) if kind == torch.int8 else y.float().to(kind)
    byte = (e + 127).masked_fill(none, 0).masked_fill(bad, 255).to(torch.uint8)
    if kind != torch.int8:
        codes = codes.view(torch.uint8).masked_fill(bad, 0x7F).view(kind)
    return codes, byte[..., 0]


def power(byte):
    return torch.where(byte == 0, 0.0, torch.exp2(byte.double() - 127)).masked_fill(byte == 255, float("nan"))


def values(codes, byte):
    """float64 [..., D] from codes [..., D] and bytes [...]."""
    return codes.float().double() * power(byte)[..., None]


def empty(pages, page, Hkv, D, kind, dev):
    """A cache whose slots read as NaN, and its scales."""
    codes = torch.full((pages, page, Hkv, D), 0x7F, dtype=torch.uint8, device=dev).view(kind)
    return codes, torch.full((pages, Hkv, page), 255, dtype=torch.uint8, device=dev).view(E8)


def tables(B, pages, dev, seed=0):
    """Scattered page ids [B, pages]."""
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(B * pages, generator=g).reshape(B, pages).to(torch.int32).to(dev)


def put(cache, scale, table, rows, kind, first=0):
    """Rows [B, T, Hkv, D] encoded into positions first .. first + T - 1."""
    page = cache.shape[1]
    codes, byte = encode(rows, kind)
    for b in range(rows.shape[0]):
        for t in range(rows.shape[1]):
            j = first + t
            p = int(table[b, j // page])
            cache.view(torch.uint8)[p, j % page] = codes[b, t].view(torch.uint8)
            scale.view(torch.uint8)[p, :, j % page] = byte[b, t]
    return values(codes, byte)


def forward_bound(o, p, v, dtype):
    """Attention over codes: P times V's power is kept in two bf16 parts (2^-16 of it
    left), scores carry fp32 errors of at most 2^-13 of P, twice (numerator and sum), o is
    rounded once."""
    pv = (p @ v.abs()).transpose(1, 2)
    return (ref.half_step(dtype) * o.abs() + (2.0 ** -16 + 2 * 2.0 ** -13) * pv) * 1.01 + \
        (2.0 ** -25 if dtype == torch.float16 else 1e-30)
