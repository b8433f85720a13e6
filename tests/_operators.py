"""Float64 references of the operators around attention and the error bounds that
their arithmetic gives, shared by the tests.

u = finfo.eps / 2 is one rounding to the type, relative to the value.
"""

import torch

U32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def seen(Tq, Tk, q_start, window, sinks, causal, lengths, B, dev):
    """[B, Tq, Tk] which keys each row sees."""
    p = q_start + torch.arange(Tq, device=dev)[None, :, None]
    j = torch.arange(Tk, device=dev)[None, None, :]
    w = Tk + 1 if window is None else window
    on = ((p - j < w) if causal else ((p - j).abs() < w)) | (j < sinks)
    if causal:
        on = on & (j <= p)
    n = torch.full((B,), Tk, device=dev) if lengths is None else lengths.clamp(0, Tk)
    n = n[:, None, None]
    return on & (j < n) & (p < n)


def attention(q, k, v, on, scale):
    """(o, P) in float64 from BTHD tensors; masked values of k and v do not count,
    whatever they are. on: [B, Tq, Tk]."""
    group = q.shape[2] // k.shape[2]
    used = on.any(1)[:, :, None, None]  # keys that some row sees
    q, k, v = q.double(), k.double().masked_fill(~used, 0), v.double().masked_fill(~used, 0)
    q = q.masked_fill(~on.any(2)[:, :, None, None], 0)
    q, k, v = (t.transpose(1, 2) for t in (q, k, v))
    k, v = (t.repeat_interleave(group, 1) for t in (k, v))
    s = (q @ k.transpose(-1, -2) * scale).masked_fill(~on[:, None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = (s - top.masked_fill(top == float("-inf"), 0)).exp()
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
    return (p @ v).transpose(1, 2), p, (q, k, v)


def forward_bound(o, p, v, dtype):
    """Per element: P and the row sum are rounded or summed with rounded P
    (u each, on sum P|v| and on o), o is rounded once (u |o|); scores carry fp32
    errors: D products and the factor, at most 2^-13 of P here (D 2^-24 sum |q k|
    scale, with |q| |k| scale below 30), twice (numerator and sum). fp16: P below
    2^-14 is off by up to 2^-25, against a sum of at least 1."""
    u = half_step(dtype)
    pv = (p @ v.abs()).transpose(1, 2)
    tol = u * (2 * o.abs() + pv) + 2 * 2.0 ** -13 * pv
    if dtype == torch.float16:
        keys = (p > 0).sum(-1).amax().item()
        tol = tol + keys * 2.0 ** -25 * (v.abs().amax() + o.abs())
    return tol * 1.01 + 1e-30


def gradients(q, k, v, on, scale, do, dtype):
    """Float64 gradients (dq, dk, dv) in BTHD and their bounds, kv heads summed over
    their group. do: rows that see nothing do not count."""
    B, Tq, H, D = q.shape
    Hkv = k.shape[2]
    o, p, (qh, kh, vh) = attention(q, k, v, on, scale)
    do = do.double().masked_fill(~on.any(2)[:, :, None, None], 0).transpose(1, 2)
    oh = o.transpose(1, 2)
    dp = do @ vh.transpose(-1, -2)
    delta = (do * oh).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    dq, dk, dv = scale * ds @ kh, scale * ds.transpose(-1, -2) @ qh, p.transpose(-1, -2) @ do
    u, f = half_step(dtype), 2.0 ** -13
    # dS: one rounding; D_i from o as the forward rounded it (its own bound, times |do|);
    # P and dP carry fp32 errors of at most f
    ob = forward_bound(o, p, vh, dtype).transpose(1, 2)
    e_delta = (do.abs() * (ob + f * oh.abs())).sum(-1, keepdim=True)
    e_ds = (u + 2 * f) * ds.abs() + p * (e_delta + 2 * f * (do.abs() @ vh.abs().transpose(-1, -2) + delta.abs()))
    e_p = (u + 2 * f) * p
    if dtype == torch.float16:
        e_ds = e_ds + 2.0 ** -25 * (p > 0)
        e_p = e_p + 2.0 ** -25 * (p > 0)
    bounds = (u * dq.abs() + scale * e_ds @ kh.abs(), scale * e_ds.transpose(-1, -2) @ qh.abs(),
              e_p.transpose(-1, -2) @ do.abs())
    fold = lambda t: t.unflatten(1, (Hkv, -1)).sum(2)  # noqa: E731
    dk, dv = fold(dk), fold(dv)
    bounds = (bounds[0], fold(bounds[1]) + u * dk.abs(), fold(bounds[2]) + u * dv.abs())
    out = [t.transpose(1, 2) for t in (dq, dk, dv)]
    return out, [t.transpose(1, 2) * 1.01 + (2.0 ** -25 if dtype == torch.float16 else 1e-30) for t in bounds]


def close(got, want, bound, what):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = (got.double() - want).abs() - bound
    worst = over.max().item() if over.numel() else 0.0
    assert worst <= 0, f"{what}: {worst:.3e} over the bound (bound there {bound.flatten()[over.argmax()].item():.3e})"


def norm_rope(x, w, cos, sin, at, interleaved, eps):
    """Float64 norm and rotation of x [B, T, H, D]; at: positions [B, T]."""
    x = x.double()
    n = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    if w is not None:
        n = n * w.double()
    if cos is None:
        return n
    c, s = cos.double()[at][:, :, None], sin.double()[at][:, :, None]
    R = 2 * c.shape[-1]
    if interleaved:
        a, b = n[..., 0:R:2], n[..., 1:R:2]
        y = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = n[..., :R // 2], n[..., R // 2:R]
        y = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([y, n[..., R:]], -1)
