"""The 8-bit cache (written, read back, attended) and attention over shared keys on the
GPU, against float64. Codes and powers are compared bit by bit, read values exactly,
attention by the bounds of tests/_operators.py and tests/_cache8.py."""

import importlib

import pytest
import torch

import _cache8 as c8
import _operators as ref

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32
I8, F8 = c8.KINDS
KINDS = pytest.mark.parametrize("kind", c8.KINDS, ids=["int8", "e4m3"])


@pytest.fixture(scope="module")
def rope(pkg):
    return importlib.import_module(f"{pkg.__name__}._qk_rope")


@pytest.fixture(scope="module")
def window(pkg):
    return importlib.import_module(f"{pkg.__name__}._window")


@pytest.fixture(scope="module")
def paged(pkg):
    return importlib.import_module(f"{pkg.__name__}._paged")


@pytest.fixture(scope="module")
def cache(pkg):
    return importlib.import_module(f"{pkg.__name__}._cache")


def randn(shape, seed, dev, dtype=BF, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(dev)


def ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def raw(t):
    return t.view(torch.uint8)


# --------------------------------------------------------------- written rows
# lengths, T, page, Hkv, D, dtype
WRITTEN = [
    ([1], 1, 8, 1, 16, BF),
    ([7, 100, 3], 3, 16, 2, 128, BF),
    ([130, 17], 17, 24, 5, 64, FP),
    ([40], 40, 64, 24, 96, F32),
    ([333, 300], 300, 16, 4, 80, BF),
    ([2000], 1999, 64, 8, 128, FP),
    ([5, 0, 2, 1000], 4, 8, 3, 32, F32),  # tokens before position 0, an idle slot, a length past the table
]


@KINDS
@pytest.mark.parametrize("case", WRITTEN, ids=[str(i) for i in range(len(WRITTEN))])
def test_append(cache, dev, kind, case):
    """Codes and powers of every row, bit by bit; every other slot as it was."""
    lengths, T, page, Hkv, D, dtype = case
    B, most = len(lengths), -(-min(max(lengths), 2000) // page)
    if max(lengths) == 1000:
        most = 9
    k, v = (randn((B, T, Hkv, D), s, dev, dtype) * 10.0 ** torch.linspace(-6, 3, Hkv, device=dev)[:, None].to(dtype) for s in (1, 2))
    table = c8.tables(B, most, dev)
    table[-1, -1] = -1 if B > 1 else table[-1, -1]
    caches = [c8.empty(B * most, page, Hkv, D, kind, dev) for _ in "kv"]
    want = [tuple(raw(t).cpu().clone() for t in c) for c in caches]
    for x, (codes, exps) in zip((k, v), want):
        c, e = c8.encode(x.cpu(), kind)
        for b, n in enumerate(lengths):
            for t in range(T):
                j = n - T + t
                if 0 <= j < most * page and int(table[b, j // page]) >= 0:
                    codes[int(table[b, j // page]), j % page] = raw(c[b, t])
                    exps[int(table[b, j // page]), :, j % page] = e[b, t]
    print("[append]", kind, case, flush=True)
    (kc, ks), (vc, vs) = caches
    assert cache.cache_append(k, v, kc, vc, table, ints(lengths, dev), ks, vs) is None
    for got, w in zip(caches, want):
        assert torch.equal(raw(got[1]).cpu(), w[1]), "powers"
        assert torch.equal(raw(got[0]).cpu(), w[0]), "codes"


@KINDS
@pytest.mark.parametrize("dtype", [BF, FP, F32])
def test_append_rows_at_the_edges(cache, dev, kind, dtype):
    """Largest values on and beside what the codes hold, halves, zeros, rows of next to
    nothing, the type's largest and smallest, infinities and NaN."""
    D, m = 32, c8.MOST[kind]
    inf, nan = float("inf"), float("nan")
    eps = torch.finfo(dtype).eps
    tops = [m, m * (1 + eps), m * (1 - eps), 2 * m, m / 2, m / 2 * (1 + 2 * eps), 1.0, 0.0, torch.finfo(dtype).max,
            torch.finfo(dtype).tiny, torch.finfo(dtype).smallest_normal * 2 ** -3, 2.0 ** -109, 2.0 ** -111, inf, -inf, nan, 128.0, 512.0]
    x = torch.zeros(1, len(tops), 1, D)
    for i, top in enumerate(tops):
        x[0, i, 0] = torch.linspace(-1, 1, D).cos() * (top if abs(top) < 1e30 else 1.0)
        x[0, i, 0, 3] = top
        if top == m:
            x[0, i, 0, 4:20] = torch.arange(16) + 0.5  # ties
            x[0, i, 0, 20:28] = torch.tensor([0.0, -0.0, 2.0 ** -10, 3 * 2.0 ** -10, -(2.0 ** -10), 2.0 ** -9, 17.0, 19.0])
    x = x.to(dtype)
    x[0, 13, 0, 5], x[0, 14, 0, 6] = inf, nan
    T = len(tops)
    (kc, ks), (vc, vs) = (c8.empty(T // 8 + 1, 8, 1, D, kind, dev) for _ in "kv")
    table = torch.arange(T // 8 + 1, dtype=torch.int32, device=dev)[None]
    cache.cache_append(x.to(dev), x.flip(1).to(dev), kc, vc, table, ints([T], dev), ks, vs)
    for got, exps, rows in ((kc, ks, x), (vc, vs, x.flip(1))):
        codes, byte = c8.encode(rows, kind)
        assert torch.equal(raw(exps).cpu().flatten()[:T], byte.flatten())
        have, want = got.cpu().flatten(0, 1)[:T, 0], codes[0, :, 0]
        if kind == I8:
            assert torch.equal(have, want)
        else:  # (minus zero is zero)
            assert torch.equal(torch.nan_to_num(have.float(), nan=-1.0), torch.nan_to_num(want.float(), nan=-1.0))
    k, v = cache.cache_read(kc, vc, table, ints([T], dev), ks, vs, tokens=T, dtype=FP if dtype == FP else BF)
    codes, byte = c8.encode(x, kind)
    want = c8.values(codes, byte).to(k.dtype)
    assert torch.equal(torch.nan_to_num(k.cpu(), nan=123.0), torch.nan_to_num(want, nan=123.0))
    assert torch.equal(v.flip(1).isnan(), k.isnan())


@KINDS
@pytest.mark.parametrize("B,T,H,Hkv,D,page,lengths,dtype,R,pairs", [
    (1, 1, 1, 1, 128, 16, [1], BF, 128, False), (3, 1, 24, 8, 128, 64, [100, 1, 65], BF, 128, True),
    (2, 40, 6, 3, 64, 16, [40, 55], FP, 32, False), (2, 300, 4, 4, 96, 24, [300, 471], F32, 96, True),
    (1, 9, 33, 11, 80, 8, [30], BF, 0, False), (2, 5, 8, 2, 128, 32, [3, 0], FP, 64, True),
])
def test_norm_rope_append(rope, dev, kind, B, T, H, Hkv, D, page, lengths, dtype, R, pairs):
    """q' and the codes of v are those of the calls apart; k' is off by half a step of the
    smallest power that holds it."""
    most = -(-max(lengths) // page)
    q, k, v = randn((B, T, H, D), 1, dev, dtype), randn((B, T, Hkv, D), 2, dev, dtype, 3.0), randn((B, T, Hkv, D), 3, dev, dtype)
    qw, kw = 1 + 0.2 * randn((D,), 4, dev, F32), 1 + 0.2 * randn((D,), 5, dev, F32)
    f = 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / max(R, 1))
    angle = torch.arange(max(lengths), dtype=torch.float64)[:, None] * f
    cos, sin = (angle.cos().float().to(dev), angle.sin().float().to(dev)) if R else (None, None)
    table, n = c8.tables(B, most, dev), ints(lengths, dev)
    (kc, ks), (vc, vs) = (c8.empty(B * most, page, Hkv, D, kind, dev) for _ in "kv")
    same = [torch.zeros(B * most, page, Hkv, D, dtype=dtype, device=dev) for _ in "kv"]
    print("[append8]", kind, B, T, H, Hkv, D, flush=True)
    got = rope.qk_norm_rope_append(q, k, v, kc, vc, table, n, qw, kw, cos, sin, interleaved=pairs, k_scale=ks, v_scale=vs)
    want = rope.qk_norm_rope_append(q, k, v, *same, table, n, qw, kw, cos, sin, interleaved=pairs)
    assert torch.equal(got, want)
    at = (n[:, None].long() - T + torch.arange(T, device=dev)).clamp_min(0)
    kn = ref.norm_rope(k, kw, cos, sin, at, pairs, 1e-6).cpu()
    codes, byte = c8.encode(v.cpu(), kind)
    kept = set()
    for b in range(B):
        for t in range(T):
            j = lengths[b] - T + t
            if j < 0:
                continue
            p, s = int(table[b, j // page]), j % page
            kept.add((p, s))
            assert torch.equal(raw(vc)[p, s].cpu(), raw(codes[b, t])) and torch.equal(raw(vs)[p, :, s].cpu(), byte[b, t])
            e = raw(ks)[p, :, s].cpu()
            unit, x = c8.power(e)[:, None], kn[b, t]
            # fp32 in front of the rounding: a few 2^-24 of the row's largest, 2^-18 here
            near = 2.0 ** -18 * x.abs().amax(-1, keepdim=True)
            top = x.abs().amax(-1, keepdim=True) / unit
            assert (top <= c8.MOST[kind] * (1 + 2.0 ** -18)).all() and (top > c8.MOST[kind] / 2 * (1 - 2.0 ** -18)).all()
            have = c8.values(kc[p, s].cpu(), e)
            half = unit / 2 if kind == I8 else torch.maximum(2.0 ** -4 * x.abs(), unit * 2.0 ** -10)
            assert ((have - x).abs() <= half + near).all()
    untouched = torch.ones(B * most, page, dtype=torch.bool)
    for p, s in kept:
        untouched[p, s] = False
    for c, e in ((kc, ks), (vc, vs)):
        assert (raw(c).cpu()[untouched] == 0x7F).all() and (raw(e).transpose(1, 2).cpu()[untouched] == 255).all()


# ------------------------------------------------------------------ read rows
@KINDS
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("lengths,tokens,start,page,Hkv,D", [
    ([1], 1, None, 8, 1, 16), ([70, 33, 0], 70, None, 16, 2, 128), ([300, 100], 50, [250, 60], 24, 3, 64),
    ([40, 5], 64, [-7, 2], 8, 5, 96), ([90], 30, [200], 64, 8, 80), ([500, 4000], 100, None, 16, 4, 64),
])
def test_read(cache, dev, kind, dtype, lengths, tokens, start, page, Hkv, D):
    """code times power, exactly; zeros outside the sequence, past the table and on bad pages."""
    B, most = len(lengths), -(-min(max(lengths), 500) // page)
    caches = []
    for s in (1, 2):
        codes, byte = c8.encode(randn((B * most, page, Hkv, D), s, dev, F32), kind)
        caches += [codes, byte.transpose(1, 2).contiguous().view(c8.E8)]
    kc, ks, vc, vs = caches
    table = c8.tables(B, most, dev)
    if B > 1:
        table[0, most // 2] = B * most
        table[1, 0] = -3
    got = cache.cache_read(kc, vc, table, ints(lengths, dev), ks, vs, tokens=tokens, start=None if start is None else ints(start, dev),
                           dtype=dtype)
    for x, c, e in ((got[0], kc, ks), (got[1], vc, vs)):
        want = torch.zeros(B, tokens, Hkv, D, dtype=torch.float64, device=dev)
        for b in range(B):
            for t in range(tokens):
                j = t + (start[b] if start else 0)
                p = int(table[b, j // page]) if 0 <= j < min(lengths[b], most * page) else -1
                if 0 <= p < B * most:
                    want[b, t] = c8.values(c[p, j % page], raw(e)[p, :, j % page])
        assert x.dtype == dtype and torch.equal(x, want.to(dtype))


# --------------------------------------------------------- attention over codes
# lengths, page, H, Hkv, D, window, sinks, dtype
PAGED = [
    ([1], 16, 1, 1, 128, None, 0, BF),
    ([0, 7, 64], 8, 24, 8, 128, None, 0, BF),
    ([1000, 333, 63, 64, 65], 16, 16, 4, 64, None, 0, FP),
    ([5000], 64, 24, 8, 128, 700, 4, BF),
    ([130, 4097], 24, 40, 2, 128, 100, 65, FP),
    ([900, 20], 136, 3, 3, 96, 64, 0, BF),
    ([70], 32, 34, 1, 80, 33, 40, FP),
    ([300] * 9, 256, 8, 8, 48, None, 0, BF),
    ([20000], 64, 4, 4, 64, None, 0, BF),
    ([33, 2000], 8, 6, 2, 16, 500, 3, FP),
]


def filled(B, L, page, Hkv, D, kind, dev, lengths, seeds=(1, 2), spread=True):
    """Caches whose slots behind the lengths read as NaN, their float64 rows [B, L, Hkv, D], the table."""
    most = -(-L // page)
    table = c8.tables(B, most, dev, seed=seeds[0])
    out, rows = [], []
    for s in seeds:
        x = randn((B, most * page, Hkv, D), s, dev, F32)
        if spread:  # rows of very different sizes
            x *= 2.0 ** randn((B, most * page, Hkv, 1), s + 50, dev, F32, 2.0)
        if s == seeds[0]:
            x = x / x.pow(2).mean(-1, keepdim=True).sqrt()
        codes, byte = c8.encode(x, kind)
        on = (torch.arange(most * page, device=dev) < ints(lengths, dev)[:, None])[:, :, None]
        byte = byte.masked_fill(~on, 255)
        codes = raw(codes).masked_fill(~on[..., None], 0x7F).view(kind)
        c, e = c8.empty(B * most, page, Hkv, D, kind, dev)
        at = table.long().flatten()
        raw(c)[at] = raw(codes).reshape(B * most, page, Hkv, D)
        raw(e)[at] = byte.reshape(B * most, page, Hkv).transpose(1, 2)
        out += [c, e]
        rows.append(c8.values(codes, byte)[:, :L].nan_to_num(0.0))
    return out, rows, table


@KINDS
@pytest.mark.parametrize("case", PAGED, ids=[str(i) for i in range(len(PAGED))])
def test_paged(paged, dev, kind, case):
    lengths, page, H, Hkv, D, w, sinks, dtype = case
    B, L = len(lengths), max(lengths)
    (kc, ks, vc, vs), (k, v), table = filled(B, L, page, Hkv, D, kind, dev, lengths)
    q = randn((B, 1, H, D), 3, dev, dtype, 2.0)
    on = torch.zeros((B, 1, L), dtype=torch.bool, device=dev)
    for b, e in enumerate(lengths):
        table[b, -(-e // page):] = -1 if b % 2 else 10 ** 9
        on[b, 0, :e] = True
        if w:
            on[b, 0, min(sinks, e):max(0, e - w)] = False
    print("[paged]", kind, case, flush=True)
    got = paged.paged_attn(q, kc, vc, table, ints(lengths, dev), window=w, sinks=sinks, k_scale=ks, v_scale=vs)
    o, p, (_, _, vh) = ref.attention(q, k, v, on, D ** -0.5)
    ref.close(got, o, c8.forward_bound(o, p, vh, dtype), "o")
    assert (got[ints(lengths, dev) == 0] == 0).all()


@KINDS
def test_paged_values_that_16_bits_hold(paged, cache, dev, kind):
    """The codes' values in a 16-bit cache: the same attention but for roundings."""
    B, L, page, H, Hkv, D = 2, 700, 16, 8, 2, 128
    (kc, ks, vc, vs), _, table = filled(B, L, page, Hkv, D, kind, dev, [700, 333], spread=False)
    n = ints([700, 333], dev)
    q = randn((B, 1, H, D), 3, dev)
    k, v = cache.cache_read(kc, vc, table, n, ks, vs, tokens=L)
    flat = torch.arange(B * 44, dtype=torch.int32, device=dev).reshape(B, 44)
    pad = lambda x: torch.nn.functional.pad(x, (0, 0, 0, 0, 0, 4)).reshape(B * 44, 16, Hkv, D)  # noqa: E731
    a = paged.paged_attn(q, kc, vc, table, n, k_scale=ks, v_scale=vs)
    b = paged.paged_attn(q, pad(k), pad(v), flat, n)
    on = torch.arange(L, device=dev)[None, None] < n[:, None, None]
    o, p, (_, _, vh) = ref.attention(q, k, v, on, D ** -0.5)
    ref.close(a, o, c8.forward_bound(o, p, vh, BF), "codes")
    ref.close(b, o, ref.forward_bound(o, p, vh, BF), "values")


@KINDS
def test_paged_bad_pages(paged, dev, kind):
    """Keys on page ids that the cache lacks are not visible, whatever page 0 holds; no pages: zeros."""
    B, page, Hkv, D = 2, 16, 2, 64
    (kc, ks, vc, vs), _, _ = filled(7, page, page, Hkv, D, kind, dev, [16] * 7)
    raw(ks)[0], raw(vs)[0] = 255, 255
    q = randn((B, 1, 4, D), 3, dev)
    table = ints([[3, 99, 1], [4, -5, 2]], dev)
    n = ints([41, 48], dev)
    rows = [c8.values(c, raw(e).transpose(1, 2)) for c, e in ((kc, ks), (vc, vs))]
    k, v = (torch.stack([torch.cat([x[3], x[1]]), torch.cat([x[4], x[2]])]) for x in rows)
    on = torch.arange(32, device=dev)[None, None] < ints([25, 32], dev)[:, None, None]
    o, p, (_, _, vh) = ref.attention(q, k, v, on, D ** -0.5)
    call = lambda t, n, a=kc, b=vc, s=ks, u=vs: paged.paged_attn(q, a, b, t, n, k_scale=s, v_scale=u)  # noqa: E731
    got = call(table, n)
    ref.close(got, o, c8.forward_bound(o, p, vh, BF), "o")
    assert torch.equal(call(table, ints([41, 2 ** 31 - 1], dev)), got)
    assert (call(table, ints([-4, 48], dev))[0] == 0).all()
    assert (call(table, n, kc[:0], vc[:0], ks[:0], vs[:0]) == 0).all()


@pytest.mark.parametrize("kind", [None] + c8.KINDS, ids=["same", "int8", "e4m3"])
@pytest.mark.parametrize("B,H,Hkv,D,page", [(3, 64, 64, 64, 16), (70, 16, 8, 64, 8), (256, 8, 8, 128, 16), (300, 4, 4, 64, 32)])
def test_paged_ragged_batches(paged, dev, kind, B, H, Hkv, D, page):
    """Launches whose workgroups go by length: idle slots, equal and very different lengths."""
    g = torch.Generator().manual_seed(B)
    lengths = torch.randint(0, 600, (B,), generator=g).tolist()
    lengths[0], lengths[-1], lengths[B // 2] = 0, 0, 1000
    lengths[1] = lengths[2] = 300
    L = max(lengths)
    n = ints(lengths, dev)
    q = randn((B, 1, H, D), 3, dev, BF, 2.0)
    if kind is None:
        most = -(-L // page)
        k, v = (randn((B, most * page, Hkv, D), s, dev) for s in (1, 2))
        table = torch.arange(B * most, dtype=torch.int32, device=dev).reshape(B, most)
        got = paged.paged_attn(q, k.view(B * most, page, Hkv, D), v.view(B * most, page, Hkv, D), table, n)
        k, v = k[:, :L], v[:, :L]
    else:
        (kc, ks, vc, vs), (k, v), table = filled(B, L, page, Hkv, D, kind, dev, lengths, spread=False)
        got = paged.paged_attn(q, kc, vc, table, n, k_scale=ks, v_scale=vs)
    on = (torch.arange(L, device=dev) < n[:, None])[:, None]
    for b0 in range(0, B, 64):
        s = slice(b0, b0 + 64)
        o, p, (_, _, vh) = ref.attention(q[s], k[s], v[s], on[s], D ** -0.5)
        ref.close(got[s], o, (ref if kind is None else c8).forward_bound(o, p, vh, BF), "o")
    assert (got[n == 0] == 0).all()


# ------------------------------------------------------------------ shared keys
# per, groups, prefix, rests, page, H, Hkv, D, dtype
SHARED = [
    (2, 1, 100, [1, 5], 16, 1, 1, 128, BF),
    (8, 1, 4100, [30, 1, 7, 300, 64, 2, 31, 33], 64, 24, 8, 128, BF),
    (16, 2, 777, [10] * 32, 16, 16, 4, 64, FP),
    (5, 3, 64, [3, 4, 5, 6, 7] * 3, 8, 6, 2, 128, FP),
    (3, 1, 33, [1, 200, 900], 24, 40, 2, 128, BF),
    (11, 1, 1000, [9] * 11, 32, 3, 3, 96, BF),
    (40, 1, 513, [17] * 40, 16, 10, 1, 80, FP),
    (1, 4, 200, [5, 6, 7, 8], 64, 8, 8, 64, BF),
    (64, 1, 2048, [3] * 64, 64, 24, 8, 128, BF),
    (130, 2, 300, [20] * 260, 64, 4, 1, 64, BF),
    (70, 1, 150, [40] * 70, 16, 16, 2, 128, FP),
]


@pytest.mark.parametrize("kind", [None] + c8.KINDS, ids=["same", "int8", "e4m3"])
@pytest.mark.parametrize("case", SHARED, ids=[str(i) for i in range(len(SHARED))])
def test_shared(paged, dev, kind, case):
    """Against float64; an idle slot, a sequence that ends inside the shared keys; every sequence has copies
    of its own, and only the longest of a run has pages for the shared keys that are any."""
    per, groups, prefix, rests, page, H, Hkv, D, dtype = case
    if kind is not None and D % 16:
        pytest.skip("head dim of an 8-bit cache")
    B = per * groups
    lengths = [prefix + r for r in rests]
    if per > 2:
        lengths[1] = 0
        lengths[per - 1] = max(prefix // 2 - 3, 1)
    L = max(lengths)
    q = randn((B, 1, H, D), 3, dev, dtype, 2.0)
    n = ints(lengths, dev)
    if kind is None:
        most = -(-L // page)
        table = c8.tables(B, most, dev)
        k, v = (randn((B, most * page, Hkv, D), s, dev, dtype) for s in (1, 2))
        for x in (k, v):
            x.view(groups, per, *x.shape[1:])[:, :, :prefix] = x.view(groups, per, *x.shape[1:])[:, :1, :prefix].clone()
        on = (torch.arange(most * page, device=dev) < n[:, None])[:, :, None, None]
        kc, vc = (torch.empty(B * most, page, Hkv, D, dtype=dtype, device=dev) for _ in "kv")
        for c, x in ((kc, k), (vc, v)):
            c[table.long().flatten()] = x.masked_fill(~on, float("nan")).reshape(B * most, page, Hkv, D)
        k, v, scales = k[:, :L], v[:, :L], {}
    else:
        (kc, ks, vc, vs), (k, v), table = filled(B, L, page, Hkv, D, kind, dev, [L] * B, spread=False)
        at = torch.arange(B, device=dev) // per * per
        for c, e in ((kc, ks), (vc, vs)):  # the first sequence's shared rows to every one of its run
            for j in range(prefix):
                src, dst = table[at, j // page].long(), table[:, j // page].long()
                raw(c)[dst, j % page] = raw(c)[src, j % page]
                raw(e)[dst, :, j % page] = raw(e)[src, :, j % page]
        k, v = (x.clone() for x in (k, v))
        for x in (k, v):
            x[:, :prefix] = x[at, :prefix]
        scales = dict(k_scale=ks, v_scale=vs)
    first = [g * per + max(range(per), key=lambda i: (lengths[g * per + i], -i)) for g in range(groups)]
    for b in range(B):
        if b not in first:
            table[b, :prefix // page] = -1 if b % 2 else 10 ** 9
    on = (torch.arange(L, device=dev) < n[:, None])[:, None]
    print("[shared]", kind, case, flush=True)
    got = paged.paged_attn(q, kc, vc, table, n, shared=prefix, groups=groups, **scales)
    o, p, (_, _, vh) = ref.attention(q, k, v, on, D ** -0.5)
    # Where many rows share the keys, codes become 16-bit values (exactly) and P is rounded
    # once to the type, u of P, as over a 16-bit cache: that bound. Elsewhere P keeps two parts.
    once = kind is None or (per * (H // Hkv) > 16 and D in (64, 128))
    bound = ref.forward_bound(o, p, vh, dtype) if once else c8.forward_bound(o, p, vh, dtype)
    ref.close(got, o, bound, "o")
    assert (got[n == 0] == 0).all()


@pytest.mark.parametrize("kind", [None] + c8.KINDS, ids=["same", "int8", "e4m3"])
@pytest.mark.parametrize("page,D", [(8, 128), (64, 64), (24, 128)])
def test_shared_long(paged, dev, kind, page, D):
    """Many tiles of rows over a long prefix, pages that are none of the cache's among its own."""
    prefix, rests, H, Hkv = 40000, [3, 70], 256, 2
    B, L = 2, prefix + max(rests)
    most = -(-L // page)
    n = ints([prefix + r for r in rests], dev)
    q = randn((B, 1, H, D), 3, dev, BF, 2.0)
    table = torch.randperm(B * most, generator=torch.Generator().manual_seed(3)).to(torch.int32).reshape(B, most).to(dev)
    table[0, :prefix // page] = table[1, :prefix // page]
    bad = torch.tensor([5, 700 // page * 3, prefix // page // 2], device=dev)
    k, v = (randn((B * most, page, Hkv, D), s, dev) for s in (1, 2))
    scales = {}
    if kind is not None:
        coded = [c8.encode(x, kind) for x in (k, v)]
        k, v = (c8.values(*c).to(BF) for c in coded)
        (kc, vc), (ks, vs) = ([c[0] for c in coded], [c[1].transpose(1, 2).contiguous().view(c8.E8) for c in coded])
        scales = dict(k_scale=ks, v_scale=vs)
    else:
        kc, vc = k, v
    rows = [torch.stack([x[table[b].long()].flatten(0, 1)[:L] for b in range(B)]) for x in (k, v)]
    for x in rows:
        x[:, :prefix] = x[1:, :prefix]
    table[:, bad] = ints([-1, B * most, -5], dev)
    on = (torch.arange(L, device=dev) < n[:, None])[:, None].clone()
    for p in bad.tolist():
        on[..., p * page:(p + 1) * page] = False
    got = paged.paged_attn(q, kc, vc, table, n, shared=prefix, **scales)
    o, p, (_, _, vh) = ref.attention(q, *rows, on, D ** -0.5)
    ref.close(got, o, ref.forward_bound(o, p, vh, BF), "o")  # (many rows: P in one rounding)


@pytest.mark.parametrize("kind", [None, F8], ids=["same", "e4m3"])
@pytest.mark.parametrize("page,D", [(8, 64), (16, 128)])
def test_shared_in_one_part(paged, dev, kind, page, D):
    """So many rows that none of the keys are split: one part of more than 128 tiles, whose page ids
    are held 64 tiles at a time."""
    B, H, n = 512, 128, 8300
    most = -(-n // page)
    q = randn((B, 1, H, D), 3, dev, BF, 2.0)
    table = torch.randperm(most, generator=torch.Generator().manual_seed(5)).to(torch.int32).to(dev)[None].repeat(B, 1)
    k, v = (randn((most, page, 1, D), s, dev) for s in (1, 2))
    scales = {}
    kc, vc = k, v
    if kind is not None:
        coded = [c8.encode(x, kind) for x in (k, v)]
        k, v = (c8.values(*c).to(BF) for c in coded)
        (kc, vc), (ks, vs) = ([c[0] for c in coded], [c[1].transpose(1, 2).contiguous().view(c8.E8) for c in coded])
        scales = dict(k_scale=ks, v_scale=vs)
    table[:, 40] = -1
    at = table[0].long().clamp_min(0)
    kd, vd = (x[at].flatten(0, 1)[:n, 0].double() for x in (k, v))
    on = torch.ones(n, dtype=torch.bool, device=dev)
    on[40 * page:41 * page] = False
    lengths = torch.full((B,), n, dtype=torch.int32, device=dev)
    lengths[7] = 0
    got = paged.paged_attn(q, kc, vc, table, lengths, shared=n, **scales)
    assert (got[7] == 0).all()
    got[7] = got[6]
    u = ref.half_step(BF)
    for b in range(0, B, 64):
        rows = q[b:b + 64].clone()
        if b == 0:
            rows[7] = rows[6]
        p = torch.softmax((rows.flatten(0, 2).double() @ kd.T * D ** -0.5).masked_fill(~on, float("-inf")), -1)
        o, pv = p @ vd, p @ vd.abs()
        bound = (u * (2 * o.abs() + pv) + 2 * 2.0 ** -13 * pv) * 1.01  # that of _operators.forward_bound
        ref.close(got[b:b + 64].flatten(0, 2), o, bound, "o")


@pytest.mark.parametrize("shared", [1, 31, 64, 500, 2 ** 40])
def test_shared_sizes(paged, dev, shared):
    """Any number of shared keys that the sequences have in common, more than any holds too."""
    page, Hkv, D = 16, 2, 64
    one = torch.arange(40, dtype=torch.int32, device=dev)[None].repeat(6, 1)
    kc, vc = (randn((40, page, Hkv, D), s, dev) for s in (1, 2))
    q = randn((6, 1, 4, D), 3, dev)
    n = ints([640, 1, 0, 500, 64, 33], dev)
    got = paged.paged_attn(q, kc, vc, one, n, shared=shared)
    on = (torch.arange(640, device=dev) < n[:, None])[:, None]
    k, v = (x.view(1, 640, Hkv, D).expand(6, -1, -1, -1) for x in (kc, vc))
    o, p, (_, _, vh) = ref.attention(q, k, v, on, D ** -0.5)
    ref.close(got, o, ref.forward_bound(o, p, vh, BF), "o")
    assert torch.equal(paged.paged_attn(q, kc, vc, one, n, shared=0), paged.paged_attn(q, kc, vc, one, n))
    none = ints([0, -4, 0, 0, 0, 0], dev)
    assert (paged.paged_attn(q, kc, vc, one, none, shared=shared) == 0).all()


def test_shared_idle_slots_see_nothing(paged, dev):
    """NaN in the shared values reaches those that see them, not the idle slots beside them."""
    page, Hkv, D = 16, 1, 128
    kc, vc = (randn((20, page, Hkv, D), s, dev) for s in (1, 2))
    vc[3, 5] = float("nan")
    t = torch.arange(20, dtype=torch.int32, device=dev)[None].repeat(5, 1)
    got = paged.paged_attn(randn((5, 1, 2, D), 3, dev), kc, vc, t, ints([320, 0, 300, 0, 0], dev), shared=290)
    assert got[[0, 2]].isnan().all() and (got[[1, 3, 4]] == 0).all()


# ------------------------------------------------------------------- together
@KINDS
def test_prompt_in_pieces_then_tokens(rope, window, paged, cache, dev, kind):
    """As they are used: a prompt in two pieces into the cache, each attending to what was read
    back; two answers to it that share its keys, token by token, the new ones in pages of their own.
    The whole against float64 over the cache's values."""
    T, cut, new, page, H, Hkv, D, answers = 150, 90, 12, 16, 6, 2, 128, 3
    qkv = randn((1, T, H + 2 * Hkv, D), 5, dev)
    qw, kw = 1 + 0.1 * randn((D,), 6, dev, F32), 1 + 0.1 * randn((D,), 7, dev, F32)
    f = 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    angle = torch.arange(T + new, dtype=torch.float64)[:, None] * f
    cos, sin = angle.cos().float().to(dev), angle.sin().float().to(dev)
    pages = -(-(T + new) // page)
    whole = T // page
    (kc, ks), (vc, vs) = (c8.empty(answers * pages, page, Hkv, D, kind, dev) for _ in "kv")
    table = c8.tables(answers, pages, dev)
    table[1:, :whole] = table[:1, :whole]
    s = dict(k_scale=ks, v_scale=vs)
    for a, b in ((0, cut), (cut, T)):
        q, k, v = qkv[:, a:b].split([H, Hkv, Hkv], 2)
        n = ints([b], dev)
        qp = rope.qk_norm_rope_append(q, k, v, kc, vc, table[:1], n, qw, kw, cos, sin, **s)
        kr, vr = cache.cache_read(kc, vc, table[:1], n, ks, vs, tokens=b)
        got = window.window_attn(qp, kr, vr, window=None)
        on = ref.seen(b - a, b, a, None, 0, True, None, 1, dev)
        o, p, (_, _, vh) = ref.attention(qp, kr, vr, on, D ** -0.5)
        ref.close(got, o, ref.forward_bound(o, p, vh, BF), "prompt")
    for c, e in ((kc, ks), (vc, vs)):  # the page that the prompt ends in: a copy for each answer
        for b in range(1, answers):
            raw(c)[int(table[b, whole])] = raw(c)[int(table[0, whole])]
            raw(e)[int(table[b, whole])] = raw(e)[int(table[0, whole])]
    for t in range(new):
        q, k, v = randn((answers, 1, H + 2 * Hkv, D), 20 + t, dev).split([H, Hkv, Hkv], 2)
        n = ints([T + t + 1] * answers, dev)
        qp = rope.qk_norm_rope_append(q, k, v, kc, vc, table, n, qw, kw, cos, sin, **s)
        got = paged.paged_attn(qp, kc, vc, table, n, shared=T, **s)
        kr, vr = cache.cache_read(kc, vc, table, n, ks, vs, tokens=T + t + 1)
        on = torch.ones(answers, 1, T + t + 1, dtype=torch.bool, device=dev)
        o, p, (_, _, vh) = ref.attention(qp, kr, vr, on, D ** -0.5)
        ref.close(got, o, c8.forward_bound(o, p, vh, BF), "token")
        apart = paged.paged_attn(qp, kc, vc, table, n, **s)
        ref.close(apart, o, c8.forward_bound(o, p, vh, BF), "token, without sharing")


@KINDS
def test_other_stream_and_graph(rope, paged, cache, dev, kind):
    """On a stream of its own, and captured once and replayed on new contents with eager work
    between the replays: the eager bits every time."""
    B, T, L, page, H, Hkv, D = 4, 3, 200, 16, 8, 2, 64
    (kc, ks, vc, vs), _, table = filled(B, L, page, Hkv, D, kind, dev, [L] * B)
    q, k, v = (randn((B, T, h, D), i, dev) for i, h in enumerate((H, Hkv, Hkv)))
    n = ints([L, 150, 0, 77], dev)
    w = 1 + 0.1 * randn((D,), 4, dev, F32)

    def step():
        qp = rope.qk_norm_rope_append(q, k, v, kc, vc, table, n, w, w, k_scale=ks, v_scale=vs)
        cache.cache_append(k + 1, v, kc, vc, table, n - T, ks, vs)
        last = qp[:, -1:].contiguous()
        a = paged.paged_attn(last, kc, vc, table, n, k_scale=ks, v_scale=vs)
        b = paged.paged_attn(last, kc, vc, table, n, k_scale=ks, v_scale=vs, shared=60, groups=2)
        return [qp, a, b, *cache.cache_read(kc, vc, table, n, ks, vs, tokens=L)]

    def same(x, y):
        return all(torch.equal(torch.nan_to_num(a, nan=9.0), torch.nan_to_num(b, nan=9.0)) for a, b in zip(x, y))

    want = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step()
    torch.cuda.current_stream().wait_stream(s)
    assert same(got, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for i in range(4):
        for x, h in ((q, H), (k, Hkv), (v, Hkv)):
            x.copy_(randn(tuple(x.shape), 30 + 3 * i + h, dev))
        n.copy_(ints([L - i, 150, i * 9, 77], dev))
        g.replay()
        torch.cuda.synchronize()
        first = [t.clone() for t in out]
        assert same(step(), first)


@KINDS
def test_offsets_beyond_32_bits(paged, cache, dev, kind):
    """Pages past 2^32 bytes of a cache are written, read and attended."""
    page, Hkv, D = 64, 8, 128
    pages = (1 << 32) // (page * Hkv * D) + 40
    kc, vc = (torch.empty(pages, page, Hkv, D, dtype=torch.uint8, device=dev).view(kind) for _ in "kv")
    ks, vs = (torch.empty(pages, Hkv, page, dtype=torch.uint8, device=dev).view(c8.E8) for _ in "kv")
    table = (pages - 1 - torch.arange(6, dtype=torch.int32, device=dev)).reshape(2, 3)
    n = ints([192, 100], dev)
    k, v = randn((2, 100, Hkv, D), 1, dev), randn((2, 100, Hkv, D), 2, dev)
    raw(ks)[table.long()] = 0
    raw(vs)[table.long()] = 0
    raw(kc)[table.long()] = 0
    raw(vc)[table.long()] = 0
    cache.cache_append(k, v, kc, vc, table, n, ks, vs)
    got = cache.cache_read(kc, vc, table, n, ks, vs, tokens=192)
    want = [c8.values(*c8.encode(x, kind)).to(BF) for x in (k, v)]
    for g, w in zip(got, want):
        assert torch.equal(g[0, 92:], w[0]) and torch.equal(g[1, :100], w[1]) and (g[0, :92] == 0).all()
    q = randn((2, 1, 16, D), 3, dev)
    o, p, (_, _, vh) = ref.attention(q, *got, torch.arange(192, device=dev)[None, None] < n[:, None, None], D ** -0.5)
    ref.close(paged.paged_attn(q, kc, vc, table, n, k_scale=ks, v_scale=vs), o, c8.forward_bound(o, p, vh, BF), "o")


@KINDS
def test_cache_orders_and_views(paged, cache, rope, dev, kind):
    """Heads before slots, k and v side by side, a table that is a view: the same bits as dense ones."""
    B, page, H, Hkv, D = 3, 16, 4, 2, 64
    kv = torch.randint(0, 120, (9, 2, page, Hkv, D), dtype=torch.uint8, device=dev)
    e = torch.randint(118, 124, (9, 2, Hkv, page), dtype=torch.uint8, device=dev)
    wide = torch.randint(0, 9, (B, 8), dtype=torch.int32, device=dev)
    table, n = wide[:, 2:6], ints([60, 1, 33], dev)
    q = randn((B, 1, H, D), 2, dev)
    k, v, ks, vs = kv[:, 0].view(kind), kv[:, 1].view(kind), e[:, 0].view(c8.E8), e[:, 1].view(c8.E8)
    dense = [raw(t).clone(memory_format=torch.contiguous_format).view(t.dtype) for t in (k, v, ks, vs)]
    want = paged.paged_attn(q, dense[0], dense[1], table.contiguous(), n, k_scale=dense[2], v_scale=dense[3])
    assert torch.isfinite(want).all()
    assert torch.equal(paged.paged_attn(q, k, v, table, n, k_scale=ks, v_scale=vs), want)
    heads = [raw(t).transpose(1, 2).contiguous().transpose(1, 2).view(kind) for t in (k, v)]
    assert torch.equal(paged.paged_attn(q, *heads, table, n, k_scale=ks, v_scale=vs), want)
    kn, vn = randn((B, 1, 2 * Hkv, D), 3, dev)[:, :, ::2], randn((B, 1, Hkv, 2 * D), 4, dev)[..., :D]
    uniq, m = torch.arange(9, dtype=torch.int32, device=dev).reshape(B, 3), ints([48, 1, 17], dev)
    cache.cache_append(kn, vn, k, v, uniq, m, ks, vs)
    cache.cache_append(kn.contiguous(), vn.contiguous(), dense[0], dense[1], uniq, m, dense[2], dense[3])
    for a, b in zip((k, v, ks, vs), dense):
        assert torch.equal(raw(a), raw(b))
    a = cache.cache_read(k, v, table, n, ks, vs, tokens=50)
    b = cache.cache_read(*dense[:2], table.contiguous(), n, *dense[2:], tokens=50)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_empty_calls(paged, cache, rope, dev):
    """No tokens, no sequences, no pages: nothing is written, zeros are read."""
    (kc, ks), (vc, vs) = (c8.empty(4, 16, 2, 64, I8, dev) for _ in "kv")
    before = raw(kc).clone()
    t, n = torch.zeros(2, 2, dtype=torch.int32, device=dev), ints([5, 0], dev)
    x = randn((2, 0, 2, 64), 1, dev)
    cache.cache_append(x, x, kc, vc, t, n, ks, vs)
    assert cache.cache_read(kc, vc, t, n, ks, vs, tokens=0)[0].shape == (2, 0, 2, 64)
    assert (cache.cache_read(kc[:0], vc[:0], t, n, ks[:0], vs[:0], tokens=3)[1] == 0).all()
    assert (cache.cache_read(kc, vc, t[:, :0], n, ks, vs, tokens=3)[1] == 0).all()
    y = randn((2, 1, 2, 64), 1, dev)
    cache.cache_append(y, y, kc[:0], vc[:0], t, n, ks[:0], vs[:0])
    cache.cache_append(y, y, kc, vc, t[:, :0], n, ks, vs)
    got = rope.qk_norm_rope_append(y, y, y, kc[:0], vc[:0], t, n, k_scale=ks[:0], v_scale=vs[:0])
    assert torch.isfinite(got).all() and torch.equal(raw(kc), before)
    assert cache.cache_read(kc, vc, t[:0], n[:0], ks, vs, tokens=3)[0].shape == (0, 3, 2, 64)
    assert (paged.paged_attn(y, kc, vc, t[:, :0], n, k_scale=ks, v_scale=vs) == 0).all()


def test_refusals(paged, cache, rope, dev):
    (kc, ks), (vc, vs) = (c8.empty(4, 16, 2, 64, I8, dev) for _ in "kv")
    t, n = torch.zeros(1, 2, dtype=torch.int32, device=dev), ints([5], dev)
    x, q = randn((1, 1, 2, 64), 1, dev), randn((1, 1, 4, 64), 2, dev)

    def all_three(text, k=kc, v=vc, a=ks, b=vs, table=t, lengths=n, x=x, read=True):
        for f in (lambda: cache.cache_append(x, x, k, v, table, lengths, a, b),
                  lambda: rope.qk_norm_rope_append(x, x, x, k, v, table, lengths, k_scale=a, v_scale=b),
                  lambda: paged.paged_attn(x, k, v, table, lengths, k_scale=a, v_scale=b),
                  lambda: cache.cache_read(k, v, table, lengths, a, b, tokens=3))[:4 if read else 3]:
            with pytest.raises(ValueError, match=text):
                f()

    all_three("dtype", k=kc.to(BF), v=vc.to(BF))
    all_three("differs", v=raw(vc).view(F8))
    all_three("float8_e8m0fnu", a=raw(ks))
    all_three("float8_e8m0fnu", b=vs[:, :1])
    all_three("float8_e8m0fnu", a=ks[:3])
    all_three("contiguous and 8-byte", a=torch.zeros(4, 2, 32, dtype=torch.uint8, device=dev)[:, :, ::2].view(c8.E8))
    all_three("int32", lengths=n.long())
    all_three("page_table", table=t[0])
    all_three("16-byte aligned", k=torch.zeros(4 * 16 * 2 * 64 + 8, dtype=torch.int8, device=dev)[8:].view(4, 16, 2, 64))
    all_three("head_dim", x=randn((1, 1, 2, 32), 1, dev), read=False)
    y = randn((1, 1, 2, 24), 1, dev)
    small = [torch.zeros(4, 16, 2, 24, dtype=torch.int8, device=dev) for _ in "kv"]
    all_three("multiples of 16", k=small[0], v=small[1], x=y)
    for f in (lambda k, v, a, b: cache.cache_append(x, x, k, v, t, n, a, b),
              lambda k, v, a, b: rope.qk_norm_rope_append(x, x, x, k, v, t, n, k_scale=a, v_scale=b)):
        with pytest.raises(ValueError, match="same memory"):
            f(kc, kc, ks, vs)
        with pytest.raises(ValueError, match="same memory"):
            f(kc, vc, ks, ks)
        with pytest.raises(ValueError, match="expanded"):
            f(kc[:1].expand(4, -1, -1, -1), vc, ks, vs)
        with pytest.raises(ValueError, match="expanded"):
            f(kc, vc, ks[:1].expand(4, -1, -1), vs)
    with pytest.raises(ValueError, match="go together"):
        paged.paged_attn(q, kc, vc, t, n, k_scale=ks)
    with pytest.raises(ValueError, match="go together"):
        rope.qk_norm_rope_append(q, x, x, kc, vc, t, n, v_scale=vs)
    with pytest.raises(ValueError, match="differs from q"):
        paged.paged_attn(q, kc, vc, t, n)
    with pytest.raises(ValueError, match="start"):
        cache.cache_read(kc, vc, t, n, ks, vs, tokens=3, start=ints([1, 2], dev))
    with pytest.raises(ValueError, match="-1 tokens"):
        cache.cache_read(kc, vc, t, n, ks, vs, tokens=-1)
    with pytest.raises(ValueError, match="bfloat16 or float16"):
        cache.cache_read(kc, vc, t, n, ks, vs, tokens=1, dtype=F32)
    with pytest.raises(ValueError, match="shapes do not match"):
        cache.cache_append(x, x[:, :, :1], kc, vc, t, n, ks, vs)
    with pytest.raises(ValueError, match="no gradient"):
        cache.cache_append(x.clone().requires_grad_(True), x, kc, vc, t, n, ks, vs)
    k2, v2 = randn((4, 16, 2, 64), 1, dev), randn((4, 16, 2, 64), 2, dev)
    for kw, text in ((dict(shared=-1), "shared -1"), (dict(groups=0), "groups"), (dict(groups=2), "groups"),
                     (dict(shared=4, window=3), "window"), (dict(shared=4, sinks=1), "window")):
        with pytest.raises(ValueError, match=text):
            paged.paged_attn(q, k2, v2, t, n, **kw)


def test_append_is_a_change_of_the_cache(cache, dev):
    (kc, ks), (vc, vs) = (c8.empty(4, 16, 2, 64, F8, dev) for _ in "kv")
    before = [x._version for x in (kc, ks, vc, vs)]
    x = randn((1, 1, 2, 64), 1, dev)
    cache.cache_append(x, x, kc, vc, torch.zeros(1, 1, dtype=torch.int32, device=dev), ints([5], dev), ks, vs)
    assert all(x._version > b for x, b in zip((kc, ks, vc, vs), before))
