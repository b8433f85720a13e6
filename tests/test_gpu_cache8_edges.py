"""What the 8-bit cache and attention over shared keys do at their edges: values that a
sequence must not see, values beyond fp16's range, runs that are shorter than the shared
keys, wide tables and far pages. Bounds and references as in test_gpu_cache8.py."""

import importlib

import pytest
import torch

import _cache8 as c8
import _operators as ref

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32
I8, F8 = c8.KINDS
CODES = pytest.mark.parametrize("kind", c8.KINDS, ids=["int8", "e4m3"])
KINDS = pytest.mark.parametrize("kind", [None] + c8.KINDS, ids=["same", "int8", "e4m3"])


@pytest.fixture(scope="module")
def rope(pkg):
    return importlib.import_module(f"{pkg.__name__}._qk_rope")


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


class Pages:
    """Rows k, v [B, L, Hkv, D] (fp32) in scattered pages, of `kind` (None: of dtype); at:
    whose rows a sequence's are. k, v become what the cache holds, in float64."""

    def __init__(self, k, v, at, page, kind, dtype, wide=0):
        dev, (B, L, Hkv, D) = k.device, k.shape
        self.most = -(-L // page) + wide
        self.table = c8.tables(B, self.most, dev, seed=L)[torch.as_tensor(at, device=dev)]
        own = c8.tables(B, self.most, dev, seed=L)
        self.scales, out = {}, []
        for name, x in (("k", k), ("v", v)):
            x = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, self.most * page - L))
            if kind is None:
                c, e, x = x.to(dtype), None, x.to(dtype).double()
                held = torch.empty(B * self.most, page, Hkv, D, dtype=dtype, device=dev)
                held[own.long().flatten()] = c.reshape(B * self.most, page, Hkv, D)
            else:
                c, e = c8.encode(x, kind)
                x = c8.values(c, e)
                held, s = c8.empty(B * self.most, page, Hkv, D, kind, dev)
                raw(held)[own.long().flatten()] = raw(c).reshape(B * self.most, page, Hkv, D)
                raw(s)[own.long().flatten()] = e.reshape(B * self.most, page, Hkv).transpose(1, 2)
                self.scales[f"{name}_scale"] = s
            setattr(self, name, held)
            out.append(x[torch.as_tensor(at, device=dev)][:, :L])
        self.rows = out

    def attn(self, paged, q, n, **kw):
        return paged.paged_attn(q, self.k, self.v, self.table, n, **self.scales, **kw)


def seen(n, L):
    return (torch.arange(L, device=n.device) < n[:, None])[:, None]


def bound(kind, o, p, v, dtype, columns, D):
    """P is rounded once over 16-bit pages and over tiles (more than 64 columns), else kept in two parts."""
    once = kind is None or (columns > 64 and D in (64, 128))
    return (ref if once else c8).forward_bound(o, p, v, dtype)


# ------------------------------------------------------ keys behind a sequence's end
# run's lengths, shared, groups, H, Hkv, D, page, dtype: 2 and 15 columns, two tiles of 16, more than 64 by tiles
# of 128 rows or, of other head dims, by tiles of 32
ENDS = [
    ([320, 1, 0, 290, 289, 64, 96], 290, 1, 2, 1, 128, 16, BF),
    ([1200, 1000, 999, 513, 512, 511, 128], 1000, 1, 12, 4, 64, 24, FP),
    ([100, 2100, 2000, 1990, 1024, 7, 2000, 1536], 2000, 2, 24, 8, 128, 64, BF),
    ([3000, 2900, 2048, 2047, 2049, 64, 0, 1], 2900, 1, 32, 2, 128, 64, BF),
    ([640, 641, 700, 63, 64, 65, 127, 128, 129, 320], 641, 1, 16, 2, 64, 8, FP),
    ([900, 850, 33, 450], 850, 1, 40, 2, 96, 16, BF),
    ([500, 499, 64, 500, 0], 2000, 1, 40, 2, 128, 16, BF),
]


@KINDS
@pytest.mark.parametrize("poison", [float("nan"), float("inf")], ids=["nan", "inf"])
@pytest.mark.parametrize("case", ENDS, ids=[str(i) for i in range(len(ENDS))])
def test_shared_keys_behind_the_end_of_a_sequence(paged, dev, kind, case, poison):
    """NaN or infinities in shared rows that a sequence does not have do not reach it, in k or in v: the
    sequences that end before them are exact, the others NaN or infinite."""
    run, shared, groups, H, Hkv, D, page, dtype = case
    lengths = run * groups
    B, per, L = len(lengths), len(run), max(run)
    q = randn((B, 1, H, D), 3, dev, dtype, 2.0)
    k, v = (randn((B, L, Hkv, D), s, dev, F32) for s in (1, 2))
    longest = run.index(L)
    first = [b // per * per + longest for b in range(B)]
    for x in (k, v):
        x[:, :min(shared, L)] = x[first, :min(shared, L)]
    n = ints(lengths, dev)
    on = seen(n, L)
    ends = sorted({m for m in run if 0 < m < min(shared, L)})
    for bad in (ends[0], ends[len(ends) // 2], ends[-1]):  # the first key that one of the sequences does not have
        for which in ("k", "v"):
            kp, vp = k.clone(), v.clone()
            (kp if which == "k" else vp)[:, bad, :, 3 % D] = poison
            pages = Pages(kp, vp, range(B), page, kind, dtype)
            print("[ends]", kind, case, poison, bad, which, flush=True)
            got = pages.attn(paged, q, n, shared=shared, groups=groups)
            safe = n <= bad
            rows = [x.masked_fill(~on.transpose(1, 2)[..., None], 0).nan_to_num(0.0, 0.0, 0.0) for x in pages.rows]
            o, p, (_, _, vh) = ref.attention(q, *rows, on, D ** -0.5)
            tol = bound(kind, o, p, vh, dtype, per * (H // Hkv), D)
            ref.close(got[safe], o[safe], tol[safe], "sequences that end before it")
            if which == "v":  # (an infinity in k may be a score of minus infinity)
                assert not torch.isfinite(got[~safe]).flatten(1).all(1).any()


# ------------------------------------------------------- values that fp16 does not have
@CODES
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B", [5, 20, 40])  # 10 columns, 40, 80 (by tiles of 128 rows)
def test_fp16_queries_over_values_beyond_fp16(paged, cache, dev, kind, D, B):
    """fp16 rows at the type's largest value, which their codes round up beyond it, and rows of a bf16
    model far beyond: finite results, the same whatever the number of columns."""
    H, Hkv, page, L = 4, 2, 16, 700
    most = -(-L // page)
    table = torch.arange(most, dtype=torch.int32, device=dev)[None].repeat(B, 1)
    n = ints([L] * B, dev)
    q = randn((B, 1, H, D), 3, dev, FP)
    q[..., 5] = 0
    for dtype, top, keys in ((FP, 65504.0, L), (BF, 1e6, L), (FP, 65504.0, 1)):
        k, v = (randn((1, L, Hkv, D), s, dev, F32) for s in (1, 2))
        k[:, 7:7 + keys:3, :, 5] = top       # no query looks at this channel
        v[:, 10:10 + keys:7, :, 3] = top / 8  # a seventh of the weights: within fp16 together
        v[:, 400:400 + keys:7, 0, 9] = -top / 8
        v[:, 100, :, 11] = top
        v[:, 300, :, 11] = -top
        (kc, ks), (vc, vs) = (c8.empty(most, page, Hkv, D, kind, dev) for _ in "kv")
        cache.cache_append(k.to(dtype), v.to(dtype), kc, vc, table[:1], n[:1], ks, vs)
        rows = [c8.values(c.flatten(0, 1)[:L], raw(s).transpose(1, 2).flatten(0, 1)[:L])[None].expand(B, -1, -1, -1)
                for c, s in ((kc, ks), (vc, vs))]
        assert rows[0].abs().max() > 65520 and rows[1].abs().max() > 65520
        o, p, (_, _, vh) = ref.attention(q, *rows, seen(n, L), D ** -0.5)
        assert o.abs().max() < 65000
        apart = paged.paged_attn(q, kc, vc, table, n, k_scale=ks, v_scale=vs)
        ref.close(apart, o, c8.forward_bound(o, p, vh, FP), "not shared")
        for shared in (L, 333):
            got = paged.paged_attn(q, kc, vc, table, n, shared=shared, k_scale=ks, v_scale=vs)
            ref.close(got, o, bound(kind, o, p, vh, FP, B * (H // Hkv), D), f"{dtype}, {shared} shared")


# ----------------------------------------------------------------- codes of nothing
@CODES
def test_rows_of_next_to_nothing_are_codes_of_zero(rope, cache, dev, kind):
    """Byte 0 goes with codes 0, whatever the signs of the values were."""
    x = -torch.full((1, 3, 1, 32), 2.0 ** -112, device=dev)
    x[0, 1] = -0.0
    x[0, 2, 0, 1::2] *= -1
    table, n = torch.zeros(1, 1, dtype=torch.int32, device=dev), ints([3], dev)
    for write in (lambda *c: cache.cache_append(x, x, c[0], c[2], table, n, c[1], c[3]),
                  lambda *c: rope.qk_norm_rope_append(x, x * 0, x, c[0], c[2], table, n, k_scale=c[1], v_scale=c[3])):
        (kc, ks), (vc, vs) = (c8.empty(1, 8, 1, 32, kind, dev) for _ in "kv")
        write(kc, ks, vc, vs)
        for codes, byte in ((kc, ks), (vc, vs)):
            assert (raw(codes)[0, :3] == 0).all() and (raw(byte)[0, 0, :3] == 0).all()


def test_append_without_pages_anywhere(rope, cache, dev):
    """A cache without pages and tables without columns: q', and nothing is written."""
    (kc, ks), (vc, vs) = (c8.empty(0, 16, 2, 64, I8, dev) for _ in "kv")
    y = randn((2, 1, 2, 64), 1, dev)
    t, n = torch.zeros(2, 0, dtype=torch.int32, device=dev), ints([5, 0], dev)
    got = rope.qk_norm_rope_append(y, y, y, kc, vc, t, n, k_scale=ks, v_scale=vs)
    same = [torch.zeros(0, 16, 2, 64, dtype=BF, device=dev) for _ in "kv"]
    assert torch.equal(got, rope.qk_norm_rope_append(y, y, y, *same, t, n))
    cache.cache_append(y, y, kc, vc, t, n, ks, vs)


# --------------------------------------- runs that are shorter than the shared keys said
@KINDS
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("shared", [1, 64, 500, 5000, 2 ** 40])
@pytest.mark.parametrize("groups,lengths", [
    (1, [33, 640, 1, 0, 500, 64]), (2, [33, 600, 640, 0, 0, -4]), (2, [0, 0, 0, 500, 4200, 64]), (3, [1, 0, 9000, 8999, 0, 63]),
], ids=["one", "idle behind", "idle before", "three"])
def test_tiles_of_shorter_runs(paged, dev, kind, D, shared, groups, lengths):
    """More than 64 columns: the longest of a run is not the first, a run is idle beside a live one,
    `shared` is more than any sequence holds, so that parts leave and page ids are found again."""
    B, H, Hkv, page, L = len(lengths), 128, 2, 16, max(lengths)
    per = B // groups
    if per * (H // Hkv) <= 64:
        pytest.fail("no tiles")
    k, v = (randn((groups, L, Hkv, D), s, dev, F32) for s in (1, 2))
    at = [b // per for b in range(B)]
    k, v = k.repeat_interleave(per, 0), v.repeat_interleave(per, 0)
    pages = Pages(k, v, [a * per for a in at], page, kind, BF)
    n, q = ints(lengths, dev), randn((B, 1, H, D), 3, dev)
    got = pages.attn(paged, q, n, shared=shared, groups=groups)
    on = seen(n, L)
    o, p, (_, _, vh) = ref.attention(q, *pages.rows, on, D ** -0.5)
    ref.close(got, o, bound(kind, o, p, vh, BF, per * (H // Hkv), D), "o")
    assert (got[n <= 0] == 0).all()
    assert torch.equal(pages.attn(paged, q, n, shared=shared, groups=groups), got), "the same bits again"


@KINDS
@pytest.mark.parametrize("H,Hkv,D", [(2, 1, 128), (20, 2, 64), (64, 2, 64), (64, 2, 128), (64, 2, 80)])
def test_idle_slots_beside_poison(paged, dev, kind, H, Hkv, D):
    """NaN in the shared values reaches those that see them, not the idle slots beside them."""
    k, v = (randn((1, 320, Hkv, D), s, dev, F32).repeat(5, 1, 1, 1) for s in (1, 2))
    v[:, 53] = float("nan")
    pages = Pages(k, v, [0] * 5, 16, kind, BF)
    got = pages.attn(paged, randn((5, 1, H, D), 3, dev), ints([320, 0, 300, 0, 0], dev), shared=290)
    assert got[[0, 2]].isnan().all() and (got[[1, 3, 4]] == 0).all()


# ------------------------------------------------------------- bounds, sizes, places
@CODES
@pytest.mark.parametrize("per,prefix,rest,page,H,Hkv,D,dtype", [
    (6, 700, 40, 16, 9, 3, 128, BF), (8, 4100, 30, 64, 24, 8, 128, BF), (16, 777, 10, 16, 16, 4, 64, FP), (32, 333, 60, 8, 8, 4, 64, BF),
    (60, 513, 17, 64, 1, 1, 128, FP), (7, 300, 20, 16, 10, 2, 16, BF), (20, 300, 20, 16, 10, 5, 48, FP), (70, 100, 9, 8, 4, 4, 32, BF),
])
def test_few_columns_keep_two_parts(paged, dev, kind, per, prefix, rest, page, H, Hkv, D, dtype):
    """Up to 64 columns, or of other head dims, P is kept in two parts over codes: the bound of that."""
    L = prefix + rest
    k, v = (randn((1, L, Hkv, D), s, dev, F32).repeat(per, 1, 1, 1) for s in (1, 2))
    pages = Pages(k, v, [0] * per, page, kind, dtype)
    q, n = randn((per, 1, H, D), 3, dev, dtype, 2.0), ints([L - b % rest for b in range(per)], dev)
    o, p, (_, _, vh) = ref.attention(q, *pages.rows, seen(n, L), D ** -0.5)
    ref.close(pages.attn(paged, q, n, shared=prefix), o, c8.forward_bound(o, p, vh, dtype), "o")


@KINDS
@pytest.mark.parametrize("B,groups,shared,H,Hkv,D", [
    (6, 1, 0, 8, 2, 128), (40, 1, 0, 16, 4, 64), (8, 1, 1000, 24, 8, 128), (32, 4, 700, 16, 4, 64), (60, 1, 900, 24, 8, 128),
    (30, 1, 900, 24, 8, 96),
])
def test_wide_tables(paged, dev, kind, B, groups, shared, H, Hkv, D):
    """Tables far wider than any sequence is long: many parts, most of them without keys."""
    page, L = 16, 1200
    per = B // groups
    at = [b // per * per for b in range(B)]
    k, v = (randn((B, L, Hkv, D), s, dev, F32) for s in (1, 2))
    for x in (k, v):
        x[:, :shared] = x[at, :shared]
    pages = Pages(k, v, range(B), page, kind, BF, wide=2000 // B * 8)
    n = ints([L - 13 * (b % 10) for b in range(B)], dev)
    pages.table[:, -(-L // page):] = -7
    q = randn((B, 1, H, D), 3, dev)
    o, p, (_, _, vh) = ref.attention(q, *pages.rows, seen(n, L), D ** -0.5)
    ref.close(pages.attn(paged, q, n, shared=shared, groups=groups), o, bound(kind, o, p, vh, BF, per * (H // Hkv), D), "o")


@KINDS
@pytest.mark.parametrize("far", ["pages", "slots"])
@pytest.mark.parametrize("B", [2, 20, 40])  # 4, 40 and 80 columns
def test_strides_beyond_32_bits(paged, dev, kind, far, B):
    """Pages 2^32 bytes apart, and slots 2^28 apart, as a view into a larger cache has them."""
    H, Hkv, D, page, pages = 4, 2, 64, 8, 3
    dtype = BF if kind is None else kind
    size = 2 if kind is None else 1
    strides = ((1 << 32) // size, Hkv * D, D, 1) if far == "pages" else ((1 << 31) // size, (1 << 28) // size, D, 1)
    extent = sum((a - 1) * b for a, b in zip((pages, page, Hkv, D), strides)) + 1
    k, v = (randn((1, pages * page, Hkv, D), s, dev, F32) for s in (1, 2))
    held, scales, rows = [], {}, []
    for name, x in (("k", k), ("v", v)):
        view = torch.empty(extent, dtype=dtype, device=dev).as_strided((pages, page, Hkv, D), strides)
        if kind is None:
            view.copy_(x.view(pages, page, Hkv, D))
            x = x.to(dtype).double()
        else:
            c, e = c8.encode(x, kind)
            raw(view).copy_(raw(c).view(pages, page, Hkv, D))
            scales[f"{name}_scale"] = e.view(pages, page, Hkv).transpose(1, 2).contiguous().view(c8.E8)
            x = c8.values(c, e)
        held.append(view)
        rows.append(x.expand(B, -1, -1, -1))
    table = torch.arange(pages, dtype=torch.int32, device=dev)[None].repeat(B, 1)
    n = ints([24 - b % 5 for b in range(B)], dev)
    q = randn((B, 1, H, D), 3, dev)
    o, p, (_, _, vh) = ref.attention(q, *rows, seen(n, 24), D ** -0.5)
    for shared in (0, 17):
        print("[far]", kind, far, B, shared, flush=True)
        got = paged.paged_attn(q, *held, table, n, shared=shared, **scales)
        ref.close(got, o, bound(kind, o, p, vh, BF, B * 2, D), "o")


@KINDS
def test_tiles_captured_and_replayed(paged, dev, kind):
    """A captured call over tiles, replayed on other lengths, queries and tables with eager work between the
    replays: the eager bits every time."""
    B, H, Hkv, D, page, L, shared = 24, 24, 8, 128, 16, 800, 600
    k, v = (randn((1, L, Hkv, D), s, dev, F32).repeat(B, 1, 1, 1) for s in (1, 2))
    pages = Pages(k, v, [0] * B, page, kind, FP)
    q, n = randn((B, 1, H, D), 3, dev, FP), ints([L - b for b in range(B)], dev)
    pages.attn(paged, q, n, shared=shared)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = pages.attn(paged, q, n, shared=shared)
    for i in range(4):
        q.copy_(randn(tuple(q.shape), 10 + i, dev, FP))
        n.copy_(ints([max(0, L - 30 * i * (b % 24) - b) for b in range(B)], dev))
        pages.table.copy_(pages.table.roll(1, 1))
        g.replay()
        torch.cuda.synchronize()
        first = out.clone()
        assert torch.isfinite(first).all() and torch.equal(pages.attn(paged, q, n, shared=shared), first)


@KINDS
@pytest.mark.parametrize("B,H,Hkv,D,page,lengths", [
    (64, 8, 8, 128, 16, "ragged 3000"), (64, 8, 8, 128, 64, "equal 2500"), (64, 16, 8, 128, 16, "one 3000"), (64, 8, 8, 128, 16, "ragged 1000"),
    (256, 4, 4, 128, 16, "ragged 1400"), (5, 32, 32, 128, 64, "ragged 7000"), (130, 8, 8, 64, 8, "ragged 2500"),
])
def test_longest_first(paged, dev, kind, B, H, Hkv, D, page, lengths):
    """Batches whose workgroups go by length, and those that do not: few keys, sequences of one length; idle
    slots, lengths past the table and below 0 among them."""
    how, L = lengths.split()
    L = int(L)
    g = torch.Generator().manual_seed(B)
    n = {"ragged": torch.randint(0, L, (B,), generator=g), "equal": torch.full((B,), L), "one": torch.full((B,), 5)}[how].int()
    n[B // 3] = L
    if how == "ragged":
        n[1], n[B - 1] = 0, -9
    want = n.clamp(0, L)
    if how == "ragged":
        n[B // 3] = 2 ** 31 - 1
    k, v = (randn((1, L, Hkv, D), s, dev, F32).expand(B, -1, -1, -1).clone() for s in (1, 2))
    k *= 1 + torch.arange(B, device=dev)[:, None, None, None] % 5 / 4
    v += torch.arange(B, device=dev)[:, None, None, None] % 7 - 3
    most = -(-L // page)
    want = torch.where(n > L, torch.tensor(most * page), want).to(dev)
    k, v = (torch.nn.functional.pad(x, (0, 0, 0, 0, 0, most * page - L)) for x in (k, v))
    pages = Pages(k, v, range(B), page, kind, BF)
    q = randn((B, 1, H, D), 3, dev)
    got = pages.attn(paged, q, n.to(dev))
    on = seen(want, most * page)
    for b0 in range(0, B, 16):
        s = slice(b0, b0 + 16)
        o, p, (_, _, vh) = ref.attention(q[s], *(x[s] for x in pages.rows), on[s], D ** -0.5)
        ref.close(got[s], o, bound(kind, o, p, vh, BF, 1, D), "o")
    assert (got[want == 0] == 0).all()
