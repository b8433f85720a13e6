"""The operators around attention on the GPU, against float64: norms with rotation
(forward, gradients, the form that fills a paged cache), sliding-window attention
with sinks (forward and gradients) and attention of one token over pages. Bounds
are those of tests/_operators.py."""

import importlib

import pytest
import torch

import _operators as ref

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def rope(pkg):
    return importlib.import_module(f"{pkg.__name__}._qk_rope")


@pytest.fixture(scope="module")
def window(pkg):
    return importlib.import_module(f"{pkg.__name__}._window")


@pytest.fixture(scope="module")
def paged(pkg):
    return importlib.import_module(f"{pkg.__name__}._paged")


def randn(shape, seed, dev, dtype=BF, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(dev)


def tables(P, R, dev):
    if not R:
        return None, None
    f = 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    a = torch.arange(P, dtype=torch.float64)[:, None] * f
    return a.cos().float().to(dev), a.sin().float().to(dev)


# ------------------------------------------------------- norms and rotation
# B, T, H, Hkv, D, R, interleaved, dtype, weights, positions
ROPE = [
    (1, 1, 1, 1, 128, 128, False, BF, True, None),
    (2, 5, 3, 1, 128, 128, True, FP, True, "shared"),
    (1, 333, 24, 8, 128, 64, False, BF, True, None),
    (3, 17, 16, 4, 64, 64, False, FP, True, "batch"),
    (1, 50, 5, 5, 64, 32, True, F32, True, None),
    (2, 9, 7, 7, 80, 80, True, BF, False, "batch"),
    (1, 40, 2, 1, 96, 48, False, F32, True, "shared"),
    (1, 70, 40, 40, 8, 0, False, BF, True, None),
    (4, 1, 33, 11, 120, 16, False, FP, False, "batch"),
    (1, 2000, 2, 2, 128, 128, True, BF, True, None),
]


def rope_case(c, dev, seed=0):
    B, T, H, Hkv, D, R, interleaved, dtype, weights, positions = c
    P = T + 7
    q, k = randn((B, T, H, D), seed, dev, dtype, 2.0), randn((B, T, Hkv, D), seed + 1, dev, dtype, 0.5)
    qw = 1 + 0.2 * randn((D,), seed + 2, dev, F32) if weights else None
    kw = 1 + 0.2 * randn((D,), seed + 3, dev, F32) if weights else None
    cos, sin = tables(P, R, dev)
    g = torch.Generator().manual_seed(seed + 4)
    pos = None
    if positions:
        pos = torch.randint(0, P, (T,) if positions == "shared" else (B, T), generator=g).to(dev)
    at = torch.arange(T, device=dev).expand(B, T) if pos is None else pos.expand(B, T)
    return q, k, qw, kw, cos, sin, pos, at


def rope_bound(y, x, w, dtype):
    """One rounding of y; in fp32: the sum of squares and the root (at most 16
    roundings), two factors, two products and their sum, on values up to the row's
    largest."""
    top = y.abs().amax(-1, keepdim=True) * 2
    return (ref.half_step(dtype) * y.abs() + 32 * ref.U32 * top) * 1.01


@pytest.mark.parametrize("case", ROPE, ids=[str(i) for i in range(len(ROPE))])
def test_norm_rope(rope, dev, case):
    q, k, qw, kw, cos, sin, pos, at = rope_case(case, dev)
    print("[rope]", case, flush=True)
    qo, ko = rope.qk_norm_rope(q, k, qw, kw, cos, sin, eps=1e-5, positions=pos, interleaved=case[6])
    for got, x, w in ((qo, q, qw), (ko, k, kw)):
        want = ref.norm_rope(x, w, cos, sin, at, case[6], 1e-5)
        assert got.dtype == x.dtype and got.is_contiguous()
        ref.close(got, want, rope_bound(want, x, w, case[7]), "row")


@pytest.mark.parametrize("case", ROPE, ids=[str(i) for i in range(len(ROPE))])
def test_norm_rope_gradients(rope, dev, case):
    """Against the formula in float64 (autograd of the float64 form) and, in the
    same form, against differences along a direction."""
    q, k, qw, kw, cos, sin, pos, at = rope_case(case, dev, seed=20)
    leaves = [t for t in (q, k, qw, kw) if t is not None]
    for t in leaves:
        t.requires_grad_(True)
    print("[rope grad]", case, flush=True)
    dqo, dko = randn(q.shape, 31, dev, case[7]), randn(k.shape, 32, dev, case[7])
    out = rope.qk_norm_rope(q, k, qw, kw, cos, sin, eps=1e-5, positions=pos, interleaved=case[6])
    got = torch.autograd.grad(out, leaves, (dqo, dko))
    wide = [t.detach().double().requires_grad_(True) for t in leaves]
    full = wide if qw is not None else [*wide, None, None]

    def loss(x):
        y = [ref.norm_rope(x[i], x[i + 2], cos, sin, at, case[6], 1e-5) for i in (0, 1)]
        return (y[0] * dqo.double()).sum() + (y[1] * dko.double()).sum()

    want = torch.autograd.grad(loss(full), wide)
    u = ref.half_step(case[7])
    for g, w, x, dy in zip(got[:2], want[:2], (q, k), (dqo, dko)):
        # fp32 before the one rounding: values up to the row's largest |r u| (r up to its inverse norm)
        r = 1 / (x.detach().double().pow(2).mean(-1, keepdim=True) + 1e-5).sqrt()
        scale = r * dy.double().abs().amax(-1, keepdim=True) * 3 * (1 + x.detach().double().abs() * r)
        assert g.dtype == x.dtype
        ref.close(g, w, (u * w.abs() + 64 * ref.U32 * scale) * 1.01, "dx")
    for i, x, dy in ((2, q, dqo), (3, k, dko)):
        if qw is None:
            continue
        xd = x.detach().double()
        r = 1 / (xd.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt()
        terms = (dy.double().abs().amax(-1, keepdim=True) * 1.5 * (xd * r).abs()).sum((0, 1, 2))
        # at most 128 additions behind one another, and 32 roundings inside a term
        ref.close(got[i], want[i], 160 * ref.U32 * terms + 1e-30, "dw")
    d = [randn(t.shape, 40 + i, dev, F32).double() for i, t in enumerate(wide)]
    with torch.no_grad():
        h = 1e-6
        step = [[t + s * h * x for t, x in zip(wide, d)] for s in (1, -1)]
        step = [x if qw is not None else [*x, None, None] for x in step]
        slope = (loss(step[0]) - loss(step[1])) / (2 * h)
        along = sum((g.double() * x).sum() for g, x in zip(got, d))
        size = sum((g.double() * x).pow(2).sum() for g, x in zip(got, d)).sqrt()
    # the type's roundings are independent: a sum of n of them is off by about u sqrt(sum squares)
    assert (slope - along).abs() <= 8 * u * size + 1e-5 * size + 1e-6, (slope, along)


def test_norm_rope_strides_and_types(rope, dev):
    """Views of one projection, a batch expanded from one sequence, weights of another
    type, rows that are not 16-byte aligned and shifted tables."""
    B, T, H, D = 2, 19, 4, 64
    qkv = randn((B, T, 3, H, D), 1, dev)
    q, k = qkv[:, :, 0], qkv[:, :, 1]
    w = (1 + 0.1 * randn((D + 1,), 2, dev, F32))[1:]
    cos, sin = tables(T, D, dev)
    want = rope.qk_norm_rope(q.contiguous(), k.contiguous(), w.clone(), w.clone(), cos, sin)
    for got, x in zip(rope.qk_norm_rope(q, k, w, w, cos, sin), want):
        assert torch.equal(got, x)
    odd = torch.empty(B * T * H * D + 1, device=dev, dtype=BF)[1:].view(B, T, H, D).copy_(q)
    assert torch.equal(rope.qk_norm_rope(odd, k, w, w, cos, sin)[0], want[0])
    one = q[:1].expand(3, T, H, D)
    got = rope.qk_norm_rope(one, one, w, w, cos, sin)[0]
    assert torch.equal(got, want[0][:1].expand_as(got))
    got = rope.qk_norm_rope(q, k, w.to(BF), None, cos, sin)
    assert torch.equal(got[0], rope.qk_norm_rope(q, k, w.to(BF).float(), None, cos, sin)[0])
    pos = torch.tensor([5, -3, 10 ** 6], device=dev)
    got = rope.qk_norm_rope(q[:, :3], k[:, :3], w, w, cos, sin, positions=pos)  # clamped to the table
    pos = torch.tensor([5, 0, T - 1], device=dev)
    assert torch.equal(got[0], rope.qk_norm_rope(q[:, :3], k[:, :3], w, w, cos, sin, positions=pos)[0])
    empty = rope.qk_norm_rope(q[:, :0], k[:, :0], w, w, cos, sin)
    assert empty[0].shape == (B, 0, H, D)


def cache_of(B, max_len, page, Hkv, D, dev, dtype=BF, seed=7, fill=float("nan")):
    """An empty cache of NaN, its pages dealt at random, one page more than used."""
    most = -(-max_len // page)
    n = B * most + 1
    g = torch.Generator().manual_seed(seed)
    table = (torch.randperm(n, generator=g)[:B * most]).to(torch.int32).reshape(B, most).to(dev)
    shape = (n, page, Hkv, D)
    return torch.full(shape, fill, device=dev, dtype=dtype), torch.full(shape, fill, device=dev, dtype=dtype), table


@pytest.mark.parametrize("B,T,H,Hkv,D,page,lengths,dtype", [
    (1, 1, 24, 8, 128, 64, [1], BF), (3, 1, 4, 4, 64, 16, [17, 0, 64], FP), (2, 70, 6, 2, 96, 32, [70, 95], BF),
    (2, 5, 2, 1, 128, 8, [3, 40], F32),
])
def test_append(rope, dev, B, T, H, Hkv, D, page, lengths, dtype):
    """Rows land at their places, turned by their positions; every other slot, an
    idle sequence's and those of tokens before position 0 among them, stays."""
    q, k, v = (randn((B, T, h, D), s, dev, dtype) for h, s in ((H, 1), (Hkv, 2), (Hkv, 3)))
    kc, vc, table = cache_of(B, 100, page, Hkv, D, dev, dtype, fill=3.0)
    n = torch.tensor(lengths, dtype=torch.int32, device=dev)
    cos, sin = tables(100, 16 * (D // 16), dev)
    w = 1 + 0.2 * randn((D,), 4, dev, F32)
    kc0, vc0 = kc.clone(), vc.clone()
    print("[append]", B, T, H, Hkv, D, page, lengths, dtype, flush=True)
    qo = rope.qk_norm_rope_append(q, k, v, kc, vc, table, n, w, w, cos, sin)
    at = n[:, None] - T + torch.arange(T, device=dev)
    want_q, want_k = rope.qk_norm_rope(q, k, w, w, cos, sin, positions=at)
    for b in range(B):
        for t in range(T):
            p = int(at[b, t])
            if p < 0:
                continue
            page_id = int(table[b, p // page])
            assert torch.equal(qo[b, t], want_q[b, t])
            assert torch.equal(kc[page_id, p % page], want_k[b, t])
            assert torch.equal(vc[page_id, p % page], v[b, t])
            kc0[page_id, p % page], vc0[page_id, p % page] = kc[page_id, p % page], vc[page_id, p % page]
    assert torch.equal(kc, kc0) and torch.equal(vc, vc0)


def test_append_bad_pages(rope, dev):
    """Page ids outside the cache and tokens past the table write nothing."""
    q, k, v = (randn((3, 1, 2, 64), s, dev) for s in (1, 2, 3))
    kc, vc, _ = cache_of(3, 16, 8, 2, 64, dev, fill=3.0)
    table = torch.tensor([[-1, 0], [kc.shape[0], 0], [0, 0]], dtype=torch.int32, device=dev)
    n = torch.tensor([3, 4, 17], dtype=torch.int32, device=dev)
    rope.qk_norm_rope_append(q, k, v, kc, vc, table, n)
    assert (kc == 3).all() and (vc == 3).all()
    none = kc[:0]
    assert rope.qk_norm_rope_append(q, k, v, none, none, table, n).shape == q.shape


# ------------------------------------------------------------------- windows
# B, Tq, Tk, H, Hkv, D, window, sinks, causal, lengths, dtype
WINDOW = [
    (1, 1, 1, 1, 1, 128, 1, 0, True, None, BF),
    (1, 1, 700, 6, 2, 128, 300, 4, True, None, BF),
    (2, 1, 65, 4, 4, 64, 9, 70, True, [65, 30], FP),
    (1, 63, 63, 2, 1, 64, 7, 2, True, None, BF),
    (1, 130, 130, 2, 2, 128, None, 0, True, None, FP),
    (2, 200, 200, 4, 2, 128, 50, 3, True, [200, 77], BF),
    (1, 257, 1000, 3, 1, 64, 300, 130, True, None, BF),
    (2, 300, 300, 2, 2, 128, 40, 0, False, [0, 261], FP),
    (1, 400, 400, 2, 1, 128, 65, 333, False, None, BF),
    (1, 190, 500, 2, 2, 64, 1, 1, False, None, FP),
    (1, 500, 500, 16, 2, 64, 128, 64, True, None, BF),
    (3, 129, 129, 1, 1, 80, 64, 5, True, [129, 1, 64], BF),
    (1, 70, 90, 3, 3, 24, 33, 2, False, None, FP),
    (1, 1100, 1100, 2, 1, 128, 256, 4, True, None, FP),
    (1, 640, 640, 1, 1, 128, None, 0, False, None, BF),
    # key tiles of the forward cut into parts; blocks of keys of the backward cut into parts
    (1, 100, 3000, 2, 1, 128, None, 0, True, None, BF),
    (2, 70, 2500, 4, 2, 64, 2000, 100, True, [2500, 2460], FP),
    (1, 1100, 1100, 4, 1, 64, None, 0, True, None, BF),
    (1, 900, 900, 2, 2, 128, 100, 300, False, None, BF),
    (1, 1000, 1300, 2, 1, 128, 700, 1, True, None, FP),
]


def window_case(c, dev, seed=0):
    B, Tq, Tk, H, Hkv, D, w, sinks, causal, lengths, dtype = c
    q = randn((B, Tq, H, D), seed, dev, dtype, 2.0)
    k, v = randn((B, Tk, Hkv, D), seed + 1, dev, dtype), randn((B, Tk, Hkv, D), seed + 2, dev, dtype)
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=dev)
    if n is not None:  # what lies behind a sequence may be anything
        for b, e in enumerate(lengths):
            k[b, e:], v[b, e:] = float("nan"), float("inf")
            q[b, max(0, e - (Tk - Tq)):] = float("nan")
    on = ref.seen(Tq, Tk, Tk - Tq, w, sinks, causal, n, B, dev)
    return q, k, v, n, on, dict(window=w, sinks=sinks, causal=causal, lengths=n)


@pytest.mark.parametrize("case", WINDOW, ids=[str(i) for i in range(len(WINDOW))])
def test_window(window, dev, case):
    q, k, v, n, on, kw = window_case(case, dev)
    print("[window]", case, flush=True)
    got = window.window_attn(q, k, v, **kw)
    o, p, (_, _, vh) = ref.attention(q, k, v, on, q.shape[-1] ** -0.5)
    ref.close(got, o, ref.forward_bound(o, p, vh, q.dtype), "o")
    assert (got.masked_select(~on.any(2)[:, :, None, None].expand_as(got)) == 0).all()


@pytest.mark.parametrize("case", WINDOW, ids=[str(i) for i in range(len(WINDOW))])
def test_window_gradients(window, dev, case):
    q, k, v, n, on, kw = window_case(case, dev, seed=50)
    do = randn(q.shape, 60, dev, q.dtype)
    if n is not None:
        do.masked_fill_(~on.any(2)[:, :, None, None], float("nan"))  # gradients of rows that nothing reads
    for t in (q, k, v):
        t.requires_grad_(True)
    print("[window grad]", case, flush=True)
    out = window.window_attn(q, k, v, scale=0.11, **kw)
    got = torch.autograd.grad(out, (q, k, v), do)
    want, bound = ref.gradients(q.detach(), k.detach(), v.detach(), on, 0.11, do, q.dtype)
    for name, g, w, b in zip(("dq", "dk", "dv"), got, want, bound):
        ref.close(g, w, b, name)
    again = torch.autograd.grad(window.window_attn(q, k, v, scale=0.11, **kw), (q, k, v), do)
    for x, y in zip(got, again):
        assert torch.equal(x, y)


# As WINDOW, windows and sequences whose gradients round P and dS once.
LONG = [
    (2, 1300, 1300, 4, 2, 64, 400, 30, False, [1300, 700], FP),
    (2, 1500, 1500, 4, 2, 128, 600, 4, True, [1500, 1], BF),
    (1, 1029, 2051, 6, 1, 64, 900, 200, True, None, BF),
    (1, 1111, 1111, 2, 2, 128, 300, 513, False, None, FP),
    (2, 128, 1024, 3, 3, 96, 511, 1, True, [1024, 960], BF),
]


@pytest.mark.parametrize("case", LONG, ids=[str(i) for i in range(len(LONG))])
def test_window_long(window, dev, case):
    test_window(window, dev, case)
    test_window_gradients(window, dev, case)


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp16"])
@pytest.mark.parametrize("D,T,w,sinks,causal", [(64, 700, 22, 1, False), (128, 900, 36, 4, True), (80, 300, 250, 0, True)])
def test_window_gradients_of_few_keys(window, dev, D, T, w, sinks, causal, dtype):
    """Where rows see few keys, P and dS keep what their rounding takes away: what is left
    is D_i (its o in two roundings), fp32 sums and the outputs' own rounding, whose error
    alone is 1 here. Independent errors add up in squares: 1.25 leaves 0.75 of it for
    the others; one rounding of dS as large as the outputs' would give 1.41 or more."""
    c = (1, T, T, 4, 2, D, w, sinks, causal, None, dtype)
    q, k, v, n, on, kw = window_case(c, dev, seed=120)
    do = randn(q.shape, 130, dev, dtype)
    for t in (q, k, v):
        t.requires_grad_(True)
    got = torch.autograd.grad(window.window_attn(q, k, v, scale=0.11, **kw), (q, k, v), do)
    want, _ = ref.gradients(q.detach(), k.detach(), v.detach(), on, 0.11, do, dtype)
    for name, g, x in zip(("dq", "dk", "dv"), got, want):
        ideal = (x.to(dtype).double() - x).norm()
        assert (g.double() - x).norm() <= 1.25 * ideal, (name, ((g.double() - x).norm() / ideal).item())


# As WINDOW, enough heads for the forward's workgroups of 128 rows.
MANY_HEADS = [
    (8, 257, 320, 48, 8, 64, 90, 70, True, [320, 0, 63, 64, 200, 319, 190, 256], BF),
    (4, 600, 600, 60, 20, 128, 200, 5, False, None, FP),
    (2, 1400, 1400, 52, 4, 64, 300, 130, True, None, FP),
    (16, 130, 500, 40, 8, 128, None, 0, True, [500] * 15 + [431], BF),
    (3, 500, 500, 96, 8, 64, 64, 200, False, [500, 301, 12], BF),
    (1, 1030, 1030, 128, 4, 128, 450, 64, True, None, BF),
]


@pytest.mark.parametrize("case", MANY_HEADS, ids=[str(i) for i in range(len(MANY_HEADS))])
def test_window_many_heads(window, dev, case):
    assert case[0] * case[3] * -(-case[1] // 128) >= 1024
    test_window(window, dev, case)
    test_window_gradients(window, dev, case)


def test_window_gradients_against_differences(window, dev):
    """Along a direction, the float64 form's differences against the kernels' gradients."""
    c = (1, 150, 150, 4, 2, 64, 60, 3, True, None, FP)
    q, k, v, n, on, kw = window_case(c, dev, seed=70)
    do = randn(q.shape, 80, dev, FP)
    for t in (q, k, v):
        t.requires_grad_(True)
    got = torch.autograd.grad(window.window_attn(q, k, v, **kw), (q, k, v), do)
    _, bound = ref.gradients(q.detach(), k.detach(), v.detach(), on, 0.125, do, FP)
    d = [randn(t.shape, 90 + i, dev, F32).double() for i, t in enumerate((q, k, v))]
    h = 1e-5

    def loss(s):
        x = [t.detach().double() + s * h * y for t, y in zip((q, k, v), d)]
        return (ref.attention(*x, on, 0.125)[0] * do.double()).sum()

    slope = (loss(1) - loss(-1)) / (2 * h)
    along = sum((g.double() * y).sum() for g, y in zip(got, d))
    room = sum((b * y.abs()).sum() for b, y in zip(bound, d))
    assert (slope - along).abs() <= room + 1e-4, (slope, along, room)
    size = sum((g.double() * y).pow(2).sum() for g, y in zip(got, d)).sqrt()
    assert (slope - along).abs() <= 0.02 * size, (slope, along, size)  # roundings of 2^-11 that average out


def test_window_strides(window, dev):
    """Interleaved views, BHTD storage, one sequence's keys for a whole batch, heads
    expanded from one, rows that are not aligned: the same bits as dense copies."""
    B, T, H, D = 2, 150, 4, 64
    qkv = randn((B, T, 3, H, D), 3, dev)
    q, k, v = qkv.unbind(2)
    kw = dict(window=40, sinks=2)
    want = window.window_attn(*(t.contiguous() for t in (q, k, v)), **kw)
    assert torch.equal(window.window_attn(q, k, v, **kw), want)
    bh = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    assert torch.equal(window.window_attn(*bh, **kw), want)
    odd = [torch.empty(t.numel() + 1, device=dev, dtype=BF)[1:].view(t.shape).copy_(t) for t in (q, k, v)]
    assert torch.equal(window.window_attn(*odd, **kw), want)
    k1, v1 = k[:1].expand_as(k), v[:1].expand_as(v)
    assert torch.equal(window.window_attn(q, k1, v1, **kw), window.window_attn(q, k1.contiguous(), v1.contiguous(), **kw))
    kh, vh = (t[:, :, :1].expand_as(t) for t in (k, v))
    got = window.window_attn(q, kh, vh, **kw)
    assert torch.equal(got, window.window_attn(q, k[:, :, :1], v[:, :, :1], **kw))
    # gradients of broadcast inputs: those of the copies, summed
    leaf = k[:1].detach().clone().requires_grad_(True)
    g, = torch.autograd.grad(window.window_attn(q, leaf.expand_as(k), v, **kw), leaf, want)
    dense = k[:1].expand_as(k).contiguous().requires_grad_(True)
    gd, = torch.autograd.grad(window.window_attn(q, dense, v, **kw), dense, want)
    assert torch.equal(g, gd.sum(0, keepdim=True))
    # an expanded gradient of the output
    leaf = q.detach().clone().requires_grad_(True)
    window.window_attn(leaf, k, v, **kw).sum().backward()
    ones = q.detach().clone().requires_grad_(True)
    window.window_attn(ones, k, v, **kw).backward(torch.ones_like(q))
    assert torch.equal(leaf.grad, ones.grad)


def test_window_unread_keys(window, dev):
    """Keys that no row of a call sees are not read: those past the last row (a
    buffer longer than the sequence) and those that slid out of every window."""
    B, T, H, D = 1, 90, 2, 128
    q, k, v = (randn((B, s, H, D), i, dev) for i, s in enumerate((T, 600, 600)))
    kw = dict(window=20, sinks=3)
    clean = window.window_attn(q, k, v, q_start=300, **kw)
    bad = torch.ones(600, dtype=torch.bool, device=dev)
    bad[:3] = False
    bad[300 - 19:300 + T] = False
    for x in (float("nan"), float("inf"), torch.finfo(BF).min):
        k2, v2 = k.clone(), v.clone()
        k2[:, bad], v2[:, bad] = x, x
        assert torch.equal(window.window_attn(q, k2, v2, q_start=300, **kw), clean)
        one = window.window_attn(q[:, :1], k2, v2, q_start=300, **kw)
        assert torch.isfinite(one).all()
    # a key's own values reach the rows that see it only, also in k's case within a block
    k2 = k.clone()
    k2[:, 320] = float("nan")
    got = window.window_attn(q, k2, v, q_start=300, **kw)
    rows = torch.arange(T, device=dev) + 300
    hit = (rows >= 320) & (rows < 340)
    assert torch.isnan(got[:, hit]).all() and torch.equal(got[:, ~hit], clean[:, ~hit])


def test_window_empty(window, dev):
    q = torch.zeros((2, 0, 2, 64), device=dev, dtype=BF, requires_grad=True)
    k = torch.zeros((2, 5, 2, 64), device=dev, dtype=BF, requires_grad=True)
    out = window.window_attn(q, k, k, window=3)
    assert out.shape == q.shape
    gq, gk = torch.autograd.grad(out.sum(), (q, k))
    assert gq.shape == q.shape and (gk == 0).all()


def test_window_some_gradients(window, dev):
    """Leaves that need none get none, the others the same bits; once only."""
    q, k, v, _, _, kw = window_case((1, 90, 90, 2, 1, 64, 30, 2, True, None, BF), dev)
    do = randn(q.shape, 9, dev)
    every = [t.clone().requires_grad_(True) for t in (q, k, v)]
    want = torch.autograd.grad(window.window_attn(*every, **kw), every, do)
    for i in range(3):
        x = [t.clone().requires_grad_(j == i) for j, t in enumerate((q, k, v))]
        got, = torch.autograd.grad(window.window_attn(*x, **kw), x[i], do)
        assert torch.equal(got, want[i])
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(window.window_attn(*every, **kw), every, do, create_graph=True)
    with torch.no_grad():
        assert not window.window_attn(*every, **kw).requires_grad


def test_refusals(rope, window, paged, dev):
    """What the Python entries refuse before any launch."""
    x = torch.zeros(2, 8, 4, 64, device=dev, dtype=BF)
    n = torch.ones(2, dtype=torch.int32, device=dev)
    c = torch.zeros(3, 8, 4, 64, device=dev, dtype=BF)
    t = torch.zeros(2, 1, dtype=torch.int32, device=dev)
    cos = torch.zeros(8, 32, device=dev)

    def bad(match, f, *a, **kw):
        with pytest.raises(ValueError, match=match):
            f(*a, **kw)

    bad("dtype", rope.qk_norm_rope, x, x.half())
    bad("dtype", rope.qk_norm_rope, x.double(), x.double())
    bad("4 dimensions", rope.qk_norm_rope, x, x[0])
    bad("tokens", rope.qk_norm_rope, x, x[:, :3])
    bad("head_dim", rope.qk_norm_rope, x[..., :60], x[..., :60])
    bad("head_dim", rope.qk_norm_rope, x, x[..., :32])
    bad("q_weight", rope.qk_norm_rope, x, x, torch.ones(32, device=dev))
    bad("k_weight", rope.qk_norm_rope, x, x, None, torch.ones(64))
    bad("together", rope.qk_norm_rope, x, x, None, None, cos)
    bad("cos", rope.qk_norm_rope, x, x, None, None, cos.double(), cos.double())
    bad("rotated", rope.qk_norm_rope, x, x, None, None, cos[:, :12].contiguous(), cos[:, :12].contiguous())
    bad("table of 4", rope.qk_norm_rope, x, x, None, None, cos[:4], cos[:4])
    bad("positions", rope.qk_norm_rope, x, x, None, None, cos, cos, positions=cos[:, 0])
    bad("positions", rope.qk_norm_rope, x, x, None, None, cos, cos, positions=n)
    bad("fp32|float16|dtype", window.window_attn, x.float(), x.float(), x.float(), window=4)
    bad("shapes", window.window_attn, x, x, x[:, :4], window=4)
    bad("share", window.window_attn, x, x[:, :, :3], x[:, :, :3], window=4)
    bad("window", window.window_attn, x, x, x, window=0)
    bad("sinks", window.window_attn, x, x, x, window=4, sinks=-1)
    bad("scale", window.window_attn, x, x, x, window=4, scale=0.0)
    bad("rows", window.window_attn, x, x[:, :4], x[:, :4], window=4)
    bad("rows", window.window_attn, x, x, x, window=4, q_start=1)
    bad("lengths", window.window_attn, x, x, x, window=4, lengths=n.long())
    bad("lengths", window.window_attn, x, x, x, window=4, lengths=n[:1])
    bad("tokens", paged.paged_attn, x, c, c, t, n)
    q = x[:, :1]
    bad("page_table", paged.paged_attn, q, c, c, t[:1], n)
    bad("page_table", paged.paged_attn, q, c, c, t.long(), n)
    bad("lengths", paged.paged_attn, q, c, c, t, n.cpu())
    bad("multiple of 8", paged.paged_attn, q, c[:, :4], c[:, :4], t, n)
    bad("cache shapes", paged.paged_attn, q, c, c[:2], t, n)
    bad("contiguous", paged.paged_attn, q, c.transpose(1, 3).contiguous().transpose(1, 3), c, t, n)
    bad("gradient", paged.paged_attn, q.clone().requires_grad_(True), c, c, t, n)
    bad("gradient", rope.qk_norm_rope_append, q.clone().requires_grad_(True), q, q, c, c, t, n)
    bad("match", rope.qk_norm_rope_append, q, q[:, :, :2], q[:, :, :2], c, c, t, n)


def test_refusals_of_gradients_and_numbers(rope, window, paged, dev):
    """Tensors whose gradient would be lost, caches that cannot be written, sizes that are no numbers."""
    c = torch.zeros(3, 8, 4, 64, device=dev, dtype=BF)
    q = torch.zeros(2, 1, 4, 64, device=dev, dtype=BF)
    t = torch.zeros(2, 1, dtype=torch.int32, device=dev)
    n = torch.ones(2, dtype=torch.int32, device=dev)
    cos, w = torch.zeros(8, 32, device=dev), torch.ones(64, device=dev)
    leaf = lambda x: x.clone().requires_grad_(True)  # noqa: E731

    def bad(match, f, *a, **kw):
        with pytest.raises(ValueError, match=match):
            f(*a, **kw)

    bad("gradient", rope.qk_norm_rope, q, q, None, None, leaf(cos), cos)
    bad("gradient", rope.qk_norm_rope_append, q, q, q, c, c, t, n, leaf(w), w)
    bad("gradient", rope.qk_norm_rope_append, q, q, q, c, c, t, n, w, leaf(w))
    bad("gradient", rope.qk_norm_rope_append, q, q, q, c, leaf(c), t, n)
    bad("gradient", rope.qk_norm_rope_append, q, q, q, c, c, t, n, None, None, cos, leaf(cos))
    bad("expanded", rope.qk_norm_rope_append, q, q, q, c[:1].expand(3, 8, 4, 64), c, t, n)
    bad("expanded", rope.qk_norm_rope_append, q, q, q, c, c[:, :, :1].expand(3, 8, 4, 64), t, n)
    for eps in (-1e-6, float("nan"), float("inf")):
        bad("eps", rope.qk_norm_rope, q, q, eps=eps)
    for scale in (float("nan"), float("inf"), 1e300, 1e-300, -1.0):
        bad("scale", window.window_attn, q, q, q, window=4, scale=scale)
        bad("scale", paged.paged_attn, q, c, c, t, n, scale=scale)
    with torch.no_grad():  # nothing to lose
        rope.qk_norm_rope(q, q, None, None, leaf(cos), cos)
        rope.qk_norm_rope_append(q, q, q, c, leaf(c), t, n, leaf(w), leaf(w))


def test_append_is_a_change_of_the_cache(rope, window, dev):
    """A backward pass that kept the cache refuses to run on what an append made of it."""
    c = torch.randn(1, 16, 2, 64, device=dev, dtype=BF)
    x = torch.randn(1, 1, 2, 64, device=dev, dtype=BF)
    q = torch.randn(1, 16, 2, 64, device=dev, dtype=BF, requires_grad=True)
    t, n = torch.zeros(1, 1, dtype=torch.int32, device=dev), torch.full((1,), 16, dtype=torch.int32, device=dev)
    out = window.window_attn(q, c, c.clone(), window=4)
    rope.qk_norm_rope_append(x, x, x, c, c.clone(), t, n)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


@pytest.mark.parametrize("dim", [0, 1, 2])
def test_cache_orders(paged, dev, dim):
    """Pages, slots or heads outermost in memory: the cache is read where it lies."""
    c = [torch.randn(5, 16, 2, 64, device=dev, dtype=BF) for _ in "kv"]
    q = torch.randn(2, 1, 4, 64, device=dev, dtype=BF)
    t = torch.tensor([[4, 0], [2, 3]], dtype=torch.int32, device=dev)
    n = torch.tensor([31, 9], dtype=torch.int32, device=dev)
    there = [x.transpose(0, dim).contiguous().transpose(0, dim) for x in c]
    assert torch.equal(paged.paged_attn(q, *there, t, n), paged.paged_attn(q, *c, t, n))


# --------------------------------------------------------------------- pages
# lengths, page, H, Hkv, D, window, sinks, dtype
PAGED = [
    ([1], 16, 1, 1, 128, None, 0, BF),
    ([0, 7, 64], 8, 24, 8, 128, None, 0, BF),
    ([1000, 333, 31, 32, 33], 16, 16, 4, 64, None, 0, FP),
    ([5000], 64, 24, 8, 128, 700, 4, BF),
    ([130, 4097], 24, 40, 2, 128, 100, 33, FP),
    ([900, 20], 136, 3, 3, 96, 64, 0, BF),
    ([70], 32, 34, 1, 80, 33, 40, FP),
    ([300] * 9, 256, 8, 8, 24, None, 0, BF),
    ([20000], 64, 4, 4, 64, None, 0, BF),
]


@pytest.mark.parametrize("case", PAGED, ids=[str(i) for i in range(len(PAGED))])
def test_paged(paged, dev, case):
    lengths, page, H, Hkv, D, w, sinks, dtype = case
    B, L = len(lengths), max(lengths)
    k, v = randn((B, L, Hkv, D), 1, dev, dtype), randn((B, L, Hkv, D), 2, dev, dtype)
    q = randn((B, 1, H, D), 3, dev, dtype, 2.0)
    kc, vc, table = cache_of(B, L + page, page, Hkv, D, dev, dtype)  # slots not written stay NaN
    n = torch.tensor(lengths, dtype=torch.int32, device=dev)
    on = torch.zeros((B, 1, L), dtype=torch.bool, device=dev)
    for b, e in enumerate(lengths):
        for p in range(0, e, page):
            m = min(page, e - p)
            kc[table[b, p // page], :m], vc[table[b, p // page], :m] = k[b, p:p + m], v[b, p:p + m]
        table[b, -(-e // page):] = -1 if b % 2 else 10 ** 9
        on[b, 0, :e] = True
        if w:
            on[b, 0, min(sinks, e):max(0, e - w)] = False
    print("[paged]", case, flush=True)
    got = paged.paged_attn(q, kc, vc, table, n, window=w, sinks=sinks)
    o, p, (_, _, vh) = ref.attention(q, k, v, on, D ** -0.5)
    ref.close(got, o, ref.forward_bound(o, p, vh, dtype), "o")
    assert (got[n == 0] == 0).all()


@pytest.mark.parametrize("first", [0, 4096])
def test_paged_split_without_keys(paged, dev, first):
    """A split whose pages all are bad, the first or one in the middle, beside others."""
    page, Hkv, D, L = 64, 1, 64, 16384
    kc, vc = randn((L // page, page, Hkv, D), 1, dev), randn((L // page, page, Hkv, D), 2, dev)
    q = randn((1, 1, 2, D), 3, dev)
    table = torch.arange(L // page, dtype=torch.int32, device=dev)[None].clone()
    table[:, first // page:(first + 2048) // page] = -7
    n = torch.tensor([9000], dtype=torch.int32, device=dev)
    on = torch.arange(L, device=dev)[None, None] < 9000
    on[..., first:first + 2048] = False
    got = paged.paged_attn(q, kc, vc, table, n)
    o, p, (_, _, vh) = ref.attention(q, kc.view(1, L, Hkv, D), vc.view(1, L, Hkv, D), on, D ** -0.5)
    ref.close(got, o, ref.forward_bound(o, p, vh, BF), "o")


def test_paged_bad_pages_and_long_lengths(paged, dev):
    """Keys on page ids that the cache lacks are not visible; a length past the table
    is the table's; a cache without pages gives zeros."""
    B, page, Hkv, D = 2, 16, 2, 64
    kc, vc = randn((7, page, Hkv, D), 1, dev), randn((7, page, Hkv, D), 2, dev)
    q = randn((B, 1, 4, D), 3, dev)
    table = torch.tensor([[3, 99, 1], [0, -5, 2]], dtype=torch.int32, device=dev)
    n = torch.tensor([41, 48], dtype=torch.int32, device=dev)
    got = paged.paged_attn(q, kc, vc, table, n)
    k = torch.stack([torch.cat([kc[3], kc[1]]), torch.cat([kc[0], kc[2]])])
    v = torch.stack([torch.cat([vc[3], vc[1]]), torch.cat([vc[0], vc[2]])])
    on = torch.arange(32, device=dev)[None, None] < torch.tensor([25, 32], device=dev)[:, None, None]
    o, p, (_, _, vh) = ref.attention(q, k, v, on, D ** -0.5)
    ref.close(got, o, ref.forward_bound(o, p, vh, BF), "o")
    long = torch.tensor([41, 2 ** 31 - 1], dtype=torch.int32, device=dev)
    assert torch.equal(paged.paged_attn(q, kc, vc, table, long), got)
    neg = torch.tensor([-4, 48], dtype=torch.int32, device=dev)
    assert (paged.paged_attn(q, kc, vc, table, neg)[0] == 0).all()
    assert (paged.paged_attn(q, kc[:0], vc[:0], table, n) == 0).all()


def test_paged_cache_views(rope, paged, dev):
    """k and v side by side in one allocation, heads before slots, a table that is a
    view of a wider one: the same bits as dense ones."""
    B, H, Hkv, D, page = 3, 4, 2, 64, 16
    kv = randn((9, 2, page, Hkv, D), 1, dev)
    wide = torch.randint(0, 9, (B, 8), dtype=torch.int32, device=dev)
    table, n = wide[:, 2:6], torch.tensor([60, 1, 33], dtype=torch.int32, device=dev)
    q = randn((B, 1, H, D), 2, dev)
    k, v = kv[:, 0], kv[:, 1]
    want = paged.paged_attn(q, k.contiguous(), v.contiguous(), table.contiguous(), n)
    assert torch.equal(paged.paged_attn(q, k, v, table, n), want)
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v)]
    assert torch.equal(paged.paged_attn(q, *heads_first, table, n), want)
    every_other = torch.stack([table, table + 100], 2).flatten(1)[:, ::2]
    assert torch.equal(paged.paged_attn(q, k, v, every_other, n), want)
    kn, vn = randn((B, 1, Hkv, D), 3, dev), randn((B, 1, Hkv, D), 4, dev)
    dense = [t.clone(memory_format=torch.contiguous_format) for t in (k, v)]
    uniq = torch.arange(9, dtype=torch.int32, device=dev).reshape(B, 3)[:, :3]
    m = torch.tensor([48, 1, 17], dtype=torch.int32, device=dev)
    rope.qk_norm_rope_append(q, kn, vn, k, v, uniq, m)
    rope.qk_norm_rope_append(q, kn, vn, *dense, uniq, m)
    assert torch.equal(k, dense[0]) and torch.equal(v, dense[1])


# ------------------------------------------------------------------- together
@pytest.mark.parametrize("H,Hkv,D,w,sinks", [(6, 2, 128, 100, 4), (4, 4, 64, None, 0)])
def test_prompt_then_tokens(rope, window, paged, dev, H, Hkv, D, w, sinks):
    """A prompt and its next tokens as they are used: norms and rotation into the
    cache, windowed attention over the prompt, then token by token over the pages;
    the whole against one windowed call over all tokens."""
    B, T, new, page = 2, 150, 20, 16
    total = T + new
    x = randn((B, total, H + 2 * Hkv, D), 5, dev)
    q, k, v = x.split([H, Hkv, Hkv], 2)
    qw, kw = 1 + 0.1 * randn((D,), 6, dev, F32), 1 + 0.1 * randn((D,), 7, dev, F32)
    cos, sin = tables(total, D, dev)
    kc, vc, table = cache_of(B, total, page, Hkv, D, dev)
    rows = []

    def lengths(n):
        return torch.full((B,), n, dtype=torch.int32, device=dev)

    qp = rope.qk_norm_rope_append(q[:, :T], k[:, :T], v[:, :T], kc, vc, table, lengths(T), qw, kw, cos, sin)
    qr, kr = rope.qk_norm_rope(q, k, qw, kw, cos, sin)
    assert torch.equal(qp, qr[:, :T])
    rows.append(window.window_attn(qp, kr[:, :T], v[:, :T], window=w, sinks=sinks))
    for t in range(T, total):
        s = slice(t, t + 1)
        qt = rope.qk_norm_rope_append(q[:, s], k[:, s], v[:, s], kc, vc, table, lengths(t + 1), qw, kw, cos, sin)
        assert torch.equal(qt, qr[:, s])
        rows.append(paged.paged_attn(qt, kc, vc, table, lengths(t + 1), window=w, sinks=sinks))
        # the same token against the contiguous keys so far
        flat = window.window_attn(qt, kr[:, :t + 1], v[:, :t + 1], window=w, sinks=sinks)
        u = ref.half_step(BF)
        assert ((flat.double() - rows[-1].double()).abs() <= 4 * u * (flat.double().abs() + 1)).all()
    got = torch.cat(rows, 1)
    on = ref.seen(total, total, 0, w, sinks, True, None, B, dev)
    o, p, (_, _, vh) = ref.attention(qr, kr, v, on, D ** -0.5)
    ref.close(got, o, ref.forward_bound(o, p, vh, BF), "o")


def test_other_stream_and_graph(rope, window, paged, dev):
    """On a stream of its own, and captured once and replayed on new contents with
    eager work between the replays: the eager bits every time."""
    B, T, H, Hkv, D, page = 2, 200, 4, 2, 64, 16
    q, k, v = randn((B, T, H, D), 1, dev), randn((B, T, Hkv, D), 2, dev), randn((B, T, Hkv, D), 3, dev)
    w = 1 + 0.1 * randn((D,), 4, dev, F32)
    cos, sin = tables(T, D, dev)
    kc, vc, table = cache_of(B, T, page, Hkv, D, dev)
    n = torch.full((B,), T, dtype=torch.int32, device=dev)
    do = randn(q.shape, 5, dev)

    def step():
        qp = rope.qk_norm_rope_append(q, k, v, kc, vc, table, n, w, w, cos, sin)
        _, kr = rope.qk_norm_rope(q, k, w, w, cos, sin)
        o = window.window_attn(qp, kr, v, window=50, sinks=2)
        one = paged.paged_attn(qp[:, -1:], kc, vc, table, n, window=50, sinks=2)
        leaves = [t.detach().requires_grad_(True) for t in (qp, kr, v)]
        grads = torch.autograd.grad(window.window_attn(*leaves, window=50, sinks=2), leaves, do)
        return [qp, kr, o, one, *grads]

    eager = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip(got, eager):
        assert torch.equal(x, y)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # two graphs live at once
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for rep in range(3):
        print("[graph] replay", rep, flush=True)
        for i, t in enumerate((q, k, v, do)):
            t.copy_(randn(t.shape, 100 + 10 * rep + i, dev))
        torch.cuda.synchronize()
        for graph, out in graphs:
            kc.fill_(float("nan"))
            graph.replay()
            torch.cuda.synchronize()
            for x, y in zip(out, step()):
                assert torch.equal(x, y)


def test_offsets_beyond_32_bits(rope, window, paged, dev):
    """A cache, a key buffer and a token range of more than 2^31 values: what lies
    behind that is read and written where it is. (Nothing else in them is touched, so
    they stay uninitialised.)"""
    H, Hkv, D, page = 4, 4, 128, 64
    pages = 66000  # 2.16e9 values
    kc, vc = (torch.empty((pages, page, Hkv, D), device=dev, dtype=BF) for _ in range(2))
    ids = torch.tensor([[pages - 1, 3, pages - 2]], dtype=torch.int32, device=dev)
    q, k, v = (randn((1, 150, H, D), s, dev) for s in (1, 2, 3))
    n = torch.tensor([150], dtype=torch.int32, device=dev)
    qp = rope.qk_norm_rope_append(q, k, v, kc, vc, ids, n)
    kn = rope.qk_norm_rope(q, k)[1]
    small = [torch.stack([t[i] for i in ids[0].tolist()]) for t in (kc, vc)]
    assert torch.equal(small[0].flatten(0, 1)[:150], kn[0]) and torch.equal(small[1].flatten(0, 1)[:150], v[0])
    near = torch.arange(3, dtype=torch.int32, device=dev)[None]
    assert torch.equal(paged.paged_attn(qp[:, -1:], kc, vc, ids, n), paged.paged_attn(qp[:, -1:], *small, near, n))
    # the same memory as one long sequence, its rows at the far end
    kf, vf = kc.view(1, pages * page, Hkv, D), vc.view(1, pages * page, Hkv, D)
    T = kf.shape[1]
    kf[:, T - 200:], vf[:, T - 200:] = randn((1, 200, Hkv, D), 4, dev), randn((1, 200, Hkv, D), 5, dev)
    tail = kf[:, T - 200:].clone(), vf[:, T - 200:].clone()
    for rows in (1, 100):  # (tiles begin at other keys than in the tail alone, so not the same bits)
        far = window.window_attn(qp[:, :rows], kf, vf, window=90)
        on = ref.seen(rows, 200, 200 - rows, 90, 0, True, None, 1, dev)
        o, p, (_, _, vh) = ref.attention(qp[:, :rows], *tail, on, D ** -0.5)
        ref.close(far, o, ref.forward_bound(o, p, vh, BF), "far rows")
    x = kc.view(1, -1, 32, D)  # tokens of 32 heads
    x[:, -5:] = randn((1, 5, 32, D), 6, dev)
    at = torch.arange(x.shape[1], device=dev)
    cos, sin = tables(8, D, dev)
    got = rope.qk_norm_rope(x, x[:, :, :1], None, None, cos, sin, positions=at % 8)[0][:, -5:]
    assert torch.equal(got, rope.qk_norm_rope(x[:, -5:], x[:, -5:, :1], None, None, cos, sin, positions=(at % 8)[-5:])[0])


def test_training_keeps_no_memory(rope, window, dev):
    q, k, v = (randn((1, 300, 4, 64), s, dev).requires_grad_(True) for s in (1, 2, 3))
    cos, sin = tables(300, 64, dev)

    def step():
        qr, kr = rope.qk_norm_rope(q, k, None, None, cos, sin)
        window.window_attn(qr, kr, v, window=64).float().square().sum().backward()
        for t in (q, k, v):
            t.grad = None

    step()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    for _ in range(5):
        step()
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() == before


def test_two_streams_at_once(window, paged, dev):
    """Calls in flight on two streams, with workspaces of their own: the bits of the
    calls one after another."""
    sets = []
    for i in range(2):
        q, k, v, _, _, kw = window_case((1, 100, 3000, 2, 1, 128, None, 0, True, None, BF), dev, seed=10 * i)
        kc, vc = randn((40, 64, 2, 128), 90 + i, dev), randn((40, 64, 2, 128), 95 + i, dev)
        table = torch.randperm(40, generator=torch.Generator().manual_seed(i)).to(torch.int32).view(1, 40).to(dev)
        n = torch.tensor([2500 - 700 * i], dtype=torch.int32, device=dev)
        sets.append(lambda q=q, k=k, v=v, kw=kw, kc=kc, vc=vc, t=table, n=n: (
            window.window_attn(q, k, v, **kw), paged.paged_attn(q[:, :1], kc, vc, t, n)))
    want = [f() for f in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(4):
        for i, (f, s) in enumerate(zip(sets, streams)):
            with torch.cuda.stream(s):
                got[i].append(f())
    torch.cuda.synchronize()
    for w, runs in zip(want, got):
        for r in runs:
            assert all(torch.equal(a, b) for a, b in zip(r, w))


# fp16: T, D, window, sinks, causal, do's size and whether it varies from row to row, v's size
SMALL_FP16 = [
    (8192, 64, None, 0, False, 1e-2, False, 1.0),
    (8192, 128, None, 0, False, 1e-3, False, 1.0),
    (4096, 128, None, 0, False, 1e-5, False, 1.0),
    (4100, 64, 1500, 70, True, 1e-3, True, 0.01),
    (8192, 64, None, 0, False, 30.0, False, 1.0),
    (700, 128, 20, 4, True, 1e-3, False, 1.0),
]


@pytest.mark.parametrize("case", SMALL_FP16, ids=[str(i) for i in range(len(SMALL_FP16))])
def test_window_fp16_gradients_of_any_size(window, dev, case):
    """P and dS of many keys, and of small gradients of the output, lie below fp16's normal numbers
    (dS of 8192 keys and gradients of 1e-3: below its smallest one), and of large ones above its
    largest; the gradients do not show it. Independent errors add up in squares: the outputs' own
    rounding counts 1, that of P or dS as a normal number 1, everything else 0.75 of that (as above)."""
    T, D, w, sinks, causal, size, varies, vsize = case
    q, k, v = randn((1, T, 2, D), 140, dev, FP, 2.0), randn((1, T, 1, D), 141, dev, FP), randn((1, T, 1, D), 142, dev, FP, vsize)
    do = randn((1, T, 2, D), 143, dev, F32, size)
    if varies:  # rows 2^0 to 2^-9 as large
        do = do * 2.0 ** -(torch.arange(T, device=dev) % 10)[None, :, None, None]
    do = do.to(FP)
    on = ref.seen(T, T, 0, w, sinks, causal, None, 1, dev)
    for t in (q, k, v):
        t.requires_grad_(True)
    got = torch.autograd.grad(window.window_attn(q, k, v, window=w, sinks=sinks, causal=causal, scale=0.06), (q, k, v), do)
    want, _ = ref.gradients(q.detach(), k.detach(), v.detach(), on, 0.06, do, FP)
    worst = {}
    for name, g, x in zip(("dq", "dk", "dv"), got, want):
        ideal = (x.to(FP).double() - x).norm()
        worst[name] = ((g.double() - x).norm() / ideal).item()
    print("[fp16]", case, worst, flush=True)
    assert all(x <= 1.6 for x in worst.values()), worst


def test_window_fp16_gradients_beyond_ds(window, dev):
    """dS past fp16's largest number where dq, dk and dv are well inside it: few keys of small k,
    q and large do; a row with an infinite do takes its own keys' gradients with it and no others'."""
    T, D = 300, 64
    q, k = randn((1, T, 2, D), 150, dev, FP, 0.01), randn((1, T, 2, D), 151, dev, FP, 0.01)
    v, do = randn((1, T, 2, D), 152, dev, FP, 8.0), randn((1, T, 2, D), 153, dev, FP, 3000.0)
    for t in (q, k, v):
        t.requires_grad_(True)
    for scale in (0.125, 0.01):
        on = ref.seen(T, T, 0, 3, 0, True, None, 1, dev)
        got = torch.autograd.grad(window.window_attn(q, k, v, window=3, scale=scale), (q, k, v), do)
        want, bound = ref.gradients(q.detach(), k.detach(), v.detach(), on, scale, do, FP)
        for name, g, x, b in zip(("dq", "dk", "dv"), got, want, bound):
            assert x.abs().max() < 60000
            ref.close(g, x, b, name)
    bad = do.clone()
    bad[:, 200] = float("inf")
    hurt = torch.autograd.grad(window.window_attn(q, k, v, window=3, scale=scale), (q, k, v), bad)
    far = torch.ones(T, dtype=torch.bool, device=dev)
    far[128:256] = False  # (the rows and keys that share a workgroup with it may be reached by 0 times it)
    for g, x in zip(hurt, got):
        assert torch.equal(g[:, far], x[:, far]) and not torch.isfinite(g[:, 200]).all()


@pytest.mark.parametrize("causal", [True, False])
def test_window_sinks_that_are_all_keys(window, dev, causal):
    """Sinks that reach every key, alone or with the window: the bits of a call without a window."""
    q, k, v = (randn((1, 700, h, 64), s, dev).requires_grad_(True) for s, h in enumerate((4, 2, 2)))
    do = randn((1, 700, 4, 64), 3, dev)

    def run(w, s):
        o = window.window_attn(q, k, v, window=w, sinks=s, causal=causal)
        return [o, *torch.autograd.grad(o, (q, k, v), do)]

    want = run(None, 0)
    for w, s in ((64, 700), (1, 10 ** 9), (700, 30)) + (((100, 600), (599, 101)) if causal else ()):
        assert all(torch.equal(x, y) for x, y in zip(run(w, s), want)), (w, s)


# As WINDOW: many sinks and narrow windows, whose blocks' parts are long
MANY_SINKS = [
    (1, 3000, 3000, 2, 1, 128, 33, 700, True, None, BF),
    (2, 2100, 2300, 8, 8, 64, 16, 1000, False, [2300, 1500], FP),
    (1, 1700, 1700, 40, 40, 128, 10, 600, True, None, FP),
    (1, 1500, 1500, 6, 2, 64, 64, 1500, False, None, BF),
]


@pytest.mark.parametrize("case", MANY_SINKS, ids=[str(i) for i in range(len(MANY_SINKS))])
def test_window_many_sinks(window, dev, case):
    test_window(window, dev, case)
    test_window_gradients(window, dev, case)


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp16"])
@pytest.mark.parametrize("D,T,Tk,start,w,sinks", [(128, 200, 8000, 0, None, 0), (64, 300, 3000, 60, 2900, 4), (128, 900, 5000, 0, None, 0)])
def test_window_gradients_of_few_keys_by_position(window, dev, D, T, Tk, start, w, sinks, dtype):
    """A prompt at the beginning of a long buffer of keys: its rows see few of them whatever the window
    is, and the bound is that of few keys above."""
    q, k, v = randn((1, T, 4, D), 160, dev, dtype, 2.0), randn((1, Tk, 2, D), 161, dev, dtype), randn((1, Tk, 2, D), 162, dev, dtype)
    do = randn(q.shape, 163, dev, dtype)
    on = ref.seen(T, Tk, start, w, sinks, True, None, 1, dev)
    for t in (q, k, v):
        t.requires_grad_(True)
    got = torch.autograd.grad(window.window_attn(q, k, v, window=w, sinks=sinks, q_start=start, scale=0.11), (q, k, v), do)
    want, _ = ref.gradients(q.detach(), k.detach(), v.detach(), on, 0.11, do, dtype)
    ratios = {}
    for name, g, x in zip(("dq", "dk", "dv"), got, want):
        ratios[name] = ((g.double() - x).norm() / (x.to(dtype).double() - x).norm()).item()
    print("[few keys]", D, T, Tk, start, ratios, flush=True)
    assert all(x <= 1.25 for x in ratios.values()), ratios


# As WINDOW, and q_start: rows at the beginning or in the middle of the keys
PLACED = [
    (1, 300, 900, 2, 1, 128, 100, 4, True, None, BF, 0),
    (2, 257, 1500, 4, 2, 64, 200, 30, True, [1500, 700], FP, 600),
    (1, 200, 1000, 2, 2, 128, 50, 700, True, None, BF, 100),   # sinks above the rows
    (1, 300, 1200, 2, 2, 128, 64, 200, False, None, BF, 500),  # and below them
    (1, 190, 800, 2, 1, 64, 50, 400, False, None, FP, 0),
    (3, 150, 700, 3, 1, 64, 33, 0, False, [700, 0, 301], BF, 250),
    (1, 2000, 2600, 1, 1, 64, None, 0, True, None, BF, 300),   # blocks of keys cut into parts
    (1, 2000, 2500, 2, 1, 128, 40, 100, True, None, FP, 200),  # sinks' blocks cut into parts
    (1, 70, 6000, 2, 1, 128, None, 0, True, None, FP, 3000),   # key tiles of the forward cut into parts
    (1, 200, 700, 3, 3, 80, 60, 5, True, None, BF, 250),
    (2, 1, 500, 4, 2, 64, 90, 3, True, None, FP, 77),
]


@pytest.mark.parametrize("case", PLACED, ids=[str(i) for i in range(len(PLACED))])
def test_window_placed_rows(window, dev, case):
    """Forward and gradients where q_start is not Tk - Tq; keys that no row sees may hold anything and
    have gradients of exact zeros."""
    B, Tq, Tk, H, Hkv, D, w, sinks, causal, lengths, dtype, start = case
    q, do = randn((B, Tq, H, D), 170, dev, dtype, 2.0), randn((B, Tq, H, D), 171, dev, dtype)
    k, v = randn((B, Tk, Hkv, D), 172, dev, dtype), randn((B, Tk, Hkv, D), 173, dev, dtype)
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=dev)
    on = ref.seen(Tq, Tk, start, w, sinks, causal, n, B, dev)
    dead_rows, dead_keys = ~on.any(2), ~on.any(1)
    q[dead_rows], do[dead_rows] = float("nan"), float("nan")
    k[dead_keys], v[dead_keys] = float("nan"), float("inf")
    for t in (q, k, v):
        t.requires_grad_(True)
    kw = dict(window=w, sinks=sinks, causal=causal, lengths=n, q_start=start, scale=0.11)
    print("[placed]", case, flush=True)
    o, p, (_, _, vh) = ref.attention(q.detach(), k.detach(), v.detach(), on, 0.11)
    bound = ref.forward_bound(o, p, vh, dtype)
    with torch.no_grad():
        ref.close(window.window_attn(q, k, v, **kw), o, bound, "o")
    out = window.window_attn(q, k, v, **kw)
    ref.close(out.detach(), o, bound, "o of training")
    got = torch.autograd.grad(out, (q, k, v), do)
    want, bounds = ref.gradients(q.detach(), k.detach(), v.detach(), on, 0.11, do, dtype)
    for name, g, x, b in zip(("dq", "dk", "dv"), got, want, bounds):
        ref.close(g, x, b, name)
    assert (got[0][dead_rows] == 0).all() and (got[1][dead_keys] == 0).all() and (got[2][dead_keys] == 0).all()


# -------------------------------------------------- promises of the C entries
@pytest.fixture(scope="module")
def lib(pkg):
    return importlib.import_module(f"{pkg.__name__}._capi")


def _at(t):
    return [t.data_ptr(), *t.stride()[:3]]


@pytest.mark.parametrize("dtype,code", [(BF, 0), (FP, 1), (F32, 2)])
@pytest.mark.parametrize("Hkv,interleaved", [(2, 0), (0, 1)])
def test_c_norm_rope_in_place(rope, lib, dev, dtype, code, Hkv, interleaved):
    """Outputs that are the inputs, and q alone (no kv heads, null k)."""
    B, T, H, D = 2, 37, 6, 96
    q, k = randn((B, T, H, D), 1, dev, dtype), randn((B, T, 2, D), 2, dev, dtype)
    w = 1 + 0.1 * randn((D,), 3, dev, F32)
    cos, sin = tables(T, D, dev)
    want = rope.qk_norm_rope(q, k, w, w, cos, sin, interleaved=bool(interleaved))
    k0, none = k.clone(), [None, 0, 0, 0]
    rc = lib.LIB.solattn_qk_norm_rope(
        *_at(q), *(_at(k) if Hkv else none), B, T, H, Hkv, D, code, w.data_ptr(), w.data_ptr(), cos.data_ptr(), sin.data_ptr(),
        T, D, interleaved, None, 0, 1e-6, *_at(q), *(_at(k) if Hkv else none), torch.cuda.current_stream().cuda_stream)
    assert rc == 0, lib.LIB.solattn_last_error()
    assert torch.equal(q, want[0]) and torch.equal(k, want[1] if Hkv else k0)


def test_c_norm_rope_backward_of_q_alone(rope, lib, dev):
    """No kv heads in the backward pass, one weight's gradient or the other's left out."""
    B, T, H, D = 1, 50, 5, 64
    q, g = randn((B, T, H, D), 1, dev), randn((B, T, H, D), 2, dev)
    w = (1 + 0.1 * randn((D,), 3, dev, F32)).requires_grad_(True)
    cos, sin = tables(T, D, dev)
    leaf = q.clone().requires_grad_(True)
    want = torch.autograd.grad(rope.qk_norm_rope(leaf, q, w, None, cos, sin)[0], (leaf, w), g)
    need = lib.LIB.solattn_qk_norm_rope_bwd_workspace_bytes(D)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    none, dq, dw = [None, 0, 0, 0], torch.empty_like(q), torch.empty(D, device=dev)
    for with_w in (True, False):
        rc = lib.LIB.solattn_qk_norm_rope_bwd(
            *_at(q), *none, *_at(g), *none, B, T, H, 0, D, 0, w.data_ptr(), None, cos.data_ptr(), sin.data_ptr(), T, D, 0, None,
            0, 1e-6, *_at(dq), *none, dw.data_ptr() if with_w else None, None, ws.data_ptr() if with_w else None,
            need if with_w else 0, torch.cuda.current_stream().cuda_stream)
        assert rc == 0, lib.LIB.solattn_last_error()
        assert torch.equal(dq, want[0]) and torch.equal(dw, want[1])
        dq.fill_(0)


@pytest.mark.parametrize("dtype,code", [(BF, 0), (FP, 1)])
def test_c_window_backward_without_o_lo(lib, dev, dtype, code):
    """The forward's o_lo left out of both calls: o alone gives D_i, within the bounds of o as rounded."""
    B, T, H, Hkv, D, w = 1, 333, 4, 2, 128, 90
    q, do = randn((B, T, H, D), 1, dev, dtype, 2.0), randn((B, T, H, D), 4, dev, dtype)
    k, v = randn((B, T, Hkv, D), 2, dev, dtype), randn((B, T, Hkv, D), 3, dev, dtype)
    L, stream = lib.LIB, torch.cuda.current_stream().cuda_stream
    o, lse = torch.empty_like(q), torch.empty(B, H, T, device=dev)
    need = L.solattn_window_attn_workspace_bytes(B, T, T, H, Hkv, D, 0, w, 3, 1, 1)
    ws = torch.empty(max(need, 256), dtype=torch.uint8, device=dev)
    sizes = [B, T, T, H, Hkv, D, code, 0, None, w, 3, 1, 0.11]
    assert L.solattn_window_attn(*_at(q), *_at(k), *_at(v), *sizes, *_at(o), lse.data_ptr(), None, ws.data_ptr(), need,
                                 stream) == 0, L.solattn_last_error()
    need = L.solattn_window_attn_bwd_workspace_bytes(B, T, T, H, Hkv, D, w, 3, 1)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    assert L.solattn_window_attn_bwd(*_at(q), *_at(k), *_at(v), *_at(o), *_at(do), lse.data_ptr(), None, *sizes, *_at(dq),
                                     *_at(dk), *_at(dv), ws.data_ptr(), need, stream) == 0, L.solattn_last_error()
    on = ref.seen(T, T, 0, w, 3, True, None, B, dev)
    want, bound = ref.gradients(q, k, v, on, 0.11, do, dtype)
    for name, g, x, b in zip(("dq", "dk", "dv"), (dq, dk, dv), want, bound):
        ref.close(g, x, b, name)


def test_window_refuses_wrapped_positions(window, dev):
    x = torch.zeros(1, 8, 2, 64, device=dev, dtype=BF)
    for start in (2 ** 63 - 1, 2 ** 63 - 8, 2 ** 62, -2 ** 63):
        for rows in (x, x[:, :1]):
            with pytest.raises(ValueError, match="rows"):
                window.window_attn(rows, x, x, window=4, q_start=start)


def test_append_refuses_one_cache_for_both(rope, dev):
    """k and v of a token would race for the same slot."""
    kv = torch.zeros(3, 2, 8, 2, 64, device=dev, dtype=BF)
    x = torch.ones(1, 1, 2, 64, device=dev, dtype=BF)
    t, n = torch.zeros(1, 1, dtype=torch.int32, device=dev), torch.ones(1, dtype=torch.int32, device=dev)
    for k, v in ((kv[:, 0], kv[:, 0]), (kv[0], kv.flatten(0, 1)[:2])):
        with pytest.raises(ValueError, match="same memory"):
            rope.qk_norm_rope_append(x, x, x, k, v, t, n)
    assert (kv == 0).all()
    rope.qk_norm_rope_append(x, x, x, kv[:, 0], kv[:, 1], t, n)  # side by side is fine
    assert (kv[0, :, 0] == 1).all() and (kv[1:] == 0).all()
