"""What the C entries of the 8-bit cache and of attention over shared keys refuse, the
sizes of their workspaces, and the reference of the codes, without a GPU: every address
is a stand-in and nothing reaches a launch."""

import importlib

import pytest
import torch

import _cache8 as c8

A = 1 << 20  # aligned, never dereferenced
EINVAL, EUNSUPPORTED, ESIZE = -1, -2, -4
TOP = (1 << 63) - 1


@pytest.fixture(scope="module")
def capi(pkg):
    return importlib.import_module(f"{pkg.__name__}._capi")


def _said(capi, got, rc, text):
    assert got == rc and text in capi.LIB.solattn_last_error(), (got, capi.LIB.solattn_last_error())


CACHE = [
    (dict(dtype=3), EINVAL, b"dtype"), (dict(ct=0), EINVAL, b"cache type"), (dict(ct=3), EINVAL, b"cache type"),
    (dict(T=0), EINVAL, b"sizes"), (dict(D=24), EUNSUPPORTED, b"head_dim"), (dict(D=144), EUNSUPPORTED, b"head_dim"),
    (dict(B=1 << 31), EUNSUPPORTED, b"many"), (dict(B=1 << 20, T=1 << 12), EUNSUPPORTED, b"many"),
    (dict(B=TOP, T=TOP), EUNSUPPORTED, b"many"), (dict(B=1 << 20, T=1 << 5), EUNSUPPORTED, b"one launch"),
    (dict(B=1 << 20, T=1 << 6, D=64), EUNSUPPORTED, b"one launch"), (dict(table=None), EINVAL, b"page table"), (dict(n=None), EINVAL, b"lengths"),
    (dict(pages=-1), EUNSUPPORTED, b"pages"), (dict(page=0), EUNSUPPORTED, b"pages"), (dict(most=1 << 28), EUNSUPPORTED, b"2^31"),
    (dict(most=TOP), EUNSUPPORTED, b"2^31"), (dict(x=None), EINVAL, b"null k"), (dict(x=A + 8), EINVAL, b"k must be 16-byte"),
    (dict(c=None), EINVAL, b"null k_cache"), (dict(c=A + 8), EINVAL, b"k_cache must be 16-byte"),
    (dict(cs=(1 << 15, 1032, 128)), EINVAL, b"k_cache must be 16-byte"), (dict(s=None), EINVAL, b"scales"),
]


def _cache_args(kw):
    o = dict(dtype=0, ct=1, B=2, T=3, Hkv=8, D=128, pages=9, page=16, most=4, x=A, c=A, cs=(16 * 1024, 1024, 128), s=A, table=A, n=A)
    o.update(kw)
    return o


@pytest.mark.parametrize("kw,rc,text", CACHE)
def test_cache_append_refusals(capi, kw, rc, text):
    o = _cache_args(kw)
    x, ss = (3 * 1024, 1024, 128), (128, 16)
    got = capi.LIB.solattn_cache_append(o["x"], *x, A, *x, o["B"], o["T"], o["Hkv"], o["D"], o["dtype"], o["c"], *o["cs"], A,
                                        *o["cs"], o["pages"], o["page"], o["ct"], o["s"], *ss, A, *ss, o["table"], 4, o["most"],
                                        o["n"], None)
    _said(capi, got, rc, text)


@pytest.mark.parametrize("kw,rc,text", CACHE + [(dict(dtype=2), EINVAL, b"dtype")])
def test_cache_read_refusals(capi, kw, rc, text):
    o = _cache_args(kw)
    x, ss = (3 * 1024, 1024, 128), (128, 16)
    got = capi.LIB.solattn_cache_read(o["c"], *o["cs"], A, *o["cs"], o["pages"], o["page"], o["ct"], o["s"], *ss, A, *ss,
                                      o["table"], 4, o["most"], o["n"], None, o["B"], o["T"], o["Hkv"], o["D"], o["dtype"],
                                      o["x"], *x, A, *x, None)
    _said(capi, got, rc, text)


@pytest.mark.parametrize("kw,rc,text", [
    (dict(ct=0), EINVAL, b"cache type"), (dict(ct=-1), EINVAL, b"cache type"), (dict(ct=3), EINVAL, b"cache type"),
    (dict(D=120), EUNSUPPORTED, b"multiples of 16"), (dict(s=None), EINVAL, b"scales"), (dict(c=A + 8), EINVAL, b"k_cache"),
    (dict(cs=(2048, 136, 128)), EINVAL, b"k_cache"), (dict(table=None), EINVAL, b"page table"), (dict(dtype=3), EINVAL, b"dtype"),
])
def test_append8_refusals(capi, kw, rc, text):
    o = _cache_args(dict(cs=(2048, 128, 128), **kw) if "cs" not in kw else kw)
    s = (128, 128, 128)
    got = capi.LIB.solattn_qk_norm_rope_append8(
        A, *s, A, *s, A, *s, 1, 1, 1, 1, o["D"], o["dtype"], A, A, None, None, 0, 0, 0, 1e-6, A, *s, o["c"], *o["cs"], A, *o["cs"],
        4, 16, o["ct"], o["s"], 16, 16, A, 16, 16, o["table"], 2, 2, A, None)
    _said(capi, got, rc, text)


def _paged(L, B=4, H=4, Hkv=2, D=128, dtype=0, ct=1, page=16, pages=9, most=64, scale=0.1, window=0, sinks=0, shared=0,
           groups=1, ks=A, vs=A, ss=(64, 16), cs=None, ws=A, need=1 << 30, q=A):
    c = cs or (page * Hkv * D, Hkv * D, D)
    return L.solattn_paged_attn_shared(q, H * D, D, A, *c, A, *c, pages, page, ct, ks, *ss, vs, *ss, A, most, most, A, B, H, Hkv,
                                       D, dtype, window, sinks, shared, groups, scale, ws, need, A, H * D, D, None)


@pytest.mark.parametrize("kw,rc,text", [
    (dict(ct=3), EINVAL, b"cache type"), (dict(ct=-1), EINVAL, b"cache type"), (dict(D=120), EUNSUPPORTED, b"multiples of 16"),
    (dict(ks=None), EINVAL, b"scales"), (dict(vs=A + 4), EINVAL, b"scales"), (dict(ss=(64, 12)), EINVAL, b"scales"),
    (dict(cs=(4096, 264, 128)), EINVAL, b"multiple of 16"), (dict(shared=-1), EINVAL, b"shared"), (dict(shared=1 << 31), EINVAL, b"shared"),
    (dict(shared=5, window=3), EINVAL, b"window"), (dict(shared=5, sinks=3), EINVAL, b"window"),
    (dict(shared=5, groups=0), EINVAL, b"groups"), (dict(shared=5, groups=3), EINVAL, b"groups"), (dict(page=12), EINVAL, b"multiple of 8"),
    (dict(dtype=2), EINVAL, b"dtype"), (dict(H=3), EINVAL, b"heads"), (dict(B=1 << 31, shared=4), EUNSUPPORTED, b"grid"),
    (dict(B=1 << 30, H=1, Hkv=1, shared=4, groups=1 << 30), EUNSUPPORTED, b"grid"), (dict(B=1 << 24, H=1, Hkv=1, need=TOP), EUNSUPPORTED, b"grid"),
    (dict(scale=0.0), EINVAL, b"scale"), (dict(most=(1 << 27) - 2), EUNSUPPORTED, b"2^31 keys"),
    (dict(most=(1 << 27) - 128, shared=4), EUNSUPPORTED, b"2^31 keys"), (dict(most=(1 << 27) - 3, shared=4), EUNSUPPORTED, b"2^31 keys"),
    (dict(shared=500, need=0), ESIZE, b"workspace"), (dict(shared=500, ws=A + 16), EINVAL, b"256"), (dict(q=A + 8), EINVAL, b"aligned"),
])
def test_paged_refusals(capi, kw, rc, text):
    if kw.get("groups") == 1 << 30:
        kw = dict(kw, need=TOP)
    _said(capi, _paged(capi.LIB, **kw), rc, text)


def test_launches_of_2_to_the_32_threads(capi):
    """The fewest rows whose workgroups, rounded up, are 2^24 of 256 threads; nothing is launched before a
    join that cannot be."""
    L, s = capi.LIB, (512, 512, 128)
    for D, T in ((128, (1 << 28) - 15), (64, (1 << 29) - 31)):
        o, ss = _cache_args(dict(D=D, T=T, B=1, Hkv=1)), (128, 16)
        rest = (o["pages"], o["page"], o["ct"], A, *ss, A, *ss, A, 4, o["most"], A)
        _said(capi, L.solattn_cache_append(A, *s, A, *s, 1, T, 1, D, 0, A, *o["cs"], A, *o["cs"], *rest, None), EUNSUPPORTED,
              b"one launch")
        _said(capi, L.solattn_cache_read(A, *o["cs"], A, *o["cs"], *rest, None, 1, T, 1, D, 0, A, *s, A, *s, None), EUNSUPPORTED,
              b"one launch")
    T = (1 << 26) - 3  # a wave a token
    _said(capi, L.solattn_qk_norm_rope_append8(
        A, *s, A, *s, A, *s, 1, T, 4, 4, 128, 0, A, A, None, None, 0, 0, 0, 1e-6, A, *s, A, *s, A, *s, 4, 16, 1, A, 64, 16, A, 64, 16,
        A, 2, 2, A, None), EUNSUPPORTED, b"grid")
    _said(capi, L.solattn_qk_norm_rope(A, *s, A, *s, 1, T, 4, 4, 128, 0, A, A, None, None, 0, 0, 0, None, 0, 1e-6, A, *s, A, *s, None),
          EUNSUPPORTED, b"grid")
    # 2^23 workgroups of two parts, 2^26 rows to join, four a workgroup; over codes a workgroup each
    for ct, B in ((0, 1 << 22), (1, 1 << 20)):
        _said(capi, _paged(L, ct=ct, B=B, H=16, Hkv=1, most=512, need=TOP), EUNSUPPORTED, b"grid")


def test_paged_workspace(capi):
    """A row's parts over shared keys and over its own, 64 at most of each; sizes that no call takes have none."""
    L = capi.LIB
    need = L.solattn_paged_attn_shared_workspace_bytes
    for B, H, Hkv, D, most, shared, groups in ((8, 24, 8, 128, 70, 4100, 1), (256, 24, 8, 128, 520, 32760, 1), (64, 16, 4, 64, 525, 8000, 4),
                                               (1, 1, 1, 64, 1000, 60000, 1), (2, 1, 1, 64, 1 << 20, 1 << 25, 1), (4, 8, 8, 128, 4, 64, 4)):
        row = B * H * (D + 2) * 4
        size = need(B, H, Hkv, D, most, 64, 0, 0, 0, shared, groups)
        assert size % row == 0 and 2 <= size // row <= 128
    for args in ((4, 4, 2, 128, 64, 16, 0, 0, 0, 5, 3), (4, 4, 2, 128, 64, 16, 0, 0, 0, -1, 1), (4, 4, 2, 128, 64, 16, 0, 0, 0, TOP, 1),
                 (TOP, 2, 1, 128, 64, 16, 0, 0, 0, 5, 1), (4, 4, 2, 128, TOP, TOP, 0, 0, 0, 5, 1), (4, 4, 2, TOP, 64, 16, 0, 0, 0, 5, 1),
                 (4, 4, 2, 128, 64, 16, 0, 0, 0, 5, 0), (4, 4, 2, 128, 64, 16, 0, 0, 0, 5, -2)):
        assert need(*args) == 0, args
    assert need(1, 24, 8, 128, 1000, 64, 0, 0, 2, 0, 1) == L.solattn_paged_attn_workspace_bytes(1, 24, 8, 128, 1000, 64, 0, 0)


def test_reference_codes():
    """The reference's e4m3 rounding against the format's arithmetic, its powers against their definition."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(2000, 64, generator=g, dtype=torch.float64) * 10.0 ** (8 * torch.rand(2000, 1, generator=g) - 4)
    x = x.float()
    x[0] = torch.linspace(0, 448, 64)
    x[1] = torch.arange(64) * 0.25
    for kind, most in c8.MOST.items():
        codes, byte = c8.encode(x, kind)
        unit = c8.power(byte)[:, None]
        top = x.double().abs().amax(-1, keepdim=True)
        assert (top <= most * unit).all() and (top > most / 2 * unit).all()
        y = x.double() / unit
        if kind == torch.int8:
            want = torch.round(y)
        else:
            step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(1e-30))).clamp_min(-6) - 3)
            want = torch.round(y / step) * step
        assert torch.equal(c8.values(codes, byte), want * unit)
        # 16 bits hold the values
        assert torch.equal(c8.values(codes, byte).to(torch.bfloat16).double(), c8.values(codes, byte))


def _calls(pkg):
    mod = lambda name: importlib.import_module(f"{pkg.__name__}.{name}")  # noqa: E731
    x = torch.zeros(1, 8, 2, 64, dtype=torch.bfloat16)
    one = x[:, :1].clone()
    c = torch.zeros(1, 8, 2, 64, dtype=torch.int8)
    s = torch.zeros(1, 2, 8, dtype=torch.uint8).view(c8.E8)
    t, n = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    rope, cache, paged = mod("_qk_rope"), mod("_cache"), mod("_paged")
    return [
        ("qk_norm_rope_append", lambda q, k, v: rope.qk_norm_rope_append(q, k, v, c, c, t, n, k_scale=s, v_scale=s), [one, one, one]),
        ("cache_append", lambda k, v: cache.cache_append(k, v, c, c, t, n, s, s), [one, one]),
        ("paged_attn", lambda q: paged.paged_attn(q, c, c, t, n, k_scale=s, v_scale=s), [one]),
        ("paged_attn", lambda q, k, v: paged.paged_attn(q, k, v, t, n, shared=3), [one, x, x]),
        ("cache_read", lambda k, v: cache.cache_read(k, v, t, n, s, s, tokens=3), [c, c]),
    ]


@pytest.mark.parametrize("i", range(5))
def test_host_tensors_recorders_and_tangents_are_refused(pkg, i):
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.autograd import forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx

    name, f, args = _calls(pkg)[i]
    with pytest.raises(ValueError, match="GPU"):
        f(*args)
    with pytest.raises(ValueError, match=f"{name} cannot be traced"):
        make_fx(f)(*args)
    with FakeTensorMode(allow_non_fake_inputs=True), pytest.raises(ValueError, match=f"{name} cannot be traced"):
        f(*args)
    for j, x in enumerate(args):
        if x.is_floating_point():
            with forward_ad.dual_level():
                y = list(args)
                y[j] = forward_ad.make_dual(x.clone(), torch.ones_like(x))
                with pytest.raises(ValueError, match=f"{name} has no forward-mode derivative"):
                    f(*y)
