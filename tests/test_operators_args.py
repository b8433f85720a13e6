"""What the C entries of the operators around attention refuse, and the sizes of their
workspaces, without a GPU: every address is a stand-in and nothing reaches a launch."""

import importlib

import pytest
import torch

A = 1 << 20  # aligned, never dereferenced
EINVAL, EUNSUPPORTED, ESIZE = -1, -2, -4


@pytest.fixture(scope="module")
def capi(pkg):
    return importlib.import_module(f"{pkg.__name__}._capi")


def _rope(L, q=A, k=A, B=1, T=10, H=4, Hkv=2, D=128, dtype=0, qw=A, cos=A, sin=A, P=10, R=128, interleaved=0,
          positions=None, qo=A, ko=A, qs=None):
    qs = qs or (T * H * D, H * D, D)
    ks = (T * Hkv * D, Hkv * D, D)
    return L.solattn_qk_norm_rope(q, *qs, k, *ks, B, T, H, Hkv, D, dtype, qw, A, cos, sin, P, R, interleaved, positions, 0,
                                  1e-6, qo, T * H * D, H * D, D, ko, *ks, None)


@pytest.mark.parametrize("kw,rc,text", [
    (dict(dtype=3), EINVAL, b"dtype"), (dict(B=0), EINVAL, b"sizes"), (dict(D=132), EUNSUPPORTED, b"head_dim"),
    (dict(D=136), EUNSUPPORTED, b"head_dim"), (dict(R=24), EUNSUPPORTED, b"rotated"),
    (dict(R=136), EUNSUPPORTED, b"rotated"), (dict(R=12, interleaved=1), EUNSUPPORTED, b"rotated"),
    (dict(cos=None), EINVAL, b"table"), (dict(P=9), EINVAL, b"table of 9"), (dict(q=None), EINVAL, b"null q"),
    (dict(q=A + 8), EINVAL, b"aligned"), (dict(qs=(5120, 508, 128)), EINVAL, b"aligned"), (dict(ko=None), EINVAL, b"null k"),
    (dict(qw=A + 4), EINVAL, b"aligned"), (dict(T=1 << 31), EINVAL, b"table of"), (dict(B=1 << 31, T=2), EUNSUPPORTED, b"many"),
])
def test_rope_refusals(capi, kw, rc, text):
    if kw.get("T") == 1 << 31:  # (the size is refused before the table is)
        rc, text = EUNSUPPORTED, b"many"
    assert _rope(capi.LIB, **kw) == rc
    assert text in capi.LIB.solattn_last_error(), capi.LIB.solattn_last_error()


def test_rope_backward_workspace(capi):
    L = capi.LIB
    assert L.solattn_qk_norm_rope_bwd_workspace_bytes(0) == 0
    need = L.solattn_qk_norm_rope_bwd_workspace_bytes(128)
    s = (1280, 128, 128)
    args = [A, *s, A, *s, A, *s, A, *s, 1, 10, 1, 1, 128, 0, A, A, A, A, 10, 128, 0, None, 0, 1e-6, A, *s, A, *s]
    assert L.solattn_qk_norm_rope_bwd(*args, A, A, A, need - 1, None) == ESIZE
    assert L.solattn_qk_norm_rope_bwd(*args, A, A, None, need, None) == ESIZE
    assert L.solattn_qk_norm_rope_bwd(*args, A, A, A + 16, need, None) == EINVAL


@pytest.mark.parametrize("kw,rc,text", [
    (dict(table=None), EINVAL, b"page table"), (dict(lengths=None), EINVAL, b"lengths"), (dict(pages=-1), EUNSUPPORTED, b"pages"),
    (dict(page=0), EUNSUPPORTED, b"pages"), (dict(page=1 << 20, most=1 << 11), EUNSUPPORTED, b"2^31"),
    (dict(cache=A + 2), EINVAL, b"k_cache"), (dict(cache=None), EINVAL, b"k_cache"),
])
def test_append_refusals(capi, kw, rc, text):
    o = dict(table=A, lengths=A, pages=4, page=16, most=2, cache=A)
    o.update(kw)
    s, c = (128, 128, 128), (2048, 128, 128)
    got = capi.LIB.solattn_qk_norm_rope_append(
        A, *s, A, *s, A, *s, 1, 1, 1, 1, 128, 0, A, A, A, A, 10, 128, 0, 1e-6, A, *s, o["cache"], *c, A, *c, o["pages"],
        o["page"], o["table"], o["most"], o["most"], o["lengths"], None)
    assert got == rc and text in capi.LIB.solattn_last_error(), capi.LIB.solattn_last_error()


def _window(L, B=1, Tq=40, Tk=100, H=4, Hkv=2, D=128, dtype=0, q_start=60, window=16, sinks=2, causal=1, scale=0.1,
            q=A, k=A, o=A, lse=None, ws=None, ws_bytes=0, kt=None):
    qs, ks = (Tq * H * D, H * D, D), (Tk * Hkv * D, kt or Hkv * D, D)
    return L.solattn_window_attn(q, *qs, k, *ks, A, *ks, B, Tq, Tk, H, Hkv, D, dtype, q_start, None, window, sinks, causal,
                                 scale, o, *qs, lse, None, ws, ws_bytes, None)


@pytest.mark.parametrize("kw,rc,text", [
    (dict(dtype=2), EINVAL, b"dtype"), (dict(H=3), EINVAL, b"heads"), (dict(Tq=0), EINVAL, b"sizes"),
    (dict(D=96), EUNSUPPORTED, b"head_dim"), (dict(q_start=61), EINVAL, b"rows"), (dict(q_start=-1), EINVAL, b"rows"),
    (dict(window=0), EINVAL, b"window"), (dict(sinks=-1), EINVAL, b"sinks"), (dict(scale=0.0), EINVAL, b"scale"),
    (dict(scale=float("nan")), EINVAL, b"scale"), (dict(q=None), EINVAL, b"null q"), (dict(o=A + 8), EINVAL, b"aligned"),
    (dict(kt=252), EINVAL, b"aligned"), (dict(kt=1 << 24), EUNSUPPORTED, b"stride"), (dict(kt=-256), EUNSUPPORTED, b"stride"),
    (dict(Tk=1 << 29, q_start=0), EUNSUPPORTED, b"keys"), (dict(B=1 << 24, H=128), EUNSUPPORTED, b"grid"),
])
def test_window_refusals(capi, kw, rc, text):
    assert _window(capi.LIB, **kw) == rc
    assert text in capi.LIB.solattn_last_error(), capi.LIB.solattn_last_error()


def test_window_workspaces(capi):
    """A short launch asks for room for its parts and refuses less; a full one for none."""
    L = capi.LIB
    assert L.solattn_window_attn_workspace_bytes(1, 16000, 16000, 24, 8, 128, 0, 4096, 4, 1, 0) == 0
    need = L.solattn_window_attn_workspace_bytes(1, 64, 8192, 2, 1, 128, 8128, 8192, 0, 1, 0)
    assert need > 0
    kw = dict(Tq=64, Tk=8192, H=2, Hkv=1, q_start=8128, window=8192, sinks=0)
    assert _window(L, **kw, ws=A, ws_bytes=need - 1) == ESIZE
    assert _window(L, **kw, ws=None, ws_bytes=need) == ESIZE
    assert _window(L, **kw, ws=A + 128, ws_bytes=need) == EINVAL
    one = L.solattn_window_attn_workspace_bytes(1, 1, 8192, 2, 1, 128, 8191, 8192, 0, 1, 0)
    assert one > 0 and one == L.solattn_paged_attn_workspace_bytes(1, 2, 1, 128, 1, 8192, 8192, 0)
    assert _window(L, Tq=1, Tk=8192, H=2, Hkv=1, q_start=8191, window=8192, sinks=0, ws=A, ws_bytes=one - 1) == ESIZE
    assert L.solattn_window_attn_workspace_bytes(1, 64, 32, 2, 1, 128, 0, 8, 0, 1, 0) == 0  # not a call that runs
    assert L.solattn_window_attn_bwd_workspace_bytes(2, 100, 100, 4, 2, 64, 100, 0, 1) >= 2 * 100 * 4 * 4


def test_window_backward_refusals(capi):
    L = capi.LIB
    s = (12800, 128, 128)
    need = L.solattn_window_attn_bwd_workspace_bytes(1, 100, 100, 1, 1, 128, 100, 0, 1)

    def call(lse=A, ws=A, ws_bytes=need, dk=A, do=A):
        return L.solattn_window_attn_bwd(A, *s, A, *s, A, *s, A, *s, do, *s, lse, None, 1, 100, 100, 1, 1, 128, 0, 0, None,
                                         100, 0, 1, 0.1, A, *s, dk, *s, A, *s, ws, ws_bytes, None)

    assert call(lse=None) == EINVAL and call(ws_bytes=need - 1) == ESIZE and call(ws=A + 8) == EINVAL
    assert call(dk=None) == EINVAL and b"null dk" in L.solattn_last_error()
    assert call(do=A + 2) == EINVAL and b"do must" in L.solattn_last_error()


@pytest.mark.parametrize("kw,rc,text", [
    (dict(dtype=2), EINVAL, b"dtype"), (dict(H=5), EINVAL, b"heads"), (dict(D=136), EUNSUPPORTED, b"head_dim"),
    (dict(page=12), EINVAL, b"multiple of 8"), (dict(pages=0), EINVAL, b"pages"), (dict(most=1 << 28), EUNSUPPORTED, b"2^31"),
    (dict(scale=-1.0), EINVAL, b"scale"), (dict(window=-1), EINVAL, b"window"), (dict(table=None), EINVAL, b"table"),
    (dict(q=A + 4), EINVAL, b"aligned"),
])
def test_paged_refusals(capi, kw, rc, text):
    o = dict(dtype=0, H=4, Hkv=2, D=128, page=16, pages=9, most=4, scale=0.1, window=0, table=A, q=A)
    o.update(kw)
    c = (o["page"] * 256, 256, 128)
    got = capi.LIB.solattn_paged_attn(o["q"], 512, 128, A, *c, A, *c, o["pages"], o["page"], o["table"], o["most"], o["most"],
                                      A, 1, o["H"], o["Hkv"], o["D"], o["dtype"], o["window"], 0, o["scale"], None, 0, A, 512,
                                      128, None)
    assert got == rc and text in capi.LIB.solattn_last_error(), capi.LIB.solattn_last_error()


def test_paged_workspace(capi):
    L = capi.LIB
    need = L.solattn_paged_attn_workspace_bytes(1, 24, 8, 128, 1000, 64, 0, 0)
    splits = need // (24 * 130 * 4)
    assert need == splits * 24 * 130 * 4 and 1 < splits <= 64
    # a window bounds what is split; enough sequences need no split, but that none has
    # more than 4096 keys where a table may hold more
    assert L.solattn_paged_attn_workspace_bytes(1, 24, 8, 128, 1000, 64, 100, 4) < need
    assert L.solattn_paged_attn_workspace_bytes(256, 24, 8, 128, 64, 64, 0, 0) == 0
    assert L.solattn_paged_attn_workspace_bytes(256, 24, 8, 128, 65, 64, 0, 0) == 256 * 24 * 2 * 130 * 4
    assert L.solattn_paged_attn_workspace_bytes(1, 24, 7, 128, 1000, 64, 0, 0) == 0
    c = (64 * 1024, 1024, 128)
    rc = L.solattn_paged_attn(A, 24 * 128, 128, A, *c, A, *c, 1000, 64, A, 1000, 1000, A, 1, 24, 8, 128, 0, 0, 0, 0.1, A,
                              need - 1, A, 24 * 128, 128, None)
    assert rc == ESIZE and b"workspace" in L.solattn_last_error()


def test_host_tensors_are_refused(pkg):
    """There is no CPU path: the operators say so."""
    x = torch.zeros(1, 8, 2, 64, dtype=torch.bfloat16)
    t = torch.zeros(1, 1, dtype=torch.int32)
    n = torch.ones(1, dtype=torch.int32)
    mod = lambda name: importlib.import_module(f"{pkg.__name__}.{name}")  # noqa: E731
    with pytest.raises(ValueError, match="GPU"):
        mod("_qk_rope").qk_norm_rope(x, x)
    with pytest.raises(ValueError, match="GPU"):
        mod("_window").window_attn(x, x, x, window=4)
    with pytest.raises(ValueError, match="GPU"):
        mod("_paged").paged_attn(x[:, :1], x, x, t, n)
    with pytest.raises(ValueError, match="GPU"):
        mod("_qk_rope").qk_norm_rope_append(x[:, :1], x[:, :1], x[:, :1], x, x, t, n)
    with pytest.raises(TypeError):
        mod("_window").window_attn(x, x, x)  # the window has no default


def test_wide_windows_and_eps(capi):
    """Windows past every key are no limit in each entry; eps is from 0 on."""
    L, top = capi.LIB, (1 << 62) + (1 << 61)
    assert L.solattn_paged_attn_workspace_bytes(1, 24, 8, 128, 1000, 64, top, top) == \
        L.solattn_paged_attn_workspace_bytes(1, 24, 8, 128, 1000, 64, 0, 0)
    one = L.solattn_window_attn_workspace_bytes(1, 1, 8192, 2, 1, 128, 8191, top, top, 1, 0)
    assert one == L.solattn_window_attn_workspace_bytes(1, 1, 8192, 2, 1, 128, 8191, 8192, 0, 1, 0) > 0
    # (the room is what is refused, not the window)
    assert _window(L, Tq=1, Tk=8192, H=2, Hkv=1, q_start=8191, window=top, sinks=top, ws=A, ws_bytes=one - 1) == ESIZE
    s = (1280, 128, 128)
    for eps in (-1e-6, float("nan")):
        assert L.solattn_qk_norm_rope(A, *s, A, *s, 1, 10, 1, 1, 128, 0, A, A, A, A, 10, 128, 0, None, 0, eps, A, *s, A, *s,
                                      None) == EINVAL
        assert b"eps" in L.solattn_last_error()


def _calls(pkg):
    """Every operator as a function of its float tensors: (name, function, arguments on the host)."""
    mod = lambda name: importlib.import_module(f"{pkg.__name__}.{name}")  # noqa: E731
    x = torch.zeros(1, 8, 2, 64, dtype=torch.bfloat16)
    one = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16)
    w, cos = torch.ones(64), torch.ones(8, 32)
    t, n = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    rope, window, paged = mod("_qk_rope"), mod("_window"), mod("_paged")
    return [
        ("qk_norm_rope", lambda *a: rope.qk_norm_rope(*a), [x, x, w, w, cos, cos]),
        ("qk_norm_rope_append", lambda q, k, v, kc, vc, qw, kw, c, s: rope.qk_norm_rope_append(
            q, k, v, kc, vc, t, n, qw, kw, c, s), [one, one, one, x, x, w, w, cos, cos]),
        ("window_attn", lambda q, k, v: window.window_attn(q, k, v, window=4), [x, x, x]),
        ("paged_attn", lambda q, kc, vc: paged.paged_attn(q, kc, vc, t, n), [one, x, x]),
    ]


@pytest.mark.parametrize("i", range(4))
def test_recorders_are_refused(pkg, i):
    """A trace would hold the outputs' allocation and no kernel: the calls refuse to be recorded."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx

    name, f, args = _calls(pkg)[i]
    with pytest.raises(ValueError, match=f"{name} cannot be traced"):
        torch.jit.trace(f, tuple(args))
    with pytest.raises(ValueError, match=f"{name} cannot be traced"):
        make_fx(f)(*args)
    with FakeTensorMode(allow_non_fake_inputs=True), pytest.raises(ValueError, match=f"{name} cannot be traced"):
        f(*args)
    with pytest.raises(ValueError, match="GPU"):  # (and only while they are)
        f(*args)


@pytest.mark.parametrize("i", range(4))
def test_tangents_are_refused(pkg, i):
    """A forward-mode derivative would be dropped: the calls refuse tensors that carry a tangent, whether
    or not these require a gradient, and take them where forward mode is off."""
    from torch.autograd import forward_ad

    name, f, args = _calls(pkg)[i]
    for j in range(len(args)):
        for leaf in (False, True):
            with forward_ad.dual_level():
                x = list(args)
                x[j] = forward_ad.make_dual(args[j].clone().requires_grad_(leaf), torch.ones_like(args[j]))
                with pytest.raises(ValueError, match=f"{name} has no forward-mode derivative"):
                    f(*x)
                with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):
                    f(*x)
                with torch.no_grad(), forward_ad._set_fwd_grad_enabled(False), pytest.raises(ValueError, match="GPU"):
                    f(*x)


@pytest.mark.parametrize("T,H,Hkv,window,sinks,causal", [
    (32760, 24, 24, 64, 1333, 0), (32760, 24, 24, 64, 4096, 0), (32760, 24, 24, 256, 300, 0), (65536, 24, 24, 128, 4000, 1),
    (12133, 24, 24, 64, 1333, 0), (32768, 24, 8, 64, 2000, 1), (32768, 1, 1, 64, 1000, 0), (100000, 2, 1, 16, 5000, 1),
])
def test_window_backward_workspace_of_many_sinks(capi, T, H, Hkv, window, sinks, causal):
    """The parts of sinks' blocks are bounded by what fills the CUs (1024 of a block's dk and dv in fp32,
    beside 512 of other blocks), and not by the length over the window: no more than twice q where q is long."""
    need = capi.LIB.solattn_window_attn_bwd_workspace_bytes(1, T, T, H, Hkv, 128, window, sinks, causal)
    rows = 2 * 4 * T * H + T * H + 1024  # two numbers a row, two for 32 rows, rounding up
    assert 0 < need <= rows + 1536 * 2 * 128 * 128 * 4
    if H == 24:
        assert need <= 2 * (T * H * 128 * 2)


@pytest.mark.parametrize("T,B,H", [(32768, 1, 24), (65536, 1, 24), (4096, 1, 1), (1000, 2, 3)])
def test_window_workspaces_of_sinks_that_are_all_keys(capi, T, B, H):
    """Sinks that reach every key are no window: the same call, the same workspace."""
    L = capi.LIB
    for causal in (0, 1):
        full = L.solattn_window_attn_bwd_workspace_bytes(B, T, T, H, H, 128, T, 0, causal)
        assert L.solattn_window_attn_bwd_workspace_bytes(B, T, T, H, H, 128, 64, T, causal) == full
        assert L.solattn_window_attn_bwd_workspace_bytes(B, T, T, H, H, 128, T, 77, causal) == full
    assert L.solattn_window_attn_bwd_workspace_bytes(B, T, T, H, H, 128, 64, T - 64, 1) == \
        L.solattn_window_attn_bwd_workspace_bytes(B, T, T, H, H, 128, T, 0, 1)
    rows = 2 * 4 * B * T * H + B * T * H + 1024
    assert L.solattn_window_attn_bwd_workspace_bytes(B, T, T, H, H, 128, T, 0, 1) <= rows + 1024 * 2 * 128 * 128 * 4


def test_window_parts_follow_what_rows_see(capi):
    """A causal call is cut by the keys up to its last position, not by those behind it."""
    need = capi.LIB.solattn_window_attn_workspace_bytes
    assert need(1, 64, 131072, 32, 32, 128, 0, 131072, 0, 1, 0) == 0  # one tile of 64 keys
    far = need(1, 256, 32000, 24, 8, 128, 31744, 32000, 0, 1, 0)
    assert need(1, 256, 32000, 24, 8, 128, 0, 32000, 0, 1, 0) == 0 < far
    row = 24 * 256 * 130 * 4
    for start in (500, 2000, 4000, 8000, 16000):
        parts = need(1, 256, 32000, 24, 8, 128, start, 32000, 0, 1, 0) // row
        assert parts <= max(1, (start + 256) // 64 // 8 + 1) and parts * row <= far
        # the keys behind the last row make no difference
        assert need(1, 256, start + 256, 24, 8, 128, start, 32000, 0, 1, 0) // row == parts
    assert need(1, 256, 32000, 24, 8, 128, 0, 32000, 0, 0, 0) == far  # (symmetric: every key is seen)


TOP = (1 << 63) - 1


def test_sizes_beyond_64_bits(capi):
    """Sizes whose sums and products pass 64 bits are refused like any that are too large: no wrapped
    position reaches a launch, no workspace's size divides by a product that became zero."""
    L = capi.LIB
    for start in (TOP, TOP - 1, TOP - 39, 1 << 62):
        assert _window(L, q_start=start) == EINVAL and b"rows" in L.solattn_last_error()
        assert _window(L, q_start=start, Tq=1) == EINVAL and b"row" in L.solattn_last_error()
        assert L.solattn_window_attn_workspace_bytes(1, 1, 100, 4, 2, 128, start, 16, 2, 1, 0) == 0
        assert L.solattn_window_attn_workspace_bytes(1, 40, 100, 4, 2, 128, start, 16, 2, 1, 0) == 0
    assert _window(L, Tq=TOP, q_start=1) == EINVAL and b"rows" in L.solattn_last_error()
    for B, H in ((1 << 62, 4), (1 << 40, 1 << 24), (1 << 31, 1), (1, 1 << 31), (1 << 16, 1 << 15), (TOP, 2)):
        assert _window(L, B=B, H=H, Hkv=1) == EUNSUPPORTED and b"grid" in L.solattn_last_error()
        assert _window(L, B=B, H=H, Hkv=1, Tq=1, q_start=9) == EUNSUPPORTED and b"grid" in L.solattn_last_error()
        assert L.solattn_window_attn_workspace_bytes(B, 64, 64, H, 1, 128, 0, 64, 0, 1, 0) == 0
        assert L.solattn_window_attn_workspace_bytes(B, 1, 64, H, 1, 128, 0, 64, 0, 1, 0) == 0
        assert L.solattn_window_attn_bwd_workspace_bytes(B, 64, 64, H, 1, 128, 64, 0, 1) == 0
        assert L.solattn_paged_attn_workspace_bytes(B, H, 1, 128, 4, 64, 0, 0) == 0
    assert L.solattn_paged_attn_workspace_bytes(1, 4, 4, 128, 1 << 40, 1 << 40, 0, 0) == 0
    assert L.solattn_paged_attn_workspace_bytes(1, 4, 4, TOP, 1000, 64, 0, 0) == 0


def test_window_forward_parts_fill_one_round(capi):
    """Parts stay within four workgroups a CU, and a launch that fills these is not cut (a batch with
    lengths has the same workspace as one without: the size does not know)."""
    need = capi.LIB.solattn_window_attn_workspace_bytes
    for B, Tq, Tk, H, Hkv, D in ((4, 2000, 2000, 16, 4, 128), (4, 1024, 4096, 16, 4, 128), (2, 4000, 4000, 8, 8, 128),
                                 (2, 517, 16000, 16, 4, 64), (8, 128, 32000, 8, 1, 128), (4, 256, 8000, 24, 8, 128)):
        parts = max(1, need(B, Tq, Tk, H, Hkv, D, Tk - Tq, Tk, 0, 1, 0) // (B * H * Tq * (D + 2) * 4))
        blocks = B * H * -(-Tq // 64)
        assert parts == 1 or parts * blocks <= 1024, (B, Tq, Tk, parts)
