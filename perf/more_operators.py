"""Measured calls of the 8-bit key-value cache and of attention over a shared prefix.

Each case is what a serving program does in one step of its kind:

* ``append``: norms, rotation and quantisation of the newest tokens into the cache's
  pages, and the sequences read back, as the next chunk of a prompt attends to them;
* ``write``: the same for keys and values that are cached as they are;
* ``read``: rows of sequences read back from their pages;
* ``paged``: attention of one new token of each sequence over 8-bit pages;
* ``shared``: the same for a batch whose sequences have their first keys in common, over
  pages of 16 or 8 bits.

What is held in 8 bits is returned as the values it stands for, by the read. Heads, head
dims and token counts are those of this repository's benchmark and tests (24 heads of
128 channels; 1000, 4100, 12133 or 32760 tokens) or generic ones.
"""

import math

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
CODES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}

_modules = {}


def _mod(name):
    if name not in _modules:
        import importlib
        entry = importlib.import_module("__graft_entry__")
        entry.load_package()
        _modules[name] = importlib.import_module(f"{entry.PKG_NAME}.{name}")
    return _modules[name]


# ------------------------------------------------------------------- cases
def _case(name, op, length, **kw):
    case = dict(name=name, op=op, B=1, length=length, page=64, H=24, Hkv=8, D=128, dtype="bf16", cache="fp8")
    if op in ("append", "write"):
        case.update(T=1, padded=False)
    if op == "append":
        case.update(R=128, interleaved=False)
    if op == "read":
        case.update(tokens=length)  # at most; the last of each sequence
    if op == "paged":
        case.update(window=0, sinks=0, idle=False)
    if op == "shared":
        case.update(groups=1, prefix=length, cache="same", idle=False)  # length: the prefix and the longest rest
    case.update(kw)
    return case


def listed():
    return [
        # One decode step of four sequences: the newest token's norms, rotation and
        # codes, and the short sequences read back. Launches and latency only.
        _case("append_step_4", "append", 100, B=4, T=1),
        # A 16K-token prompt into an empty cache of whole numbers, and back as its
        # attention reads it.
        _case("append_prompt_16k", "append", 16001, T=16001, interleaved=True, cache="int8"),
        # One chunk of two ragged prompts, no norms, heads of 64 channels, small pages.
        _case("write_chunk_1000", "write", 4100, B=2, T=1000, H=16, Hkv=4, D=64, page=16, dtype="fp16", cache="int8",
              padded=True),
        # A packed video's keys and values of 24 heads, cached once for every step.
        _case("write_video_12k", "write", 12133, T=12133, Hkv=24),
        # The last 1333 keys of eight ragged sequences, for a windowed chunk.
        _case("read_window_8", "read", 4100, B=8, tokens=1333, H=16, Hkv=4, D=64, page=16, dtype="fp16", cache="int8"),
        # Four long sequences whole.
        _case("read_long_32k", "read", 32760, B=4),
        # One new token of one sequence behind 60000, a window of 4096 and four sinks.
        _case("paged_window_1", "paged", 60000, window=4096, sinks=4),
        # One new token of each of 32 ragged sequences, small pages, an idle slot.
        _case("paged_batch_32", "paged", 16384, B=32, page=16, H=16, Hkv=4, D=64, idle=True, dtype="fp16", cache="int8"),
        # One new token of each of four long sequences.
        _case("paged_long_131k", "paged", 131072, B=4),
        # Eight answers to one 4100-token prompt, up to 300 tokens into them.
        _case("shared_8", "shared", 4400, B=8, prefix=4100),
        # Four prompts of 8000 tokens with sixteen answers each, 8-bit pages.
        _case("shared_groups_64", "shared", 8400, B=64, groups=4, prefix=8000, H=16, Hkv=4, D=64, page=16, dtype="fp16",
              cache="int8", idle=True),
        # A batch of 256 behind one 32K-token context, up to 500 tokens of their own.
        _case("shared_256", "shared", 33260, B=256, prefix=32760),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["append", "append", "write", "read", "paged", "paged", "paged", "shared", "shared", "shared", "shared"])
    H, group = rng.choice([(24, 1), (24, 3), (24, 3), (16, 4), (16, 4), (32, 8), (2 * rng.randint(1, 12), 2), (rng.randint(1, 24), 1)])
    D = rng.choice([128, 128, 128, 64, 64, 96, 80])
    kw = dict(H=H, Hkv=H // group, D=D, dtype=rng.choice(["bf16", "bf16", "fp16"]), page=rng.choice([16, 64, 64, 128]),
              cache=rng.choice(["fp8", "int8"]))
    if op in ("append", "write"):
        B = rng.randint(1, 16)
        length = _log_int(rng, 20, 16000 // B)
        T = min(length, _log_int(rng, 1, 16000))
        case = _case("", op, length, B=B, T=T, padded=rng.random() < 0.3, **kw)
        if op == "append":
            case.update(R=rng.choice([D, D, 16 * (D // 32)]), interleaved=rng.choice([False, True]))
    elif op == "read":
        B = rng.randint(1, 16)
        length = _log_int(rng, 20, 65000 // B)
        case = _case("", op, length, B=B, tokens=rng.choice([length, _log_int(rng, 1, length)]), **kw)
    elif op == "paged":
        B = _log_int(rng, 1, 64)
        case = _case("", op, _log_int(rng, 30, min(131072, 500000 // B)), B=B, **kw)
        if rng.random() < 0.4:
            case.update(window=_log_int(rng, 16, 8192), sinks=rng.choice([0, 4, 100]))
        case["idle"] = B > 1 and rng.random() < 0.3
    else:
        groups = rng.choice([1, 1, 1, 2, 3, 8])
        B = groups * _log_int(rng, 2, 256 // groups)
        prefix = _log_int(rng, 100, min(32760, 256 * 24 * 32760 // (B * H)))
        rest = _log_int(rng, 1, min(2000, 128000 // B))
        case = _case("", op, prefix + rest, B=B, groups=groups, prefix=prefix, idle=rng.random() < 0.3, **kw)
        case["cache"] = rng.choice(["same", "same", "fp8", "int8"])
    del case["name"]
    return case


# ------------------------------------------------------------------ inputs
def _lengths(case):
    """Tokens of each sequence, before the seed deals them out (within a group, where a prefix is shared)."""
    B, L = case["B"], case["length"]
    if case["op"] == "shared":
        per = B // case["groups"]
        n = [case["prefix"] + max(1, (L - case["prefix"]) * (b % per + 1) // per) for b in range(B)]
        if case["idle"]:
            n[0] = 0
        return n
    if case["op"] in ("append", "write"):
        return [max(case["T"], L - b * L // 3) if case["padded"] else L for b in range(B)] if B < 4 else \
            [max(case["T"], L * (b + 1) // B) if case["padded"] else L for b in range(B)]
    n = [max(1, L * (b + 1) // B) for b in range(B)]
    if case.get("idle"):
        n[0] = 0
    return n


def _tables(case, dev):
    """cos and sin of every position and frequency, fp32, from angles in 64 bits."""
    R = case["R"]
    freq = 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64, device=dev) / R)
    angle = torch.arange(max(_lengths(case)), dtype=torch.float64, device=dev)[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def _encode(x, kind):
    """(codes, scales) of the rows of x (fp32): the power of two that keeps the last dim's largest
    value within 127 or 448, as its exponent's byte; rows of next to nothing are zeros."""
    top = x.abs().amax(-1, keepdim=True)
    none = top < 2.0 ** -110
    m, e = torch.frexp(top / (127.0 if kind == "int8" else 448.0))
    e = (e - (m == 0.5).to(e.dtype)).masked_fill_(none, 0)
    codes = torch.ldexp(x, -e).masked_fill_(none, 0.0)
    codes = codes.round_().to(torch.int8) if kind == "int8" else codes.to(torch.float8_e4m3fn)
    return codes, (e + 127).masked_fill_(none, 0).to(torch.uint8)[..., 0].view(torch.float8_e8m0fnu)


def _power(scale):
    """The powers of two that exponent bytes stand for, in 32 bits."""
    return (scale.view(torch.uint8).to(torch.int32) << 23).view(torch.float32)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = TYPES[case["dtype"]]
    op, H, Hkv, D, B, page = (case[n] for n in ("op", "H", "Hkv", "D", "B", "page"))
    most = -(-case["length"] // page)
    groups = case.get("groups", 1)
    per = B // groups
    n = torch.tensor(_lengths(case), dtype=torch.int32, device=dev).reshape(groups, per)
    order = torch.stack([torch.randperm(per, generator=gen, device=dev) for _ in range(groups)])
    n = n.gather(1, order).reshape(B)
    # page ids of every sequence, scattered over the cache; -1 behind a sequence's last page
    ids = torch.randperm(B * most, generator=gen, device=dev).to(torch.int32).reshape(B, most)
    whole = case["prefix"] // page if op == "shared" else 0
    if whole:  # the prefix's whole pages are the same for a group
        ids[:, :whole] = ids[::per, :whole].repeat_interleave(per, 0)
        used, ids = torch.unique(ids, return_inverse=True)
        pages, ids = used.numel(), ids.to(torch.int32)
    else:
        pages = B * most
    table = torch.where(torch.arange(most, device=dev) * page < n[:, None], ids, torch.full_like(ids, -1))
    s = dict(case=case, lengths=n, table=table.contiguous())

    def cache(shift):
        """Pages of unit rows with the outlier channels of trained projections."""
        wide = (1 + 4 * (torch.rand(Hkv, D, generator=gen, device=dev) < 0.02)).float()
        x = torch.randn(pages, page, Hkv, D, generator=gen, device=dev).mul_(wide)
        if shift is not None:
            x += shift
        if whole and case["prefix"] % page:  # a page that the prefix ends in: each sequence has its own copy
            last, rows = ids[:, whole].long(), case["prefix"] % page
            x[last, :rows] = x[last[::per], :rows].repeat_interleave(per, 0)
        if case["cache"] == "same":
            return x.to(dt), None
        codes, scale = _encode(x.to(dt).float(), case["cache"])
        return codes, scale.view(torch.uint8).transpose(1, 2).contiguous().view(scale.dtype)

    if op in ("append", "write"):
        T = case["T"]
        # one projection's output, q k and v side by side; outlier channels
        qkv = torch.randn(B, T, (H + 2 * Hkv) * D, generator=gen, device=dev)
        qkv = (qkv * (1 + 4 * (torch.rand((H + 2 * Hkv) * D, generator=gen, device=dev) < 0.02))).to(dt)
        q, k, v = qkv.split([H * D, Hkv * D, Hkv * D], dim=-1)
        s.update(k=k.unflatten(-1, (Hkv, D)), v=v.unflatten(-1, (Hkv, D)), tokens=case["length"])
        if op == "append":
            s.update(q=q.unflatten(-1, (H, D)), qw=1 + 0.2 * torch.randn(D, generator=gen, device=dev),
                     kw=1 + 0.2 * torch.randn(D, generator=gen, device=dev))
            s["cos"], s["sin"] = _tables(case, dev)
    if op in ("paged", "shared"):
        toward = torch.randn(H, D, generator=gen, device=dev)
        s["q"] = (torch.randn(B, 1, H, D, generator=gen, device=dev) * 1.2 + 0.3 * toward).to(dt)
        s["k"], s["k_scale"] = cache(0.2 * toward[::H // Hkv])
        s["v"], s["v_scale"] = cache(None)
    else:
        s["k_cache"], s["k_scale"] = cache(None)
        s["v_cache"], s["v_scale"] = cache(None)
    if op == "read":
        s["tokens"] = case["tokens"]
        s["start"] = (n - case["tokens"]).clamp_min(0)
    return s


# ------------------------------------------------------------- plain forms
def _norm_turn(x, w, cos, sin, interleaved):
    """x / rms(x) * w in 32 bits, the pairs of its first channels turned; cos, sin: [B, T, 1, R/2]."""
    x = x.float()
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w
    R = 2 * cos.shape[-1]
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if interleaved else (x[..., :R // 2], x[..., R // 2:R])
    u, v = a * cos - b * sin, b * cos + a * sin
    head = torch.stack([u, v], -1).flatten(-2) if interleaved else torch.cat([u, v], -1)
    return torch.cat([head, x[..., R:]], -1)


def _put(s, x, name):
    """Rows x [B, T, Hkv, D] (fp32) into the newest slots."""
    c = s["case"]
    at = s["lengths"].long()[:, None] - c["T"] + torch.arange(c["T"], device=x.device)
    page, slot = s["table"].long().gather(1, at // c["page"]), at % c["page"]
    codes, scale = _encode(x, c["cache"])
    s[name + "_cache"].view(torch.uint8)[page, slot] = codes.view(torch.uint8)
    s[name + "_scale"].view(torch.uint8).transpose(1, 2)[page, slot] = scale.view(torch.uint8)


def _get(s, name):
    """[B, tokens, Hkv, D] of the cache from ``start`` (or 0) on, zeros past a sequence's end."""
    c, n = s["case"], s["lengths"].long()
    at = torch.arange(s["tokens"], device=n.device) + (s["start"].long()[:, None] if "start" in s else 0)
    at = at.expand(c["B"], -1)
    on = at < n[:, None]
    page = s["table"].long().gather(1, torch.where(on, at // c["page"], torch.zeros_like(at))).clamp_min(0)
    slot = at % c["page"]
    codes = s[name + "_cache"].view(torch.uint8)[page, slot].view(CODES[c["cache"]]).float()
    x = codes * _power(s[name + "_scale"]).transpose(1, 2)[page, slot][..., None]
    return x.masked_fill_(~on[:, :, None, None], 0.0).to(TYPES[c["dtype"]])


def _plain_append(s):
    c = s["case"]
    at = s["lengths"].long()[:, None] - c["T"] + torch.arange(c["T"], device=s["q"].device)
    cos, sin = s["cos"][at][:, :, None], s["sin"][at][:, :, None]
    q = _norm_turn(s["q"], s["qw"], cos, sin, c["interleaved"]).to(s["q"].dtype)
    _put(s, _norm_turn(s["k"], s["kw"], cos, sin, c["interleaved"]), "k")
    _put(s, s["v"].float(), "v")
    return q, _get(s, "k"), _get(s, "v")


def _plain_write(s):
    _put(s, s["k"].float(), "k")
    _put(s, s["v"].float(), "v")
    return _get(s, "k"), _get(s, "v")


def _plain_read(s):
    return _get(s, "k"), _get(s, "v")


def _values(s, name, at):
    """Pages ``at`` [N, pages] of the cache as fp32 [N, Hkv, keys, D]."""
    x = s[name]
    x = x.view(torch.uint8)[at].view(x.dtype).float() if s[name + "_scale"] is not None else x[at].float()
    x = x.flatten(1, 2).transpose(1, 2)
    return x if s[name + "_scale"] is None else x * _power(s[name + "_scale"].view(torch.uint8)[at]).transpose(1, 2).flatten(2)[..., None]


def _softmax(x):
    top = x.amax(-1, keepdim=True)
    p = x.sub_(top.masked_fill_(top == float("-inf"), 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    return p, total.masked_fill_(total == 0.0, 1.0)


def _plain_paged(s):
    c, n = s["case"], s["lengths"]
    B, Hkv, D = c["B"], c["Hkv"], c["D"]
    at = s["table"].clamp_min(0).long()
    k, v = _values(s, "k", at), _values(s, "v", at)
    x = s["q"].float().reshape(B, Hkv, -1, D).mul(D ** -0.5) @ k.transpose(-1, -2)
    j = torch.arange(x.shape[-1], device=x.device)
    on = j < n[:, None]
    if c["window"]:
        on = on & ((j >= n[:, None] - c["window"]) | (j < c["sinks"]))
    p, total = _softmax(x.masked_fill_(~on[:, None, None], float("-inf")))
    return (p @ v / total).reshape(B, 1, c["H"], D).to(s["q"].dtype)


def _plain_shared(s):
    """The prefix's keys once for the rows of a group, the others' behind them."""
    c, n = s["case"], s["lengths"]
    B, G, Hkv, D, page, prefix = (c[x] for x in ("B", "groups", "Hkv", "D", "page", "prefix"))
    per = B // G
    longest = n.reshape(G, per).argmax(1) + torch.arange(G, device=n.device) * per
    whole = -(-prefix // page)
    at = s["table"][longest, :whole].clamp_min(0).long()
    first = prefix // page
    rest = s["table"][:, first:].clamp_min(0).long()
    q = s["q"].float().reshape(G, per, Hkv, -1, D).mul(D ** -0.5)
    group = q.shape[3]
    k = _values(s, "k", at)[:, :, :prefix]
    x = (q.transpose(1, 2).reshape(G, Hkv, per * group, D) @ k.transpose(-1, -2)).reshape(G, Hkv, per, group, prefix)
    x = x.transpose(1, 2).reshape(B, Hkv, group, prefix)
    y = q.reshape(B, Hkv, group, D) @ _values(s, "k", rest).transpose(-1, -2)
    j = torch.arange(prefix, device=n.device)
    x.masked_fill_(~(j < n[:, None])[:, None, None], float("-inf"))
    j = first * page + torch.arange(y.shape[-1], device=n.device)
    y.masked_fill_(~((j < n[:, None]) & (j >= prefix))[:, None, None], float("-inf"))
    p, total = _softmax(torch.cat([x, y], -1))
    v = _values(s, "v", at)[:, :, :prefix]
    px = p[..., :prefix].reshape(G, per, Hkv, group, prefix).transpose(1, 2).reshape(G, Hkv, per * group, prefix)
    o = (px @ v).reshape(G, Hkv, per, group, D).transpose(1, 2).reshape(B, Hkv, group, D)
    o = o + p[..., prefix:] @ _values(s, "v", rest)
    return (o / total).reshape(B, 1, c["H"], D).to(s["q"].dtype)


# ------------------------------------------------------- the framework's calls
def _own_get(s):
    return _mod("_cache").cache_read(s["k_cache"], s["v_cache"], s["table"], s["lengths"], s["k_scale"], s["v_scale"],
                                     tokens=s["tokens"], start=s.get("start"), dtype=TYPES[s["case"]["dtype"]])


def _own_append(s):
    q = _mod("_qk_rope").qk_norm_rope_append(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["lengths"],
                                             s["qw"], s["kw"], s["cos"], s["sin"], interleaved=s["case"]["interleaved"],
                                             k_scale=s["k_scale"], v_scale=s["v_scale"])
    return q, *_own_get(s)


def _own_write(s):
    _mod("_cache").cache_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["lengths"], s["k_scale"],
                                s["v_scale"])
    return _own_get(s)


def _own_paged(s):
    c = s["case"]
    return _mod("_paged").paged_attn(s["q"], s["k"], s["v"], s["table"], s["lengths"], window=c["window"] or None,
                                     sinks=c["sinks"], k_scale=s["k_scale"], v_scale=s["v_scale"])


def _own_shared(s):
    c = s["case"]
    return _mod("_paged").paged_attn(s["q"], s["k"], s["v"], s["table"], s["lengths"], k_scale=s["k_scale"],
                                     v_scale=s["v_scale"], shared=c["prefix"], groups=c["groups"])


def run(state):
    op = state["case"]["op"]
    if own:
        return {"append": _own_append, "write": _own_write, "read": _own_get, "paged": _own_paged, "shared": _own_shared}[op](state)
    return {"append": _plain_append, "write": _plain_write, "read": _plain_read, "paged": _plain_paged,
            "shared": _plain_shared}[op](state)


# -------------------------------------------------------------------- work
def work(case):
    op, B, H, Hkv, D = (case[n] for n in ("op", "B", "H", "Hkv", "D"))
    row = 2 * D if case["cache"] == "same" else D + 1  # bytes of a row in the cache
    n = np.array(_lengths(case), dtype=np.int64)
    if op in ("append", "write", "read"):
        tokens = case["tokens"] if op == "read" else case["length"]
        out = 2 * 2 * B * tokens * Hkv * D
        if op == "read":
            read = int(np.minimum(n, tokens).sum())
            return {"bytes": 2 * read * Hkv * row + out, "flops": 2 * read * Hkv * D}
        # rows that were there are read, the new ones read in 16 bits and written in 8
        new, old = B * case["T"], int((n - case["T"]).sum())
        moved = 2 * new * Hkv * (2 * D + row) + 2 * old * Hkv * row + out
        values = 2 * new * Hkv * D
        if op == "append":
            moved += 2 * 2 * new * H * D + 4 * case["R"] * new
            values += new * H * D
        return {"bytes": moved, "flops": 8 * values}
    if op == "paged":
        if case["window"]:
            low = np.maximum(n - case["window"], 0)
            n = n - low + np.minimum(low, case["sinks"])
        keys = pairs = int(n.sum())
    else:
        per = B // case["groups"]
        pairs = int(n.sum())
        keys = int(np.maximum(n - case["prefix"], 0).sum() + np.minimum(n, case["prefix"]).reshape(-1, per).max(1).sum())
    return {"bytes": 2 * keys * Hkv * row + 2 * 2 * B * H * D, "flops": 4 * D * H * pairs}


# ------------------------------------------------------------------- exact
def _exact_rows(x, kind):
    """What the cache keeps of the rows x [..., D] (64 bits)."""
    top = x.abs().max(-1, keepdim=True).values
    safe = top.clamp_min(2.0 ** -110)
    s = torch.exp2(torch.ceil(torch.log2(safe / (127 if kind == "int8" else 448))))
    y = x / s
    if kind == "int8":
        kept = torch.round(y) * s
    else:  # three bits behind the leading one, none below 2^-9
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -30))).clamp_min(-6) - 3)
        kept = torch.round(y / step) * step * s
    return torch.where(top < 2.0 ** -110, torch.zeros_like(kept), kept)


def _exact_old(s, name, ids):
    """Pages ``ids`` of the cache as [keys, Hkv, D] in 64 bits."""
    x = s[name][ids].double().flatten(0, 1) if s[name].element_size() > 1 else \
        s[name].view(torch.uint8)[ids].view(s[name].dtype).float().double().flatten(0, 1)
    scale = s[name.split("_")[0] + "_scale"]
    return x if scale is None else x * scale.view(torch.uint8)[ids].double().sub(127).exp2().transpose(1, 2).flatten(0, 1)[..., None]


def _exact_turn(x, w, cos, sin, interleaved):
    x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + 1e-6) * w
    half = cos.shape[-1]
    i = torch.arange(half, device=x.device)
    first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    z = torch.complex(x[..., first], x[..., second]) * torch.complex(cos, sin)
    y = x.clone()
    y[..., first], y[..., second] = z.real, z.imag
    return y


def exact(case, seed):
    s = prepare(case, seed)
    op, B, H, Hkv, D, page = (case[n] for n in ("op", "B", "H", "Hkv", "D", "page"))
    dev, n = s["lengths"].device, s["lengths"].tolist()
    if op in ("append", "write", "read"):
        new = {}
        if op != "read":
            new = {x: s[x].double() for x in "kv"}
        if op == "append":
            at = s["lengths"].long()[:, None] - case["T"] + torch.arange(case["T"], device=dev)
            cos, sin = s["cos"].double()[at].unsqueeze(2), s["sin"].double()[at].unsqueeze(2)
            q = _exact_turn(s["q"].double(), s["qw"].double(), cos, sin, case["interleaved"])
            new["k"] = _exact_turn(new["k"], s["kw"].double(), cos, sin, case["interleaved"])
        outs = []
        for name in "kv":
            out = torch.zeros(B, s["tokens"], Hkv, D, dtype=torch.float64, device=dev)
            for b in range(B):
                rows = _exact_old(s, name + "_cache", s["table"][b, :-(-n[b] // page)].long())[:n[b]]
                if new:
                    rows[n[b] - case["T"]:] = _exact_rows(new[name][b], case["cache"])
                if op == "read":
                    rows = rows[max(n[b] - s["tokens"], 0):]
                out[b, :len(rows)] = rows
            outs.append(out)
        return [q, *outs] if op == "append" else outs
    out = torch.zeros(B, 1, H, D, dtype=torch.float64, device=dev)
    for b in range(B):
        if not n[b]:
            continue
        ids = s["table"][b, :-(-n[b] // page)].long()
        keep = torch.arange(n[b], device=dev)
        if case.get("window"):
            keep = keep[(keep >= n[b] - case["window"]) | (keep < case["sinks"])]
        k, v = (_exact_old(s, x, ids)[keep].transpose(0, 1) for x in "kv")  # [Hkv, keys, D]
        q = s["q"][b, 0].double().reshape(Hkv, H // Hkv, D)
        a = torch.softmax(torch.matmul(q, k.transpose(1, 2)) / math.sqrt(D), -1)
        out[b, 0] = torch.matmul(a, v).reshape(H, D)
    return out
