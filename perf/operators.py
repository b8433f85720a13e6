"""Measured calls of the operators around attention: per-head norms with the
position rotation, sliding-window attention with sinks, and attention of one new
token over a paged cache.

Each case is one call that a program makes, or a training pass's call with its
gradients:

* ``rope``: norms and rotation of q and k, as in front of every attention call;
* ``rope_train``: the same with the gradients of q, k and both weights;
* ``append``: the same for the newest tokens, k and v going into a paged cache;
* ``window``: sliding-window attention with sinks;
* ``window_train``: the same with the gradients of q, k and v;
* ``paged``: attention of one new token of each sequence over its pages.

Both ``run`` and ``exact`` take what ``prepare`` gives. Heads, head dims and token
counts are those of this repository's benchmark and tests (24 heads of 128
channels; 1000, 4100, 12133 or 32760 tokens) or generic ones.
"""

import math

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _mod(name):
    import importlib
    entry = importlib.import_module("__graft_entry__")
    entry.load_package()
    return importlib.import_module(f"{entry.PKG_NAME}.{name}")


# ------------------------------------------------------------------- cases
def _rope(name, op, T, **kw):
    case = dict(name=name, op=op, B=1, T=T, H=24, Hkv=24, D=128, R=128, dtype="bf16", interleaved=False)
    case.update(kw)
    return case


def _window(name, op, T, window, **kw):
    case = dict(name=name, op=op, B=1, Tq=T, Tk=T, H=24, Hkv=24, D=128, window=window, sinks=4, causal=True,
                padded=False, dtype="bf16")
    case.update(kw)
    return case


def _paged(name, length, **kw):
    case = dict(name=name, op="paged", B=1, length=length, page=64, H=24, Hkv=8, D=128, window=0, sinks=0, idle=False,
                dtype="bf16")
    case.update(kw)
    return case


def listed():
    return [
        # One decode step of four sequences: the newest token's norms, rotation
        # and cache rows. Launches and latency only.
        _rope("append_step_4", "append", 1, B=4, Hkv=8, length=100, page=64),
        # q and k of a 32K-token video, views of one fused qkv projection,
        # rotated in interleaved pairs: the pass in front of the headline call.
        _rope("rope_video_32k", "rope", 32760, interleaved=True),
        # A training pass's norms: batch 2, heads of 64 channels, shared kv
        # heads, the rotation on half of the channels.
        _rope("rope_train_4k", "rope_train", 4100, B=2, H=16, Hkv=4, D=64, R=32, dtype="fp16"),
        # The smallest windowed call worth making: 300 tokens, two heads.
        _window("window_300", "window", 300, 64, H=2, Hkv=1),
        # A 16K-token prompt with a 4096-token window and four sinks, shared kv heads.
        _window("window_prompt_16k", "window", 16001, 4096, Hkv=8),
        # A packed video: 1333 conditioning rows that every row sees, a window
        # of two 30x40 frames to either side.
        _window("window_video_12k", "window", 12133, 2401, sinks=1333, causal=False),
        # One chunk of a padded batch's prompts against the keys so far.
        _window("window_chunk_517", "window", 0, 8192, B=2, Tq=517, Tk=16000, H=16, Hkv=4, D=64, padded=True,
                dtype="fp16"),
        # Gradients of a short training batch, heads of 64 channels.
        _window("window_train_2k", "window_train", 2000, 512, B=2, H=16, Hkv=16, D=64),
        # Gradients of a long training sequence, shared kv heads.
        _window("window_train_8k", "window_train", 8192, 1024, Hkv=8),
        # One new token of one sequence behind 60000, of which a window of 4096
        # and four sinks are visible.
        _paged("paged_window_1", 60000, window=4096, sinks=4),
        # One new token of each of 32 sequences of ragged lengths, small pages,
        # an idle slot among them.
        _paged("paged_batch_32", 16384, B=32, page=16, H=16, Hkv=4, D=64, idle=True, dtype="fp16"),
        # One new token of each of four long sequences.
        _paged("paged_long_131k", 131072, B=4),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["rope", "rope", "rope_train", "append", "window", "window", "window_train", "window_train", "paged",
                     "paged"])
    H, group = rng.choice([(24, 1), (24, 3), (16, 4), (16, 1), (8, 8), (2 * rng.randint(1, 12), 2), (rng.randint(1, 24), 1)])
    D = rng.choice([128, 128, 128, 64, 64, 96, 80])
    heads = dict(H=H, Hkv=H // group, D=D, dtype=rng.choice(["bf16", "bf16", "fp16"]))
    if op in ("rope", "rope_train", "append"):
        pairs = rng.choice([False, True])
        kw = dict(heads, R=rng.choice([D, D, 16 * (D // 32)]), interleaved=pairs)
        if op == "append":
            length = _log_int(rng, 20, 4000)
            case = _rope("", op, min(length, _log_int(rng, 1, 500)), B=rng.randint(1, 16), length=length,
                         page=rng.choice([16, 64, 128]), **kw)
        else:
            case = _rope("", op, _log_int(rng, 1, 32760 if op == "rope" else 8000), B=rng.choice([1, 1, 2]), **kw)
            if case["B"] * case["T"] > 32760:
                case["B"] = 1
            if rng.random() < 0.2:
                case["dtype"] = "fp32"
    elif op == "paged":
        case = _paged("", _log_int(rng, 30, 60000), B=_log_int(rng, 1, 48), page=rng.choice([16, 64, 64, 256]), **heads)
        case["length"] = min(case["length"], 500000 // case["B"])
        if rng.random() < 0.4:
            case.update(window=_log_int(rng, 16, 8192), sinks=rng.choice([0, 4, 100]))
        case["idle"] = case["B"] > 1 and rng.random() < 0.3
    else:
        train = op == "window_train"
        B, Tk = rng.choice([1, 1, 2]), _log_int(rng, 40, 8000 if train else 16000)
        Tq = _log_int(rng, 1, Tk) if rng.random() < 0.3 else Tk
        if B * H * Tk > 24 * 8000:  # no more than the largest listed case of its kind
            B, Tk = 1, min(Tk, 24 * 8000 // H)
            Tq = min(Tq, Tk)
        case = _window("", op, 0, _log_int(rng, 16, 6000), B=B, Tq=Tq, Tk=Tk, sinks=rng.choice([0, 1, 4, 64, 300]),
                       causal=rng.random() < 0.7, padded=B > 1 and rng.random() < 0.5, **heads)
    del case["name"]
    return case


# ------------------------------------------------------------------ inputs
def _lengths(case):
    """Tokens of each sequence, before the seed deals them out: ragged, the longest ``length`` long."""
    B = case["B"]
    if case["op"] == "append":
        return [max(case["T"], case["length"] * (b + 1) // B) for b in range(B)]
    if case["op"] == "paged":
        n = [max(1, case["length"] * (b + 1) // B) for b in range(B)]
        if case["idle"]:
            n[0] = 0
        return n
    return [max(1, case["Tk"] - b * case["Tk"] // 3) for b in range(B)] if case["padded"] else [case["Tk"]] * B


def _tables(case, dev):
    """cos and sin of every position and frequency, fp32, from angles in 64 bits."""
    n = max(1, max(_lengths(case)) if case["op"] == "append" else case["T"])
    R = case["R"]
    freq = 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64, device=dev) / R)
    angle = torch.arange(n, dtype=torch.float64, device=dev)[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = TYPES[case["dtype"]]
    H, Hkv, D, B = case["H"], case["Hkv"], case["D"], case["B"]

    def rand(*shape, scale=1.0):
        return torch.randn(*shape, generator=gen, device=dev).mul_(scale).to(dt)

    def lengths():
        n = torch.tensor(_lengths(case), dtype=torch.int32, device=dev)
        return n[torch.randperm(B, generator=gen, device=dev)].contiguous()

    def pages(n, page):
        """Page ids of every sequence, scattered over the cache; -1 behind a sequence's last page."""
        most = max(1, -(-max(_lengths(case)) // page))
        ids = torch.randperm(B * most, generator=gen, device=dev).to(torch.int32).reshape(B, most)
        used = torch.arange(most, device=dev) * page < n[:, None]
        return torch.where(used, ids, torch.full_like(ids, -1)), B * most

    s = dict(case=case)
    if case["op"] in ("rope", "rope_train", "append"):
        T = case["T"]
        # one projection's output, q k and v side by side; outlier channels as trained projections have
        qkv = rand(B, T, (H + 2 * Hkv) * D) * (1 + 4 * (torch.rand((H + 2 * Hkv) * D, generator=gen, device=dev) < 0.02)).to(dt)
        q, k, v = qkv.split([H * D, Hkv * D, Hkv * D], dim=-1)
        s.update(q=q.unflatten(-1, (H, D)), k=k.unflatten(-1, (Hkv, D)), v=v.unflatten(-1, (Hkv, D)),
                 qw=1 + 0.2 * torch.randn(D, generator=gen, device=dev), kw=1 + 0.2 * torch.randn(D, generator=gen, device=dev))
        s["cos"], s["sin"] = _tables(case, dev)
        if case["op"] == "rope_train":
            for n in ("q", "k", "qw", "kw"):
                s[n] = s[n].detach().requires_grad_(True)
            s.update(dq=rand(B, T, H, D), dk=rand(B, T, Hkv, D))
        if case["op"] == "append":
            s["lengths"] = lengths()
            s["table"], n = pages(s["lengths"], case["page"])
            s.update(k_cache=rand(n, case["page"], Hkv, D), v_cache=rand(n, case["page"], Hkv, D))
        return s
    # normalised and rotated rows: unit variance, queries with a direction that the sink keys share
    toward = torch.randn(1, 1, H, D, generator=gen, device=dev)
    if case["op"] == "paged":
        s["lengths"] = lengths()
        s["table"], n = pages(s["lengths"], case["page"])
        s.update(q=(torch.randn(B, 1, H, D, generator=gen, device=dev) * 1.5 + 0.3 * toward).to(dt),
                 k=rand(n, case["page"], Hkv, D), v=rand(n, case["page"], Hkv, D))
        return s
    Tq, Tk = case["Tq"], case["Tk"]
    q = (torch.randn(B, Tq, H, D, generator=gen, device=dev) * 1.5 + 0.3 * toward).to(dt)
    k, v = rand(B, Tk, Hkv, D), rand(B, Tk, Hkv, D)
    few = min(case["sinks"], 4)
    k[:, :few] += 0.3 * toward[:, :, ::H // Hkv].to(dt)
    s.update(q=q, k=k, v=v, lengths=lengths() if case["padded"] else None)
    if case["op"] == "window_train":
        for n in ("q", "k", "v"):
            s[n].requires_grad_(True)
        s["do"] = rand(B, Tq, H, D)
    return s


# ------------------------------------------------------------- plain forms
def _norm(x, w, eps=1e-6):
    """(x / rms(x) in 32 bits, 1 / rms(x))"""
    x = x.float()
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)
    return x * r * w, r


def _turn(x, cos, sin, interleaved):
    """The pairs of the first channels turned by their angles; cos, sin: [B or 1, T, 1, R/2]."""
    R = 2 * cos.shape[-1]
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if interleaved else (x[..., :R // 2], x[..., R // 2:R])
    u, w = a * cos - b * sin, b * cos + a * sin
    head = torch.stack([u, w], -1).flatten(-2) if interleaved else torch.cat([u, w], -1)
    return torch.cat([head, x[..., R:]], -1)


def _plain_rope(s):
    c, T = s["case"], s["case"]["T"]
    cos, sin = s["cos"][None, :T, None], s["sin"][None, :T, None]
    q, k = s["q"].detach(), s["k"].detach()
    return [_turn(_norm(x, w.detach())[0], cos, sin, c["interleaved"]).to(x.dtype) for x, w in ((q, s["qw"]), (k, s["kw"]))]


def _plain_rope_grad(x, w, dy, cos, sin, interleaved):
    x, w, dy = x.detach().float(), w.detach(), dy.float()
    g = _turn(dy, cos, -sin, interleaved)
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
    u = g * w
    return r * (u - x * (r * r * (u * x).mean(-1, keepdim=True))), (g * x * r).sum((0, 1, 2))


def _plain_rope_train(s):
    c, T = s["case"], s["case"]["T"]
    cos, sin = s["cos"][None, :T, None], s["sin"][None, :T, None]
    dq, dqw = _plain_rope_grad(s["q"], s["qw"], s["dq"], cos, sin, c["interleaved"])
    dk, dkw = _plain_rope_grad(s["k"], s["kw"], s["dk"], cos, sin, c["interleaved"])
    return _plain_rope(s) + [dq.to(s["q"].dtype), dk.to(s["k"].dtype), dqw, dkw]


def _plain_append(s):
    c = s["case"]
    at = s["lengths"].long()[:, None] - c["T"] + torch.arange(c["T"], device=s["q"].device)  # [B, T]
    cos, sin = s["cos"][at][:, :, None], s["sin"][at][:, :, None]
    q, k = (_turn(_norm(x, w)[0], cos, sin, c["interleaved"]).to(x.dtype) for x, w in ((s["q"], s["qw"]), (s["k"], s["kw"])))
    page = s["table"].long().gather(1, at // c["page"])
    s["k_cache"][page, at % c["page"]] = k
    s["v_cache"][page, at % c["page"]] = s["v"]
    return q, s["k_cache"], s["v_cache"]


def _seen(c, lengths, dev):
    """[B or 1, Tq, Tk]: which keys each row sees."""
    p = c["Tk"] - c["Tq"] + torch.arange(c["Tq"], device=dev)[:, None]
    j = torch.arange(c["Tk"], device=dev)[None]
    near = (p - j < c["window"]) if c["causal"] else ((p - j).abs() < c["window"])
    on = near | (j < c["sinks"])
    if c["causal"]:
        on = on & (j <= p)
    on = on[None]
    if lengths is not None:
        n = lengths[:, None, None]
        on = on & (j < n) & (p < n)
    return on


def _plain_scores(s):
    """q, k, v [B, H, T, D] in 32 bits, the softmax weights [B, H, Tq, Tk] and the scale."""
    c = s["case"]
    q, k, v = (s[n].detach().float().transpose(1, 2) for n in "qkv")
    k, v = (t.repeat_interleave(c["H"] // c["Hkv"], 1) for t in (k, v))
    scale = c["D"] ** -0.5
    x = q.mul(scale) @ k.transpose(-1, -2)
    x.masked_fill_(~_seen(c, s["lengths"], x.device)[:, None], float("-inf"))
    top = x.amax(-1, keepdim=True)
    x.sub_(top.masked_fill_(top == float("-inf"), 0.0)).exp_()
    total = x.sum(-1, keepdim=True)
    x.div_(total.masked_fill_(total == 0.0, 1.0))
    return q, k, v, x, scale


def _plain_window(s):
    _, _, v, p, _ = _plain_scores(s)
    return (p @ v).transpose(1, 2).to(s["q"].dtype)


def _plain_window_train(s):
    c = s["case"]
    q, k, v, p, scale = _plain_scores(s)
    o, do = p @ v, s["do"].float().transpose(1, 2)
    dv = p.transpose(-1, -2) @ do
    ds = (do @ v.transpose(-1, -2)).sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq, dk = ds @ k, ds.transpose(-1, -2) @ q
    dk, dv = (t.unflatten(1, (c["Hkv"], -1)).sum(2) for t in (dk, dv))
    return [t.transpose(1, 2).to(s["q"].dtype) for t in (o, dq, dk, dv)]


def _plain_paged(s):
    c, n = s["case"], s["lengths"]
    B, Hkv, D = c["B"], c["Hkv"], c["D"]
    at = s["table"].clamp_min(0).long()
    k, v = (s[x][at].flatten(1, 2).float().transpose(1, 2) for x in "kv")  # [B, Hkv, L, D]
    q = s["q"].float().reshape(B, Hkv, -1, D)
    x = q.mul(D ** -0.5) @ k.transpose(-1, -2)
    j = torch.arange(x.shape[-1], device=x.device)
    on = j < n[:, None]
    if c["window"]:
        on = on & ((j >= n[:, None] - c["window"]) | (j < c["sinks"]))
    x.masked_fill_(~on[:, None, None], float("-inf"))
    top = x.amax(-1, keepdim=True)
    p = (x - top.masked_fill(top == float("-inf"), 0.0)).exp()
    total = p.sum(-1, keepdim=True)
    o = p @ v / total.masked_fill(total == 0.0, 1.0)
    return o.reshape(B, 1, c["H"], D).to(s["q"].dtype)


# ------------------------------------------------------- the framework's calls
def _own_rope(s):
    return _mod("_qk_rope").qk_norm_rope(s["q"], s["k"], s["qw"], s["kw"], s["cos"], s["sin"],
                                         interleaved=s["case"]["interleaved"])


def _own_rope_train(s):
    out = _own_rope(s)
    return [*out, *torch.autograd.grad(out, (s["q"], s["k"], s["qw"], s["kw"]), (s["dq"], s["dk"]))]


def _own_append(s):
    q = _mod("_qk_rope").qk_norm_rope_append(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["lengths"],
                                             s["qw"], s["kw"], s["cos"], s["sin"], interleaved=s["case"]["interleaved"])
    return q, s["k_cache"], s["v_cache"]


def _own_window(s):
    c = s["case"]
    return _mod("_window").window_attn(s["q"], s["k"], s["v"], window=c["window"], sinks=c["sinks"], causal=c["causal"],
                                       lengths=s["lengths"])


def _own_window_train(s):
    o = _own_window(s)
    return [o, *torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])]


def _own_paged(s):
    c = s["case"]
    return _mod("_paged").paged_attn(s["q"], s["k"], s["v"], s["table"], s["lengths"], window=c["window"] or None,
                                     sinks=c["sinks"])


def run(state):
    op = state["case"]["op"]
    if own:
        return {"rope": _own_rope, "rope_train": _own_rope_train, "append": _own_append, "window": _own_window,
                "window_train": _own_window_train, "paged": _own_paged}[op](state)
    return {"rope": _plain_rope, "rope_train": _plain_rope_train, "append": _plain_append, "window": _plain_window,
            "window_train": _plain_window_train, "paged": _plain_paged}[op](state)


# -------------------------------------------------------------------- work
def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    B, H, Hkv, D = case["B"], case["H"], case["Hkv"], case["D"]
    if case["op"] in ("rope", "rope_train", "append"):
        T, R = case["T"], case["R"]
        values, table = B * T * (H + Hkv) * D, 4 * R * T * (B if case["op"] == "append" else 1)
        if case["op"] == "append":  # v's rows too
            return {"bytes": 2 * e * (values + B * T * Hkv * D) + table, "flops": 8 * values}
        if case["op"] == "rope":
            return {"bytes": 2 * e * values + table, "flops": 8 * values}
        return {"bytes": 4 * e * values + table, "flops": 24 * values}
    if case["op"] == "paged":
        n = np.array(_lengths(case), dtype=np.int64)
        if case["window"]:
            low = np.maximum(n - case["window"], 0)
            n = n - low + np.minimum(low, case["sinks"])
        keys = int(n.sum())
        return {"bytes": e * (2 * keys * Hkv * D + 2 * B * H * D), "flops": 4 * D * H * keys}
    Tq, Tk, w, sinks = case["Tq"], case["Tk"], case["window"], case["sinks"]
    p = Tk - Tq + np.arange(Tq, dtype=np.int64)
    pairs = keys = rows = 0
    for n in _lengths(case):
        i = p[p < n]
        first = np.maximum(i - w + 1, 0)
        last = np.minimum(i, n - 1) if case["causal"] else np.minimum(i + w - 1, n - 1)
        seen = last - first + 1 + np.minimum(np.minimum(sinks, n), first)
        if not case["causal"]:  # sinks behind the window
            seen += np.maximum(np.minimum(sinks, n) - (last + 1), 0)
        pairs += int(seen.sum())
        rows += len(i)
        if len(i):
            low = int(first.min())
            keys += int(last.max()) - low + 1 + min(low, sinks, n)
    moved = e * D * (2 * keys * Hkv + rows * H + B * Tq * H)  # k, v, q of the rows that see keys, o
    if case["op"] == "window":
        return {"bytes": moved, "flops": 4 * D * H * pairs}
    # do read, dq, dk and dv written; forward 4, backward 10 with the scores made again
    return {"bytes": moved + e * D * (rows * H + B * Tq * H + 2 * B * Tk * Hkv), "flops": 14 * D * H * pairs}


# ------------------------------------------------------------------- exact
def _exact_rope(x, w, cos, sin, interleaved):
    """x [..., D] in 64 bits; cos, sin [..., R/2] broadcast to it."""
    x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + 1e-6) * w
    half = cos.shape[-1]
    i = torch.arange(half, device=x.device)
    first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    z = torch.complex(x[..., first], x[..., second]) * torch.complex(cos, sin)
    y = x.clone()
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_attend(q, k, v, p, low, high, sinks, scale):
    """One head in 64 bits: row i, at position p[i], sees the keys j < high[i] with j >= low[i] or j < sinks."""
    j = torch.arange(k.shape[0], device=q.device)
    on = (j < high[:, None]) & ((j >= low[:, None]) | (j < sinks))
    s = (q @ k.T * scale).masked_fill(~on, float("-inf"))
    a = torch.softmax(s, -1)
    return torch.where(on.any(-1, keepdim=True), a, torch.zeros_like(a)) @ v


def exact(case, seed):
    s = prepare(case, seed)
    dev, op = s["q"].device, case["op"]
    if op in ("rope", "rope_train", "append"):
        names = ("q", "k", "qw", "kw")
        x = {n: s[n].detach().double() for n in names}
        cos, sin = s["cos"].double(), s["sin"].double()
        if op == "append":
            at = (s["lengths"].long()[:, None] - case["T"] + torch.arange(case["T"], device=dev))
            cos, sin = cos[at], sin[at]
        else:
            cos, sin = cos[None, :case["T"]], sin[None, :case["T"]]
        cos, sin = cos.unsqueeze(2), sin.unsqueeze(2)
        if op == "rope_train":
            for t in x.values():
                t.requires_grad_(True)
        y = [_exact_rope(x[a], x[w], cos, sin, case["interleaved"]) for a, w in (("q", "qw"), ("k", "kw"))]
        if op == "rope":
            return y
        if op == "rope_train":
            return [t.detach() for t in y] + list(torch.autograd.grad(y, [x[n] for n in names], (s["dq"].double(), s["dk"].double())))
        page = case["page"]
        caches = [s["k_cache"].double(), s["v_cache"].double()]
        for b in range(case["B"]):
            ids = s["table"][b, at[b] // page].long()
            caches[0][ids, at[b] % page] = y[1][b]
            caches[1][ids, at[b] % page] = s["v"][b].double()
        return y[0], *caches
    B, H, D = case["B"], case["H"], case["D"]
    group, scale = H // case["Hkv"], 1 / math.sqrt(D)
    if op == "paged":
        o = torch.zeros(B, 1, H, D, dtype=torch.float64, device=dev)
        for b, n in enumerate(s["lengths"].tolist()):
            if not n:
                continue
            ids = s["table"][b, :-(-n // case["page"])].long()
            k, v = (s[x][ids].flatten(0, 1)[:n].double() for x in "kv")
            last = torch.tensor([n - 1], device=dev)
            low = last + 1 - (case["window"] or n)
            for h in range(H):
                o[b, :, h] = _exact_attend(s["q"][b, :, h].double(), k[:, h // group], v[:, h // group], last, low, last + 1,
                                           case["sinks"], scale)
        return o
    Tq, Tk, train = case["Tq"], case["Tk"], op == "window_train"
    outs = [torch.zeros(s[n].shape, dtype=torch.float64, device=dev) for n in "qqkv"]
    p = Tk - Tq + torch.arange(Tq, device=dev)
    for b in range(B):
        n = int(s["lengths"][b]) if s["lengths"] is not None else Tk
        low = p - case["window"] + 1
        if case["causal"]:
            high, sinks = torch.minimum(p + 1, torch.full_like(p, n)), case["sinks"]
        else:  # the sinks behind a row's window are its own case
            high, sinks = torch.minimum(p + case["window"], torch.full_like(p, n)), case["sinks"]
        high = torch.where(p < n, high, torch.zeros_like(high))
        for h in range(H):
            q, k, v = s["q"][b, :, h].detach().double(), s["k"][b, :, h // group].detach().double(), s["v"][b, :, h // group].detach().double()
            if train:
                for t in (q, k, v):
                    t.requires_grad_(True)
            if case["causal"]:
                o = _exact_attend(q, k, v, p, low, high, sinks, scale)
            else:
                j = torch.arange(Tk, device=dev)
                on = ((j >= low[:, None]) & (j < high[:, None])) | ((j < min(sinks, n)) & (p < n)[:, None])
                a = torch.softmax((q @ k.T * scale).masked_fill(~on, float("-inf")), -1)
                o = torch.where(on.any(-1, keepdim=True), a, torch.zeros_like(a)) @ v
            outs[0][b, :, h] = o.detach()
            if train:
                for out, g, hh in zip(outs[1:], torch.autograd.grad(o, (q, k, v), s["do"][b, :, h].double()), (h, h // group, h // group)):
                    out[b, :, hh] += g
    return outs if train else outs[0]
