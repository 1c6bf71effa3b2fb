"""Timed cases of the decoder-style attention path: rotary positions and attention with scored rules, both directions.

Rotary positions turn pairs of each head's values by angles that grow with the token's position (half or interleaved
pairs, part of the head or all of it, angles scaled for contexts longer than the trained one). Scored attention is
softmax attention over grouped key/value heads whose scores are capped by a tanh, get a bias that falls with distance,
and see only the keys that a causal, window, prefix or document rule leaves them; its backward gives dQ, dK and dV.

`kind` selects the operator, `grad` whether the backward runs too; the other entries are sizes and rules. The plain
forms below are elementary torch operations in 32 bits (angles in 64); `exact` computes the definition in 64 bits one
head at a time, with gradients by differentiation.
"""
import ctypes as C
import importlib
import math

import torch

own = False
DEV = "cuda"


# ------------------------------------------------------------------------------------------------------------- cases
def _attn(name, batch, heads, kv, lq, lk, dim, grad=True, causal=False, window=0, cap=0.0, slopes=False, docs=0,
          prefix=0):
    c = {"kind": "attn", "batch": batch, "heads": heads, "kv": kv, "lq": lq, "lk": lk, "dim": dim, "grad": grad,
         "causal": causal, "window": window, "cap": cap, "slopes": slopes, "docs": docs, "prefix": prefix}
    return dict(c, name=name) if name else c


def _rope(name, batch, seq, heads, dim, rot, layout, scaling, far, grad=True):
    c = {"kind": "rope", "batch": batch, "seq": seq, "heads": heads, "dim": dim, "rot": rot, "layout": layout,
         "scaling": scaling, "far": far, "grad": grad}
    return dict(c, name=name) if name else c


def listed():
    return [
        # the query and key heads of one new token for each of eight sequences, far into their contexts: latency
        _rope("rope_token", 8, 1, 16, 64, 64, "half", "linear", 100000, grad=False),
        # query and key heads of the MiniLM-sized encoder's batch (32 sequences of 128)
        _rope("rope_minilm", 32, 128, 24, 32, 32, "half", "plain", 0),
        # a long packed row whose positions restart with each document, part of each head turned, bands scaled
        _rope("rope_long", 2, 8192, 16, 128, 64, "interleaved", "bands", 65536),
        # one new token for each of eight padded sequences over cached keys, three query heads to a key head
        _attn("attn_token", 8, 12, 4, 1, 4096, 64, grad=False, cap=50.0, docs=1),
        # two short sentences: the smallest training call
        _attn("attn_small", 2, 4, 4, 17, 17, 32, causal=True),
        # the MiniLM-sized encoder's batch as a decoder
        _attn("attn_minilm", 32, 12, 12, 128, 128, 32, causal=True),
        # the BERT-base-sized batch, several documents packed in each row with padding behind them
        _attn("attn_bert_docs", 8, 12, 12, 512, 512, 64, docs=4),
        # a prefix that all see before a causal rest, capped scores, grouped heads of an odd width, odd lengths
        _attn("attn_prefix", 4, 8, 2, 777, 777, 80, causal=True, cap=50.0, prefix=200),
        # attention between sequences of different odd lengths with a distance bias
        _attn("attn_cross", 8, 8, 8, 77, 131, 40, slopes=True),
        # a chunk of new tokens behind a long context (inference)
        _attn("attn_chunk", 2, 12, 4, 500, 4596, 64, grad=False, causal=True),
        # a long causal row, capped, three query heads to a key head
        _attn("attn_long", 1, 12, 4, 4096, 4096, 64, causal=True, cap=30.0),
        # a long row with a sliding window and a distance bias, wide heads
        _attn("attn_window", 1, 16, 4, 8192, 8192, 128, causal=True, window=1024, slopes=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.3:
        dim = rng.choice([32, 40, 64, 80, 96, 128])
        rot = rng.choice([dim, dim, dim // 2, dim // 4])
        tokens = _log(rng, 1, 16384)
        seq = _log(rng, 1, tokens)
        return _rope(None, max(1, tokens // seq), seq, rng.choice([1, 2, 8, 12, 16, 24]), dim, rot - rot % 2,
                     rng.choice(["half", "interleaved"]), rng.choice(["plain", "linear", "ntk", "bands"]),
                     rng.choice([0, 1000, 100000, 1000000]), grad=rng.random() < 0.7)
    kv = rng.choice([1, 2, 4, 8, 12])
    heads = kv * rng.choice([1, 1, 2, 3, 4]) if kv < 8 else kv
    dim = rng.choice([32, 32, 40, 64, 64, 80, 96, 128])
    rule = dict(cap=rng.choice([0.0, 0.0, 20.0, 50.0]), slopes=rng.random() < 0.3, docs=rng.choice([0, 0, 1, 3, 6]))
    if rng.random() < 0.25:  # few new tokens over a context
        lq = rng.choice([1, 1, 1, 2, 5, 16, 60, 300])
        lk = lq + _log(rng, 1, 8192)
        return _attn(None, _log(rng, 1, 16), heads, kv, lq, lk, dim, grad=False, causal=True,
                     window=rng.choice([0, 0, 500]), **rule)
    lq = _log(rng, 2, 3000)
    batch = max(1, min(32, int(rng.uniform(0.2, 1.0) * 16000000 / (lq * lq * heads))))
    if rng.random() < 0.2:
        return _attn(None, batch, heads, kv, lq, max(1, int(lq * rng.uniform(0.4, 2.0))), dim, **rule)
    causal = rng.random() < 0.7
    prefix = rng.randint(1, lq) if causal and rng.random() < 0.3 else 0
    return _attn(None, batch, heads, kv, lq, lq, dim, causal=causal, prefix=prefix,
                 window=rng.choice([0, 0, max(1, lq // 3)]), **rule)


# ------------------------------------------------------------------------------------------------------------ inputs
BASE, TRAINED, FACTOR, LOW, HIGH = 10000.0, 4096.0, 8.0, 1.0, 32.0
AMPLITUDE = 0.1 * math.log(FACTOR) + 1.0


def _normal(gen, *shape, std=1.0):
    return torch.randn(shape, generator=gen, device=DEV).mul_(std)


def _documents(gen, batch, length, count):
    """Ids of `count` documents of about equal length packed in each row, -1 for the padding behind them."""
    jit = torch.rand(batch, count, generator=gen, device=DEV).mul_(0.6).add_(0.7)
    ends = (jit.cumsum(1) * (0.9 * length / count)).long().clamp_(1, length)
    at = torch.arange(length, device=DEV)
    ids = (at[None, :, None] >= ends[:, None, :]).sum(2)
    return torch.where(ids < count, ids, torch.full_like(ids, -1)).to(torch.int32).contiguous()


def _inputs(c, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed & ((1 << 63) - 1))
    s = {}
    if c["kind"] == "rope":
        b, n, h, d = c["batch"], c["seq"], c["heads"], c["dim"]
        s["x"] = _normal(gen, b * n, h * d)
        if c["grad"]:
            s["g"] = _normal(gen, b * n, h * d, std=1.0 / (b * n))
        start = torch.randint(0, c["far"] + 1, (b, 1), generator=gen, device=DEV)
        cut = torch.randint(1, n + 1, (b, 1), generator=gen, device=DEV)
        at = torch.arange(n, device=DEV)[None]
        s["pos"] = torch.where(at < cut, start + at, at - cut).to(torch.int32).reshape(-1).contiguous()
        return s
    b, h, kv, lq, lk, d = (c[k] for k in ("batch", "heads", "kv", "lq", "lk", "dim"))
    s["q"], s["k"], s["v"] = _normal(gen, b, lq, h, d, std=1.5), _normal(gen, b, lk, kv, d), _normal(gen, b, lk, kv, d)
    if c["grad"]:
        s["g"] = _normal(gen, b, lq, h, d, std=1.0 / (b * lq))
    if c["slopes"]:
        s["slopes"] = torch.exp2(-8.0 * torch.arange(1, h + 1, device=DEV, dtype=torch.float32) / h)
    if c["docs"]:
        s["kdoc"] = _documents(gen, b, lk, c["docs"])
        if lq == lk:
            s["qdoc"] = s["kdoc"]
        elif c["causal"] or c["docs"] == 1:  # new tokens belong to the first document of their row
            s["qdoc"] = torch.zeros(b, lq, device=DEV, dtype=torch.int32)
        else:
            s["qdoc"] = _documents(gen, b, lq, c["docs"])
    if c["prefix"]:
        s["prefix"] = torch.randint(c["prefix"] // 2, c["prefix"] + 1, (b,), generator=gen, device=DEV).to(torch.int32)
    return s


def prepare(case, seed):
    s = {"case": case, "in": _inputs(case, seed), "out": {}}
    # the buffers that a program hands to the library: outputs and what the forward leaves for the backward
    i, o = s["in"], s["out"]
    if case["kind"] == "rope":
        o["y"] = torch.empty_like(i["x"])
        if case["grad"]:
            o["dx"] = torch.empty_like(i["x"])
    else:
        o["o"] = torch.empty_like(i["q"])
        if case["grad"]:
            s["stats"] = torch.empty(2 * i["q"].numel() // case["dim"], device=DEV)
            o.update(dq=torch.empty_like(i["q"]), dk=torch.empty_like(i["k"]), dv=torch.empty_like(i["v"]))
    torch.cuda.synchronize()  # the inputs come from torch's stream, the library's calls run on its context's
    return s


# ------------------------------------------------------------------------------------------------------ plain forms
def _frequencies(c):
    """Turning speed of each pair in radians per position, and the amplitude, in 64 bits."""
    rot, scaling = c["rot"], c["scaling"]
    i = torch.arange(rot // 2, device=DEV, dtype=torch.float64)
    base = BASE * FACTOR ** (rot / max(rot - 2, 1)) if scaling == "ntk" else BASE
    f = torch.exp(i * (-2.0 * math.log(base) / rot))
    if scaling == "linear":
        f = f / FACTOR
    if scaling == "bands":  # pairs that turn often in the trained context keep their speed, slow ones are divided
        keep = ((f * (TRAINED / (2 * math.pi)) - LOW) / (HIGH - LOW)).clamp(0.0, 1.0)
        f = f * (keep + (1.0 - keep) / FACTOR)
    return f, AMPLITUDE if scaling == "bands" else 1.0


def _turn(c, x, cos, sin):
    h, d, rot = c["heads"], c["dim"], c["rot"]
    x = x.view(-1, h, d)
    y = x.clone()
    a, b = (x[..., :rot // 2], x[..., rot // 2:rot]) if c["layout"] == "half" else (x[..., 0:rot:2], x[..., 1:rot:2])
    u, v = a * cos - b * sin, b * cos + a * sin
    if c["layout"] == "half":
        y[..., :rot // 2], y[..., rot // 2:rot] = u, v
    else:
        y[..., 0:rot:2], y[..., 1:rot:2] = u, v
    return y.view(-1, h * d)


def _plain_rope(c, s):
    f, amp = _frequencies(c)
    angle = s["pos"].double()[:, None, None] * f
    cos, sin = (torch.cos(angle) * amp).float(), (torch.sin(angle) * amp).float()
    out = {"y": _turn(c, s["x"], cos, sin)}
    if c["grad"]:
        out["dx"] = _turn(c, s["g"], cos, -sin)
    return out


def _visible(c, s):
    """[B or 1, lq, lk] truth values: the keys each query sees."""
    lq, lk = c["lq"], c["lk"]
    i = torch.arange(lq, device=DEV)[:, None] + (lk - lq)  # the queries stand at the last lq of lk positions
    j = torch.arange(lk, device=DEV)[None, :]
    ok = torch.ones(1, lq, lk, device=DEV, dtype=torch.bool)
    if c["causal"]:
        ok = ok & (j <= i)
    if c["window"]:
        ok = ok & ((i - j).abs() < c["window"])
    if c["prefix"]:
        ok = ok | (j < s["prefix"].long()[:, None, None])
    if c["docs"]:
        qd, kd = s["qdoc"][:, :, None], s["kdoc"][:, None, :]
        ok = ok & (qd == kd) & (kd >= 0)
    return ok


def _plain_attn(c, s):
    b, h, kv, lq, lk, d = (c[k] for k in ("batch", "heads", "kv", "lq", "lk", "dim"))
    grp, scale = h // kv, 1.0 / math.sqrt(d)
    q = s["q"].permute(0, 2, 1, 3).contiguous()
    k, v = (s[n].permute(0, 2, 1, 3).repeat_interleave(grp, 1) for n in ("k", "v"))
    x = torch.matmul(q, k.transpose(2, 3).contiguous()) * scale
    if c["cap"]:
        t = torch.tanh(x / c["cap"])
        x = t * c["cap"]
    if c["slopes"]:
        dist = (torch.arange(lq, device=DEV)[:, None] + (lk - lq) - torch.arange(lk, device=DEV)[None, :]).abs()
        x = x - s["slopes"][:, None, None] * dist.float()
    ok = _visible(c, s)[:, None]
    x = torch.where(ok, x, torch.full_like(x[:1, :1, :1, :1], -math.inf))
    m = x.amax(3, keepdim=True)
    e = torch.exp(x - torch.where(m == -math.inf, torch.zeros_like(m), m))
    l = e.sum(3, keepdim=True)
    p = e / torch.where(l == 0, torch.ones_like(l), l)
    o = torch.matmul(p, v)
    out = {"o": o.permute(0, 2, 1, 3).contiguous()}
    if not c["grad"]:
        return out
    g = s["g"].permute(0, 2, 1, 3).contiguous()
    dv = torch.matmul(p.transpose(2, 3).contiguous(), g)
    dp = torch.matmul(g, v.transpose(2, 3).contiguous())
    ds = p * (dp - (g * o).sum(3, keepdim=True))
    if c["cap"]:
        ds = ds * (1.0 - t * t)
    dq = torch.matmul(ds, k) * scale
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), q) * scale
    out["dq"] = dq.permute(0, 2, 1, 3).contiguous()
    out["dk"], out["dv"] = (x.view(b, kv, grp, lk, d).sum(2).permute(0, 2, 1, 3).contiguous() for x in (dk, dv))
    return out


# ---------------------------------------------------------------------------------------------- the framework's calls
_LIB = None


def _ctx():
    """The package and one library context for the process, as a program keeps them."""
    global _LIB
    if _LIB is None:
        pkg = importlib.import_module("onemodel-csharp_amd")
        _LIB = pkg, pkg.Context(0)
    return _LIB


def _p(t):
    return C.c_void_p(t.data_ptr() if t is not None else None)


def _calls(state):
    """The library calls of one pass with their arguments bound."""
    pkg, ctx = _ctx()
    c, s, o, calls = state["case"], state["in"], state["out"], []

    def add(name, *args):
        calls.append((getattr(ctx.L, name), name, (ctx.h, *args)))

    if c["kind"] == "rope":
        h, d, rows, ld = c["heads"], c["dim"], c["batch"] * c["seq"], c["heads"] * c["dim"]
        r = pkg.om_rope()
        r.layout = ("half", "interleaved").index(c["layout"])
        r.scaling = ("plain", "linear", "ntk", "bands").index(c["scaling"])
        r.rot, r.base, r.factor, r.trained, r.low, r.high = c["rot"], BASE, FACTOR, TRAINED, LOW, HIGH
        r.amplitude = AMPLITUDE if c["scaling"] == "bands" else 1.0
        add("om_rope_fwd", _p(s["x"]), ld, _p(s["pos"]), 0, _p(o["y"]), ld, rows, c["seq"], h, d, C.byref(r))
        if c["grad"]:
            add("om_rope_bwd", _p(s["g"]), ld, _p(s["pos"]), 0, _p(o["dx"]), ld, rows, c["seq"], h, d, C.byref(r), 0)
        return ctx, calls
    b, h, kv, lq, lk, d = (c[k] for k in ("batch", "heads", "kv", "lq", "lk", "dim"))
    f = pkg.om_attention_scores()
    f.heads, f.kv_heads, f.scale, f.cap, f.causal, f.window = h, kv, 0.0, c["cap"], int(c["causal"]), c["window"]
    for field, name in (("slopes", "slopes"), ("q_doc", "qdoc"), ("k_doc", "kdoc"), ("prefix", "prefix")):
        setattr(f, field, s[name].data_ptr() if name in s else None)
    st = _p(state.get("stats"))
    ins = (_p(s["q"]), h * d, _p(s["k"]), _p(s["v"]), kv * d)
    add("om_attention_fwd_scored", *ins, _p(o["o"]), h * d, st, b, lq, lk, d, C.byref(f))
    if c["grad"]:
        add("om_attention_bwd_scored", *ins, _p(o["o"]), h * d, st, _p(s["g"]), h * d, _p(o["dq"]), h * d, _p(o["dk"]),
            _p(o["dv"]), kv * d, b, lq, lk, d, C.byref(f), 0)
    return ctx, calls


def run(state):
    if not own:
        return (_plain_rope if state["case"]["kind"] == "rope" else _plain_attn)(state["case"], state["in"])
    if "calls" not in state:
        state["calls"] = _calls(state)
    ctx, calls = state["calls"]
    for fn, name, args in calls:
        if fn(*args):
            raise RuntimeError("%s: %s" % (name, ctx.L.om_last_error(ctx.h).decode()))
    return state["out"]


# -------------------------------------------------------------------------------------------------------------- work
def _pairs(c):
    """Visible (query, key) pairs of one batch row; documents taken as equal."""
    lq, lk, total = c["lq"], c["lk"], 0
    n = c["docs"]
    size = 0.9 * lk / n if n else lk
    pre = 0.75 * c["prefix"]
    for i in range(lq):
        at = i + lk - lq
        lo, hi = 0, lk - 1
        if c["causal"]:
            hi = min(hi, at)
        if c["window"]:
            lo, hi = max(lo, at - c["window"] + 1), min(hi, at + c["window"] - 1)
        if n:
            mine = min(int(i * n / (0.9 * lq)), n) if lq == lk or not c["causal"] and n > 1 else 0
            if mine == n:
                continue
            dlo, dhi = mine * size, (mine + 1) * size - 1
        else:
            dlo, dhi = 0, lk - 1
        seen = max(0.0, min(hi, dhi) - max(lo, dlo) + 1)
        if pre:
            seen += max(0.0, min(dhi, pre - 1) - max(dlo, 0) + 1) - max(0.0, min(hi, dhi, pre - 1) - max(lo, dlo) + 1)
        total += seen
    return max(1.0, total)


def work(case):
    c = case
    if c["kind"] == "rope":
        n = c["batch"] * c["seq"]
        each = n * c["heads"] * c["dim"]
        times = 2 if c["grad"] else 1
        return {"bytes": times * 8 * each + 4 * n, "flops": times * 3 * n * c["heads"] * c["rot"]}
    b, h, kv, lq, lk, d = (c[k] for k in ("batch", "heads", "kv", "lq", "lk", "dim"))
    q, k = 4 * b * lq * h * d, 4 * b * lk * kv * d
    flops = 4 * b * h * d * _pairs(c)
    if not c["grad"]:
        return {"bytes": 2 * q + 2 * k, "flops": flops}
    return {"bytes": 4 * q + 4 * k, "flops": 3.5 * flops}


# ------------------------------------------------------------------------------------------------------------- exact
def _exact_rope(c, s):
    rows, h, d, rot = c["batch"] * c["seq"], c["heads"], c["dim"], c["rot"]
    base = BASE
    if c["scaling"] == "ntk":
        base = BASE * math.pow(FACTOR, rot / max(rot - 2, 1))
    pairs = []
    for i in range(rot // 2):
        f = math.pow(base, -2.0 * i / rot)
        if c["scaling"] == "linear":
            f /= FACTOR
        elif c["scaling"] == "bands":
            turns = f * TRAINED / (2 * math.pi)
            keep = min(1.0, max(0.0, (turns - LOW) / (HIGH - LOW)))
            f = f * keep + f * (1 - keep) / FACTOR
        pairs.append(f)
    amp = AMPLITUDE if c["scaling"] == "bands" else 1.0
    ang = s["pos"].double()[:, None] * torch.tensor(pairs, device=DEV, dtype=torch.float64)[None]
    z = torch.polar(torch.full_like(ang, amp), ang)[:, None, :]
    first = torch.arange(rot // 2, device=DEV)
    first, second = (first, first + rot // 2) if c["layout"] == "half" else (2 * first, 2 * first + 1)

    def turned(x, w):
        x = x.double().view(rows, h, d)
        y = torch.complex(x[..., first], x[..., second]) * w
        out = x.clone()
        out[..., first], out[..., second] = y.real, y.imag
        return out.view(rows, h * d)

    out = {"y": turned(s["x"], z)}
    if c["grad"]:
        out["dx"] = turned(s["g"], z.conj())
    return out


def exact(case, seed):
    c, s = case, _inputs(case, seed)
    if c["kind"] == "rope":
        return _exact_rope(c, s)
    b, h, kv, lq, lk, d = (c[k] for k in ("batch", "heads", "kv", "lq", "lk", "dim"))
    out = {"o": torch.empty(b, lq, h, d, device=DEV, dtype=torch.float64)}
    if c["grad"]:
        out["dq"] = torch.empty_like(out["o"])
        out["dk"] = torch.zeros(b, lk, kv, d, device=DEV, dtype=torch.float64)
        out["dv"] = torch.zeros_like(out["dk"])
    gap = torch.arange(lk - lq, lk, device=DEV)[:, None] - torch.arange(lk, device=DEV)[None]  # query minus key position
    for n in range(b):
        hide = torch.zeros(lq, lk, device=DEV, dtype=torch.bool)
        if c["causal"]:
            hide |= gap < 0
        if c["window"]:
            hide |= (gap >= c["window"]) | (gap <= -c["window"])
        if c["prefix"]:
            hide[:, :int(s["prefix"][n])] = False
        if c["docs"]:
            hide |= s["qdoc"][n][:, None] != s["kdoc"][n][None]
            hide |= (s["kdoc"][n] < 0)[None]
        for a in range(h):
            q, k, v = (t.double().contiguous().requires_grad_(c["grad"])
                       for t in (s["q"][n, :, a], s["k"][n, :, a // (h // kv)], s["v"][n, :, a // (h // kv)]))
            x = (q @ k.t().contiguous()) / math.sqrt(d)
            if c["cap"]:
                x = c["cap"] * torch.tanh(x / c["cap"])
            if c["slopes"]:
                x = x - float(s["slopes"][a]) * gap.abs().double()
            x = x.masked_fill(hide, -1e300)
            w = torch.softmax(x, 1).masked_fill(hide, 0.0)
            y = w @ v
            out["o"][n, :, a] = y.detach()
            if c["grad"]:
                dq, dk, dv = torch.autograd.grad(y, (q, k, v), s["g"][n, :, a].double())
                out["dq"][n, :, a] = dq
                out["dk"][n, :, a // (h // kv)] += dk
                out["dv"][n, :, a // (h // kv)] += dv
    return out
