"""Timed cases of training in 8 bits: activations kept for the backward pass as 8-bit floats with one power-of-two scale
to each block of 128, and products of tensors held that way.

A packed tensor holds, for each block of 128 values along its rows, e4m3 codes of x / 2^e, e the least exponent (-127 at
least) that brings the block's largest finite value to 448 or below; infinities and NaN become NaN. The library's layout,
for [rows, cols]: rows of codes padded with zeros to a multiple of 128, then rows of scale bytes (e + 127), padded with
zeros to a multiple of four.

`kind` selects the operator, the other entries are sizes:

  act     a tensor packed and unpacked again
  linear  a Linear whose products take packed operands: y = x w^T + b, and with `grad` dx = g w, dw = g^T x, db; every
          product packs its operands along its own sum. With `kept` the packed weight is in hand, as a server keeps it
  dw      the weight and bias gradient of a Linear whose input was kept packed, from a gradient in 32 bits
  gelu    GELU that keeps its input packed, and its backward
  norm    LayerNorm that keeps its normalised rows packed, and its backward

The plain forms are elementary torch operations in 32 bits (row means and variances in 64); `exact` computes the
definitions in 64 bits.
"""
import ctypes as C
import importlib
import math

import torch

own = False
DEV = "cuda"


# ------------------------------------------------------------------------------------------------------------- cases
def _case(name, kind, **sizes):
    c = dict(sizes, kind=kind)
    return dict(c, name=name) if name else c


def listed():
    return [
        # the hidden layer of a small perceptron's batch: latency
        _case("act_mlp", "act", rows=64, cols=256),
        # a long batch's feed-forward activations
        _case("act_long", "act", rows=16384, cols=4096),
        # one new token for each of four sequences through a layer whose packed weight is kept
        _case("linear_token", "linear", rows=4, inp=4096, out=4096, grad=False, kept=True),
        # odd sizes throughout, a training step
        _case("linear_ragged", "linear", rows=777, inp=1000, out=333, grad=True, kept=False),
        # the MiniLM-sized encoder's first feed-forward layer, a training step (32 sequences of 128)
        _case("linear_minilm", "linear", rows=4096, inp=384, out=1536, grad=True, kept=False),
        # a wide layer over a long batch, a training step
        _case("linear_wide", "linear", rows=16384, inp=4096, out=4096, grad=True, kept=False),
        # the MiniLM-sized encoder's first feed-forward layer with its input kept in 8 bits
        _case("dw_minilm", "dw", rows=4096, inp=384, out=1536),
        # the BERT-base-sized q|k|v projection over a long batch
        _case("dw_bert", "dw", rows=16384, inp=768, out=2304),
        # the MiniLM-sized encoder's GELU
        _case("gelu_minilm", "gelu", rows=4096, cols=1536),
        # an odd width over a long batch
        _case("gelu_odd", "gelu", rows=16001, cols=1999),
        # the MiniLM-sized encoder's LayerNorm
        _case("norm_minilm", "norm", rows=4096, cols=384),
        # wide rows over a long batch
        _case("norm_wide", "norm", rows=16384, cols=4096),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["act", "linear", "linear", "linear", "dw", "dw", "gelu", "norm"])
    rows = _log(rng, 1, 16384)
    if kind in ("act", "gelu", "norm"):
        # rows of two are left out of the norm: all their gradients are zero but for rounding
        return _case(None, kind, rows=rows, cols=_log(rng, 3 if kind == "norm" else 1, 4096))
    inp, out = _log(rng, 8, 4096), _log(rng, 8, 4096)
    if rng.random() < 0.5:  # widths as layers mostly have them
        inp, out = -(-inp // 64) * 64, -(-out // 64) * 64
    if kind == "dw":
        return _case(None, kind, rows=rows, inp=inp, out=out)
    if rng.random() < 0.3:
        return _case(None, kind, rows=rng.choice([1, 2, 3, 8, 16, 17, 40, 64]), inp=inp, out=out, grad=False, kept=True)
    return _case(None, kind, rows=rows, inp=inp, out=out, grad=rng.random() < 0.8, kept=False)


# ------------------------------------------------------------------------------------------------------------ inputs
EPS = 1e-5


def _inputs(c, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed & ((1 << 63) - 1))

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=gen, device=DEV).mul_(std)

    def activations(rows, cols):
        """Normal values whose columns have levels of their own, a few of them large, as layers' outputs have."""
        level = torch.exp(0.5 * torch.randn(cols, generator=gen, device=DEV))
        far = torch.rand(cols, generator=gen, device=DEV) < 0.01
        return normal(rows, cols) * torch.where(far, 20.0 * level, level)

    if c["kind"] in ("linear", "dw"):
        rows, inp, out = c["rows"], c["inp"], c["out"]
        s = {"x": activations(rows, inp)}
        if c["kind"] == "linear":
            s["w"], s["b"] = normal(out, inp, std=1.0 / math.sqrt(inp)), normal(out, std=0.1)
        if c["kind"] == "dw" or c["grad"]:
            s["g"] = normal(rows, out, std=1.0 / rows) * torch.exp(normal(rows, 1))
        return s
    rows, cols = c["rows"], c["cols"]
    s = {"x": activations(rows, cols)}
    if c["kind"] == "norm":
        s["x"] += normal(rows, 1, std=0.3)
        s["gamma"], s["beta"] = 1.0 + normal(cols, std=0.1), normal(cols, std=0.1)
    if c["kind"] != "act":
        s["g"] = normal(rows, cols, std=1.0 / rows)
    return s


def _strides(cols):
    """Bytes of codes and of scales of one packed row."""
    codes = -(-cols // 128) * 128
    return codes, -(-codes // 512) * 4


def _packed(rows, cols):
    return torch.empty(rows * sum(_strides(cols)), device=DEV, dtype=torch.uint8)


def prepare(case, seed):
    c, i = case, _inputs(case, seed)
    s = {"case": c, "in": i, "out": {}, "held": {}}
    # the buffers that a program hands to the library: outputs, and the packed tensors that it keeps between the calls
    o, h = s["out"], s["held"]
    if c["kind"] in ("linear", "dw"):
        rows, inp, out = c["rows"], c["inp"], c["out"]
        if c["kind"] == "dw" or c["grad"]:
            h["xt8"] = _packed(inp, rows)
            o["dw"], o["db"] = torch.empty(out, inp, device=DEV), torch.empty(out, device=DEV)
        if c["kind"] == "linear":
            h["x8"], o["y"] = _packed(rows, inp), torch.empty(rows, out, device=DEV)
            h["w8"] = _packed(out, inp)
            if c["kept"]:  # the weight is in hand packed only
                codes, e = _pack(i.pop("w"))
                to, ts = _strides(inp)
                scales = torch.zeros(out, ts, device=DEV, dtype=torch.uint8)
                scales[:, :e.shape[1]] = (e + 127).to(torch.uint8)
                h["w8"][:out * to] = codes.view(torch.uint8).reshape(-1)
                h["w8"][out * to:] = scales.reshape(-1)
            if c["grad"]:
                h["wt8"], h["g8"], h["gt8"] = _packed(inp, out), _packed(rows, out), _packed(out, rows)
                o["dx"] = torch.empty(rows, inp, device=DEV)
    else:
        rows, cols = c["rows"], c["cols"]
        h["x8"], o["y"] = _packed(rows, cols), torch.empty_like(i["x"])
        if c["kind"] != "act":
            o["dx"] = torch.empty_like(i["x"])
        if c["kind"] == "norm":
            h["rstd"] = torch.empty(rows, device=DEV)
            o["dgamma"], o["dbeta"] = torch.empty(cols, device=DEV), torch.empty(cols, device=DEV)
    torch.cuda.synchronize()  # the inputs come from torch's stream, the library's calls run on its context's
    return s


# ------------------------------------------------------------------------------------------------------ plain forms
def _two_to(e):
    """2^e in 32 bits, exactly, for exponents from -127 to 127."""
    return torch.where(e > -127, (e + 127) << 23, torch.full_like(e, 1 << 22)).view(torch.float32)


def _pack(x):
    """Codes [rows, a multiple of 128] and exponents [rows, blocks]."""
    rows, cols = x.shape
    x = torch.nn.functional.pad(x, (0, -cols % 128)).view(rows, -1, 128)
    fine = torch.isfinite(x)
    x = torch.where(fine, x, torch.zeros_like(x))
    m, e = torch.frexp(x.abs().amax(2))
    e = torch.where(m == 0, torch.full_like(e, -127), (e - 9 + (m > 0.875).int()).clamp_min(-127))
    x = x * _two_to(-e)[:, :, None]
    codes = torch.where(fine, x, torch.full_like(x, math.nan)).to(torch.float8_e4m3fn)
    return codes.view(rows, -1), e


def _value(codes, e, cols):
    v = codes.float().view(codes.shape[0], -1, 128) * _two_to(e)[:, :, None]
    return v.view(codes.shape[0], -1)[:, :cols]


def _rounded(x):
    return _value(*_pack(x), x.shape[1])


def _rounded_t(x):
    """The value of x's transpose packed, [cols, rows]."""
    return _rounded(x.t().contiguous())


def _plain_linear(c, s, held):
    rows, inp, out = c["rows"], c["inp"], c["out"]
    if c["kept"]:
        to, ts = _strides(inp)
        codes = held["w8"][:out * to].view(torch.float8_e4m3fn).view(out, to)
        e = held["w8"][out * to:].view(out, ts)[:, :to // 128].int() - 127
        w = _value(codes, e, inp)
    else:
        w = _rounded(s["w"])
    o = {"y": _rounded(s["x"]) @ w.t() + s["b"]}
    if c["grad"]:
        o["dx"] = _rounded(s["g"]) @ _rounded_t(s["w"]).t()
        o["dw"] = _rounded_t(s["g"]) @ _rounded_t(s["x"]).t()
        o["db"] = s["g"].double().sum(0).float()
    return o


def _plain_dw(c, s, held):
    xt = _rounded_t(s["x"])
    return {"dw": s["g"].t().contiguous() @ xt.t(), "db": s["g"].double().sum(0).float()}


def _plain_gelu(c, s, held):
    x, h = s["x"], _rounded(s["x"])
    y = 0.5 * x * (1.0 + torch.erf(x * math.sqrt(0.5)))
    slope = 0.5 * (1.0 + torch.erf(h * math.sqrt(0.5))) + h * torch.exp(-0.5 * h * h) * (1.0 / math.sqrt(2.0 * math.pi))
    return {"y": y, "dx": s["g"] * slope}


def _plain_norm(c, s, held):
    x, g = s["x"], s["g"]
    d = x.double()
    mean = d.mean(1, keepdim=True)
    rstd = (1.0 / torch.sqrt((d - mean).square().mean(1, keepdim=True) + EPS)).float()
    xh = (x - mean.float()) * rstd
    h, q = _rounded(xh), g * s["gamma"]
    m1, m2 = q.mean(1, keepdim=True), (q * h).mean(1, keepdim=True)
    return {"y": xh * s["gamma"] + s["beta"], "dx": rstd * (q - m1 - h * m2),
            "dgamma": (g * h).double().sum(0).float(), "dbeta": g.double().sum(0).float()}


def _plain_act(c, s, held):
    return {"y": _rounded(s["x"])}


_PLAIN = {"act": _plain_act, "linear": _plain_linear, "dw": _plain_dw, "gelu": _plain_gelu, "norm": _plain_norm}


# ---------------------------------------------------------------------------------------------- the framework's calls
_LIB = None


def _ctx():
    """The package and one library context for the process, as a program keeps them."""
    global _LIB
    if _LIB is None:
        pkg = importlib.import_module("onemodel-csharp_amd")
        _LIB = pkg, pkg.Context(0)
    return _LIB


def _calls(state):
    """The library calls of one pass with their arguments bound."""
    _, ctx = _ctx()
    c, calls = state["case"], []
    every = {**state["in"], **state["held"], **state["out"]}

    def add(name, *args):
        bound = [C.c_void_p(every[a].data_ptr()) if isinstance(a, str) else a for a in args]
        calls.append((getattr(ctx.L, name), name, (ctx.h, *bound)))

    if c["kind"] in ("linear", "dw"):
        rows, inp, out = c["rows"], c["inp"], c["out"]
        if c["kind"] == "dw":
            add("om_pack8", "x", inp, rows, inp, None, "xt8")
            add("om_linear_bwd_x8", "g", "xt8", None, None, "dw", "db", rows, inp, out, 0, 0, 0)
            return ctx, calls
        grad = c["grad"]
        add("om_pack8", "x", inp, rows, inp, "x8", "xt8" if grad else None)
        if not c["kept"]:
            add("om_pack8", "w", inp, out, inp, "w8", "wt8" if grad else None)
        add("om_gemm8", rows, out, inp, "x8", "w8", "b", "y", out, 0)
        if grad:
            add("om_pack8", "g", out, rows, out, "g8", "gt8")
            add("om_gemm8", rows, inp, out, "g8", "wt8", None, "dx", inp, 0)
            add("om_gemm8", out, inp, rows, "gt8", "xt8", None, "dw", inp, 0)
            add("om_colsum", "g", "db", rows, out, 0)
        return ctx, calls
    rows, cols = c["rows"], c["cols"]
    if c["kind"] == "act":
        add("om_pack8", "x", cols, rows, cols, "x8", None)
        add("om_unpack8", "x8", "y", cols, rows, cols, 0)
    elif c["kind"] == "gelu":
        add("om_gelu_fwd_x8", "x", "y", "x8", rows, cols)
        add("om_gelu_bwd_x8", "g", "x8", "dx", rows, cols, 0)
    else:
        add("om_layernorm_fwd_x8", "x", "gamma", "beta", "y", "x8", "rstd", rows, cols, EPS)
        add("om_layernorm_bwd_x8", "g", "x8", "gamma", "rstd", "dx", "dgamma", "dbeta", rows, cols, 0, 0)
    return ctx, calls


def run(state):
    if not own:
        return _PLAIN[state["case"]["kind"]](state["case"], state["in"], state["held"])
    if "calls" not in state:
        state["calls"] = _calls(state)
    ctx, calls = state["calls"]
    for fn, name, args in calls:
        if fn(*args):
            raise RuntimeError("%s: %s" % (name, ctx.L.om_last_error(ctx.h).decode()))
    return state["out"]


# -------------------------------------------------------------------------------------------------------------- work
def work(case):
    """Each input read once, each output written once; packed tensors that the pass itself makes are written and read."""
    c = case
    if c["kind"] in ("linear", "dw"):
        rows, inp, out = c["rows"], c["inp"], c["out"]
        x, w, g = rows * inp, inp * out, rows * out
        if c["kind"] == "dw":
            return {"bytes": 4 * x + 2 * x + 4 * g + 4 * w, "flops": 2 * rows * inp * out}
        if not c["grad"]:
            return {"bytes": (4 + 2) * x + (1 if c["kept"] else 6) * w + 4 * g, "flops": 2 * rows * inp * out}
        return {"bytes": (4 + 4) * (x + w + g) + 4 * (x + w + g), "flops": 6 * rows * inp * out}
    n = c["rows"] * c["cols"]
    return {"bytes": 10 * n if c["kind"] == "act" else 18 * n, "flops": {"act": 4, "gelu": 40, "norm": 30}[c["kind"]] * n}


# ------------------------------------------------------------------------------------------------------------- exact
def _packed64(x):
    """What a packed tensor of x [rows, cols] holds, as 64-bit values, from the definition."""
    x = x.double()
    rows, cols = x.shape
    out = torch.empty_like(x)
    for at in range(0, cols, 128):
        b = x[:, at:at + 128]
        fine = torch.isfinite(b)
        top = torch.where(fine, b, torch.zeros_like(b)).abs().max(1, keepdim=True).values
        scale = torch.exp2(torch.ceil(torch.log2(top / 448.0)).clamp(min=-127.0))
        v = b / scale
        step = torch.exp2(torch.floor(torch.log2(v.abs())).clamp(min=-6.0) - 3.0)
        out[:, at:at + 128] = torch.where(fine, torch.round(v / step) * step * scale, torch.full_like(b, math.nan))
    return out


def exact(case, seed):
    c, s = case, _inputs(case, seed)
    if c["kind"] == "act":
        return {"y": _packed64(s["x"])}
    if c["kind"] in ("linear", "dw"):
        back = c["kind"] == "dw" or c["grad"]
        o = {}
        if back:
            g = s["g"].double()
            o["db"] = torch.ones(1, c["rows"], device=DEV, dtype=torch.float64).mm(g)[0]
            left = g.t() if c["kind"] == "dw" else _packed64(s["g"].t())
            o["dw"] = left.contiguous().mm(_packed64(s["x"].t()).t().contiguous())
        if c["kind"] == "linear":
            o["y"] = torch.addmm(s["b"].double(), _packed64(s["x"]), _packed64(s["w"]).t().contiguous())
            if back:
                o["dx"] = _packed64(s["g"]).mm(_packed64(s["w"].t()).t().contiguous())
        return o
    if c["kind"] == "gelu":
        x, h = s["x"].double(), _packed64(s["x"])
        cdf = torch.special.ndtr(h)
        return {"y": x * torch.special.ndtr(x),
                "dx": s["g"].double() * (cdf + h * torch.exp(-h * h / 2) / math.sqrt(2 * math.pi))}
    # the rows that are kept are 32-bit values by definition: the statistics rounded once each, then a difference and a
    # product in 32 bits
    n = c["cols"]
    x = s["x"].double()
    mean = x.sum(1, keepdim=True) / n
    var = ((x - mean) ** 2).sum(1, keepdim=True) / n
    rstd = (var + EPS) ** -0.5
    gamma, g = s["gamma"].double(), s["g"].double()
    h = _packed64((s["x"] - mean.float()) * rstd.float())
    q = g * gamma
    dx = rstd * (q - q.sum(1, keepdim=True) / n - h * (q * h).sum(1, keepdim=True) / n)
    return {"y": (x - mean) * rstd * gamma + s["beta"].double(), "dx": dx, "dgamma": (g * h).sum(0), "dbeta": g.sum(0)}
