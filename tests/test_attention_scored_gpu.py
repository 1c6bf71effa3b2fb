"""Scored attention (om_attention_fwd_scored / om_attention_bwd_scored) against the float64 definition.

Tolerance: max|error| / max|value| per output. A score is a sum of d products and a handful of roundings: at the sizes
here |x| stays below 16 in log2 units, so 2^-24 * 16 per rounding of the score, under sqrt(d) / 2 <= 8 such roundings in
random directions for its sum, gives weights within 8e-6 of themselves at most and 1e-6 typically; outputs and gradients
are averages over weights, so 1e-5, the library's bound for fp32 paths, holds with room. dq and dk also cancel: ds = p (g . v
- delta) is the difference of two sums, each within 2^-24 sum |g v| of itself per rounding, which leaves dq (one key seen: zero)
4 such roundings times scale |k| off whatever its own size, and dk the same times the square root of the rows it sums
(Case.floor)."""
import ctypes as C
import threading

import numpy as np
import pytest

import scored_ref as R
from gpu_util import Dev, DevBuf, hip, load_pkg

pytestmark = pytest.mark.gpu
TOL = 1e-5


@pytest.fixture(scope="module")
def dev():
    return Dev()


def rng_of(*k):
    return np.random.default_rng(list(k))


class Case:
    """Inputs of a call, the rule, and the calls themselves."""

    def __init__(self, dev, B, H, Hk, lq, lk, d, seed=0, scale=0.0, cap=0.0, causal=0, window=0, slopes=False, qdoc=None,
                 kdoc=None, prefix=None, packed=False, pad=0, shift=0):
        self.dev, self.dims = dev, (B, H, Hk, lq, lk, d)
        r = rng_of(B, H, lq, lk, d, seed)
        self.q = (1.5 * r.normal(size=(B, lq, H, d))).astype(np.float32)
        self.k, self.v = (r.normal(size=(B, lk, Hk, d)).astype(np.float32) for _ in range(2))
        self.g = r.normal(size=(B, lq, H, d)).astype(np.float32)
        self.sl = np.exp2(-8.0 * np.arange(1, H + 1) / H).astype(np.float32) if slopes else None
        self.rule = dict(scale=scale, cap=cap, slopes=self.sl, causal=causal, window=window, prefix=prefix, qdoc=qdoc,
                         kdoc=kdoc)
        self.packed, self.pad, self.shift = packed, pad, shift
        f = load_pkg().om_attention_scores()
        f.heads, f.kv_heads, f.scale, f.cap, f.causal, f.window = H, Hk, scale, cap, causal, window
        self.keep = []
        for field, a, t in (("slopes", self.sl, np.float32), ("q_doc", qdoc, np.int32), ("k_doc", kdoc, np.int32),
                            ("prefix", prefix, np.int32)):
            if a is not None:
                b = dev.put(np.asarray(a, t))
                self.keep.append(b)
                setattr(f, field, b.data_ptr())
        self.form = f

    def rows(self, a, width, fill=np.nan):
        """[B, L, n, d] as rows of n*d + pad floats from `shift` floats into a buffer; (buffer, pointer, stride, reader)."""
        B, L = a.shape[:2]
        w = a.shape[2] * a.shape[3]
        ld = w + self.pad if width is None else width
        flat = np.full(self.shift + B * L * ld, fill, np.float32)
        flat[self.shift:].reshape(B * L, ld)[:, :w] = a.reshape(B * L, w)
        buf = self.dev.put(flat)
        self.keep.append(buf)

        def read():
            out = self.dev.get(buf)[self.shift:].reshape(B * L, ld)
            assert np.array_equal(out[:, w:], flat[self.shift:].reshape(B * L, ld)[:, w:], equal_nan=True)
            return out[:, :w].reshape(a.shape)
        return C.c_void_p(buf.data_ptr() + 4 * self.shift), ld, read

    def place(self):
        B, H, Hk, lq, lk, d = self.dims
        if self.packed:
            x = np.concatenate([a.reshape(B * lq, -1) for a in (self.q, self.k, self.v)], 1)
            buf = self.dev.put(x)
            self.keep.append(buf)
            ld, at = x.shape[1], buf.data_ptr()
            self.ins = (C.c_void_p(at), ld, C.c_void_p(at + 4 * H * d), C.c_void_p(at + 4 * (H + Hk) * d), ld)
        else:
            q, ldq, _ = self.rows(self.q, None)
            k, ldk, _ = self.rows(self.k, None)
            v, _, _ = self.rows(self.v, None)
            self.ins = (q, ldq, k, v, ldk)

    def forward(self, stats=True):
        B, H, Hk, lq, lk, d = self.dims
        self.place()
        self.st = self.dev.empty((max(1, 2 * B * H * lq),), fill=np.nan) if stats else None
        self.o, self.ldo, read = self.rows(np.full(self.q.shape, 3.0, np.float32), None)
        self.dev.call("om_attention_fwd_scored", *self.ins, self.o, self.ldo, self.st, B, lq, lk, d, C.byref(self.form))
        return read()

    def backward(self, acc=0, want=(1, 1, 1), start=5.0):
        B, H, Hk, lq, lk, d = self.dims
        g, ldg, _ = self.rows(self.g, None)
        outs = [self.rows(np.full(a.shape, start, np.float32), None) for a in (self.q, self.k, self.v)]
        ptr = [x[0] if w else None for x, w in zip(outs, want)]
        self.dev.call("om_attention_bwd_scored", *self.ins, self.o, self.ldo, self.st, g, ldg, ptr[0], outs[0][1], ptr[1],
                      ptr[2], outs[1][1], B, lq, lk, d, C.byref(self.form), acc)
        return [x[2]() for x in outs]

    def floor(self):
        """What cancellation in g . v - delta leaves of dq and dk (see above); none for o and dv."""
        B, H, Hk, lq, lk, d = self.dims
        if not (lq and lk and B):
            return 0.0, 0.0
        sum_gv = np.abs(self.g).sum(3).max() * np.abs(self.v).max()
        each = 2.0 ** -22 * sum_gv * (abs(self.form.scale) or d ** -0.5)
        return each * np.abs(self.k).max(), each * np.abs(self.q).max() * (lq * H / Hk) ** 0.5

    def reference(self, grad=True):
        return R.attention(self.q, self.k, self.v, g=self.g if grad else None, **self.rule)


def near(got, want, tol=TOL, what="", floor=0.0):
    assert got.shape == want.shape
    assert np.isfinite(got).all(), what
    top = float(np.abs(want).max()) if want.size else 0.0
    err = float(np.abs(got - want).max()) if want.size else 0.0
    assert err <= tol * top + floor, (what, err, top, floor)


def both(c, tol=TOL):
    want = c.reference()
    near(c.forward(), want[0], tol, "o")
    for got, ref, n, fl in zip(c.backward(), want[1:], ("dq", "dk", "dv"), (*c.floor(), 0.0)):
        near(got, ref, tol, n, fl)


def docs(B, L, seed, kinds=3, pad=True):
    r = rng_of(seed, B, L)
    return np.sort(r.integers(-1 if pad else 0, kinds, (B, L)), 1)[:, ::-1].astype(np.int32)  # padding last


SHAPES = [
    # B, H, Hk, lq, lk, d
    (1, 1, 1, 1, 1, 1),
    (2, 2, 1, 1, 1, 64),
    (1, 3, 1, 2, 5, 3),
    (2, 4, 4, 17, 17, 32),
    (1, 4, 2, 33, 65, 40),
    (2, 6, 2, 64, 64, 64),
    (1, 2, 2, 65, 63, 33),       # odd width: no 16-byte rows
    (1, 8, 1, 31, 129, 80),
    (1, 2, 1, 100, 100, 96),
    (1, 2, 1, 70, 130, 128),
    (1, 1, 1, 40, 50, 130),
    (1, 2, 1, 20, 33, 256),
    (3, 2, 1, 130, 200, 64),
    (8, 4, 4, 17, 70, 32),
    (6, 4, 4, 9, 320, 64),
    (2, 6, 2, 90, 90, 64),
    (5, 4, 2, 65, 63, 33),
    (2, 8, 1, 70, 130, 80),
    (3, 4, 2, 100, 100, 96),
    (4, 4, 1, 70, 130, 128),
]


@pytest.mark.parametrize("s", SHAPES, ids=["x".join(map(str, s)) for s in SHAPES])
def test_shapes_causal(dev, s):
    both(Case(dev, *s, causal=1))


@pytest.mark.parametrize("s", SHAPES, ids=["x".join(map(str, s)) for s in SHAPES])
def test_shapes_everything(dev, s):
    """Cap, distance bias, window, prefix and documents together."""
    B, H, Hk, lq, lk, d = s
    both(Case(dev, *s, seed=1, causal=1, window=max(1, lk // 2), cap=5.0, slopes=True, prefix=[min(3, lk)] * B,
              qdoc=docs(B, lq, 1), kdoc=docs(B, lk, 1)))


RULES = {
    "plain": {},
    "scale": dict(scale=0.25),
    "negative-scale": dict(scale=-0.3),
    "cap-small": dict(cap=0.5),
    "cap-large": dict(cap=50.0),
    "slopes": dict(slopes=True),
    "window-1": dict(window=1),
    "window-wide": dict(window=2 ** 31 - 1),
    "causal-window": dict(causal=1, window=7),
    "prefix": dict(causal=1, prefix=[0, 90]),
    "prefix-past-the-end": dict(causal=1, prefix=[2 ** 31 - 1, -4]),
    "prefix-window": dict(causal=1, window=9, prefix=[20, 1]),
}


@pytest.mark.parametrize("rule", RULES, ids=RULES.keys())
@pytest.mark.parametrize("lens", [(95, 95), (60, 140), (140, 60), (37, 90), (1, 300)], ids=lambda v: "x".join(map(str, v)))
def test_rules(dev, rule, lens):
    both(Case(dev, 2, 4, 2, *lens, 64, seed=2, **RULES[rule]))


def test_queries_before_the_first_key_see_nothing(dev):
    for c, n in ((Case(dev, 1, 2, 1, 90, 20, 32, causal=1), 70), (Case(dev, 4, 4, 2, 90, 40, 32, causal=1), 50)):
        o = c.forward()
        dq = c.backward()[0]
        assert (o[:, :n] == 0).all() and (dq[:, :n] == 0).all() and (o[:, n:] != 0).any()
        both(c)


def test_documents_in_any_order(dev):
    r = rng_of(8)
    qd, kd = r.integers(-2, 5, (2, 95)), r.integers(-2, 5, (2, 110))
    both(Case(dev, 2, 4, 2, 95, 110, 64, qdoc=qd, kdoc=kd, cap=3.0))


def test_documents_that_leave_nothing(dev):
    c = Case(dev, 2, 4, 4, 96, 100, 32, qdoc=np.full((2, 96), 4), kdoc=np.full((2, 100), 5))
    assert (c.forward() == 0).all()
    assert all((x == 0).all() for x in c.backward())


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, 3e38], ids=str)
@pytest.mark.parametrize("where", ["padding", "future", "other-document"])
def test_what_is_not_seen_has_no_effect(dev, bad, where):
    """Wild values in keys (and rows) that a query does not see change no bit of its outputs."""
    B, H, Hk, L, d = 1, 8, 4, 96, 64
    kw = dict(causal=1)
    seen = slice(0, 60)
    if where != "future":
        ids = np.where(np.arange(L)[None] < 60, 0, -1 if where == "padding" else 1)
        kw = dict(qdoc=ids, kdoc=ids)
    a, b = Case(dev, B, H, Hk, L, L, d, seed=4, **kw), Case(dev, B, H, Hk, L, L, d, seed=4, **kw)
    for x in (b.q, b.k, b.v):
        x[:, 60:, :, ::3] = bad
    a.g[:, 60:] = 0  # the later rows' own gradients would reach the earlier keys in the causal case
    b.g[:, 60:] = 0
    oa, ob = a.forward(), b.forward()
    near(ob[:, seen], a.reference(False)[:, seen])
    ga, gb = a.backward(), b.backward()
    want = a.reference()[1:]
    near(gb[0][:, seen], want[0][:, seen], what="dq")
    if where != "future":  # in the causal case the wild queries do see the early keys
        for n in (1, 2):
            near(gb[n][:, seen], want[n][:, seen], what=n)
        if where == "padding":
            assert all((x[:, 60:] == 0).all() for x in [ob] + gb)


def test_visible_nan_and_infinity_follow_ieee(dev):
    c = Case(dev, 1, 1, 1, 70, 70, 32, causal=1)
    c.k[0, 30, 0, 3] = np.nan
    o = c.forward()
    assert np.isfinite(o[0, :30]).all() and np.isnan(o[0, 30:]).all()
    near(o[:, :30], c.reference(False)[:, :30])
    c = Case(dev, 1, 1, 1, 70, 70, 32, causal=1)
    c.v[0, 10, 0, 5] = np.inf
    o = c.forward()
    assert np.isinf(o[0, 10:, 0, 5]).all() and np.isfinite(o[0, :, 0, :5]).all() and np.isfinite(o[0, :10]).all()


@pytest.mark.parametrize("lens", [(3, 300), (220, 220)], ids=str)
@pytest.mark.parametrize("power", [-30, 20])
def test_scaled_operands(dev, lens, power):
    """The same attention with values scaled by powers of two: outputs scale along (the scores are kept by `scale`)."""
    a = Case(dev, 1, 2, 1, *lens, 64, causal=1, scale=0.125)
    b = Case(dev, 1, 2, 1, *lens, 64, causal=1, scale=0.125 * 2.0 ** -power)
    b.k = np.ldexp(a.k, power)
    b.v = np.ldexp(a.v, -power)
    want = a.reference()
    near(np.ldexp(b.forward(), power), want[0], what="o")
    dq, dk, dv = b.backward()
    near(np.ldexp(dq, power), want[1], what="dq")
    near(np.ldexp(dk, 2 * power), want[2], what="dk")
    near(dv, want[3], what="dv")


@pytest.mark.parametrize("ratio", [1e4, 1e6, 1e9])
def test_rows_of_very_different_size(dev, ratio):
    """Two documents in a row whose values differ by `ratio`: each document's results keep their own precision."""
    L, ids = 128, (np.arange(128)[None] >= 50).astype(np.int32)
    c = Case(dev, 1, 4, 2, L, L, 64, seed=6, qdoc=ids, kdoc=ids)
    c.v[:, 50:] *= np.float32(ratio)
    c.g[:, 50:] *= np.float32(1.0 / ratio)
    want = c.reference()
    got = [c.forward()] + c.backward()
    for g, w, n in zip(got, want, ("o", "dq", "dk", "dv")):
        for part in (slice(0, 50), slice(50, L)):
            near(g[:, part], w[:, part], what=(n, part))


@pytest.mark.parametrize("kw", [dict(packed=True), dict(pad=4), dict(pad=1), dict(pad=3, shift=1), dict(shift=4)], ids=str)
@pytest.mark.parametrize("d", [64, 20])
def test_strides_and_alignment(dev, kw, d):
    both(Case(dev, 2, 4, 2, 95, 95, d, causal=1, **kw))


def test_accumulation_and_outputs_left_out(dev):
    c = Case(dev, 1, 4, 2, 150, 140, 64, causal=1, cap=4.0)
    want = c.reference()
    near(c.forward(), want[0])
    for got, ref in zip(c.backward(acc=1, start=2.0), want[1:]):
        near(got, ref + 2.0)
    for i in range(3):
        mask = [int(n == i) for n in range(3)]
        got = c.backward(want=mask)
        near(got[i], want[1 + i])
        assert all((got[n] == 5.0).all() for n in range(3) if n != i)


def test_forward_without_statistics(dev):
    c = Case(dev, 2, 4, 2, 95, 95, 64, causal=1)
    near(c.forward(stats=False), c.reference(False))


def test_empty_lengths(dev):
    c = Case(dev, 2, 2, 1, 3, 0, 8)
    assert (c.forward() == 0).all() and (c.backward()[0] == 0).all()
    c = Case(dev, 2, 2, 1, 0, 3, 8)
    c.forward()
    assert all((x == 0).all() for x in c.backward()[1:])
    assert all((x == 5).all() for x in c.backward(acc=1)[1:])
    Case(dev, 0, 2, 1, 3, 3, 8).forward()


@pytest.mark.parametrize("s", [(2, 4, 2, 130, 130, 64), (1, 2, 1, 1, 900, 64)], ids=str)
def test_same_bits_every_time(dev, s):
    c = Case(dev, *s, causal=1, cap=9.0)
    first = [c.forward()] + c.backward()
    for _ in range(3):
        for a, b in zip(first, [c.forward()] + c.backward()):
            assert np.array_equal(a.view(np.uint32), b.view(np.uint32))


@pytest.mark.parametrize("s", [(1, 2, 1, 700, 700, 64), (1, 4, 1, 515, 1300, 96), (2, 2, 2, 600, 600, 32), (1, 1, 1, 5, 5000, 128)],
                         ids=str)
def test_long(dev, s):
    both(Case(dev, *s, causal=1, cap=20.0))


def test_long_plain_and_windowed(dev):
    both(Case(dev, 1, 2, 2, 1025, 1025, 64, window=130, slopes=True))
    both(Case(dev, 1, 3, 1, 777, 777, 80, causal=1, prefix=[333]))
    both(Case(dev, 2, 2, 1, 640, 640, 64, qdoc=docs(2, 640, 3, 4), kdoc=docs(2, 640, 3, 4)))


@pytest.mark.parametrize("H", [1, 1024])
def test_offsets_past_32_bits(dev, H):
    """Rows so far apart that the last ones lie beyond 2^32 bytes (and 2^31 floats) from the first."""
    B, lq, lk, d, ld = 1, 8, 8, 64, 300_000_000
    w = H * d
    c = Case(dev, B, H, H, lq, lk, d, causal=1)
    want = c.reference()
    big = DevBuf((lk * ld,), np.float32)
    out = DevBuf((lk * ld,), np.float32)

    def write(buf, at, a):
        for t in range(a.shape[1]):
            row = np.ascontiguousarray(a[0, t].reshape(-1))
            assert hip().hipMemcpy(C.c_void_p(buf.data_ptr() + 4 * (t * ld + at)), row.ctypes.data, row.nbytes, 1) == 0

    def read(buf, at, shape):
        dev.ctx.sync()
        a = np.empty(shape, np.float32)
        for t in range(shape[1]):
            row = np.empty(shape[2] * shape[3], np.float32)
            assert hip().hipMemcpy(row.ctypes.data, C.c_void_p(buf.data_ptr() + 4 * (t * ld + at)), row.nbytes, 2) == 0
            a[0, t] = row.reshape(shape[2:])
        return a
    for n, a in enumerate((c.q, c.k, c.v, c.g)):
        write(big, w * n, a)

    def p(buf, n):
        return C.c_void_p(buf.data_ptr() + 4 * w * n)
    st = dev.empty((2 * H * lq,))
    ins = (p(big, 0), ld, p(big, 1), p(big, 2), ld)
    dev.call("om_attention_fwd_scored", *ins, p(out, 0), ld, st, B, lq, lk, d, C.byref(c.form))
    dev.call("om_attention_bwd_scored", *ins, p(out, 0), ld, st, p(big, 3), ld, p(out, 1), ld, p(out, 2), p(out, 3), ld, B,
             lq, lk, d, C.byref(c.form), 0)
    for n, ref in enumerate(want):
        near(read(out, w * n, ref.shape), ref, what=n)


def test_gradients_against_differences(dev):
    """The device's gradients against central differences of the float64 forward."""
    c = Case(dev, 1, 4, 2, 100, 100, 32, causal=1, cap=2.0, slopes=True, window=40)
    c.forward()
    grads = c.backward()
    r = rng_of(77)
    for n, x in enumerate((c.q, c.k, c.v)):
        for _ in range(4):
            at = tuple(r.integers(0, s) for s in x.shape)
            vals = []
            for e in (1e-4, -1e-4):
                y = [a.astype(np.float64) for a in (c.q, c.k, c.v)]
                y[n][at] += e
                vals.append((R.attention(*y, **c.rule) * c.g).sum())
            diff = (vals[0] - vals[1]) / 2e-4
            # differences: 1e-8 times a third derivative of order ten; the device's 1e-5 of the largest gradient
            assert abs(diff - grads[n][at]) <= TOL * float(np.abs(grads[n]).max()) + 1e-6, (n, at)


def _graph(dev, calls):
    """Captures calls() on the context's stream; the graph's handle."""
    dev.ctx.call("om_graph_capture_begin")
    try:
        calls()
    except Exception:
        dev.ctx.L.om_graph_capture_abort(dev.ctx.h)
        raise
    h = C.c_void_p()
    dev.ctx.call("om_graph_capture_end", C.byref(h))
    return h


class _Values(C.Structure):
    _fields_ = [("lr", C.c_float), ("step_size", C.c_float), ("sqrt_bc2", C.c_float)]


@pytest.mark.parametrize("s", [(2, 4, 2, 150, 150, 64), (2, 6, 2, 1, 700, 64)], ids=str)
def test_two_graphs_share_the_context(dev, s):
    """Captured passes of two sizes, replayed in turn with eager calls (one of which outgrows the scratch) between."""
    B, H, Hk, lq, lk, d = s
    cs = [Case(dev, *s, causal=1, cap=8.0), Case(dev, 1, H, Hk, lq + 40, lk + 40, d, slopes=True)]
    eager, graphs, outs = [], [], []
    for c in cs:
        eager.append([c.forward()] + c.backward())
        b, h, hk, q, k, w = c.dims
        o = [dev.empty((b, q, h, w)), dev.empty((b, q, h, w)), dev.empty((b, k, hk, w)), dev.empty((b, k, hk, w))]
        G = dev.put(c.g)
        c.keep.append(G)

        def calls(c=c, o=o, G=G):
            b, h, hk, q, k, w = c.dims
            dev.call("om_attention_fwd_scored", *c.ins, o[0], h * w, c.st, b, q, k, w, C.byref(c.form))
            dev.call("om_attention_bwd_scored", *c.ins, o[0], h * w, c.st, G, h * w, o[1], h * w, o[2], o[3], hk * w, b, q, k,
                     w, C.byref(c.form), 0)
        graphs.append(_graph(dev, calls))
        outs.append(o)
    vals = _Values(0.0, 0.0, 0.0)
    big = Case(dev, 2, 8, 8, 800, 1500, 128, causal=1)
    for step in range(4):
        for n in (0, 1):
            for o in outs[n]:
                dev.call("om_fill", o, C.c_float(np.nan), int(np.prod(o.shape)))
            assert dev.ctx.L.om_graph_launch(graphs[n], C.byref(vals)) == 0
            for got, ref in zip(outs[n], eager[n]):
                assert np.array_equal(dev.get(got).view(np.uint32), ref.reshape(got.shape).view(np.uint32)), (step, n)
        if step == 1:
            big.forward()
        else:
            cs[step % 2].forward()
    for h in graphs:
        assert dev.ctx.L.om_graph_destroy(h) == 0


def test_two_contexts_at_once():
    """Two threads with a context each."""
    errors = []

    def work(seed):
        try:
            dv = Dev()
            for i in range(4):
                both(Case(dv, 2, 4, 2, 120 + seed, 120 + 7 * i, 64, seed=seed, causal=1, cap=6.0))
        except BaseException as e:  # noqa: BLE001
            errors.append(e)
    ts = [threading.Thread(target=work, args=(s,)) for s in (1, 2)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not errors, errors


def test_decoder_attention_as_a_user_runs_it(dev):
    """Rotary positions in place on a packed projection, capped causal attention over grouped heads and packed documents,
    and both backward passes, against the float64 chain."""
    pkg = load_pkg()
    B, L, H, Hk, d = 2, 100, 4, 2, 64
    w, rows = (H + 2 * Hk) * d, B * L
    r = rng_of(21)
    x = r.normal(size=(rows, w)).astype(np.float32)
    g = r.normal(size=(rows, H * d)).astype(np.float32)
    ids = docs(B, L, 9)
    pos = np.concatenate([np.concatenate([np.arange((row == v).sum()) for v in sorted(set(row), reverse=True)]) for row in ids])
    rp = pkg.om_rope()
    rp.layout, rp.scaling, rp.rot, rp.amplitude, rp.base, rp.factor = 0, 0, 32, 1.0, 10000.0, 1.0
    f = R.rope_speeds(32)
    c = Case(dev, B, H, Hk, L, L, d, causal=1, cap=15.0, qdoc=ids, kdoc=ids)
    X, P = dev.put(x), dev.put(pos.astype(np.int32))
    dev.call("om_rope_fwd", X, w, P, 0, X, w, rows, L, H + Hk, d, C.byref(rp))
    at = X.data_ptr()
    O, DX, ST = dev.empty((rows, H * d)), dev.empty((rows, w)), dev.empty((2 * rows * H,))
    ins = (C.c_void_p(at), w, C.c_void_p(at + 4 * H * d), C.c_void_p(at + 4 * (H + Hk) * d), w)
    dev.call("om_attention_fwd_scored", *ins, O, H * d, ST, B, L, L, d, C.byref(c.form))
    t = DX.data_ptr()
    dev.call("om_attention_bwd_scored", *ins, O, H * d, ST, dev.put(g), H * d, C.c_void_p(t), w, C.c_void_p(t + 4 * H * d),
             C.c_void_p(t + 4 * (H + Hk) * d), w, B, L, L, d, C.byref(c.form), 0)
    dev.call("om_rope_bwd", DX, w, P, 0, DX, w, rows, L, H + Hk, d, C.byref(rp), 0)
    xh = x.reshape(rows, H + 2 * Hk, d)
    turned = R.rope(xh[:, :H + Hk], pos, 32, "half", f)
    q, k, v = turned[:, :H], turned[:, H:], xh[:, H + Hk:]
    o, dq, dk, dv = R.attention(q.reshape(B, L, H, d), k.reshape(B, L, Hk, d), v.reshape(B, L, Hk, d),
                                g=g.reshape(B, L, H, d), **c.rule)
    near(dev.get(O), o.reshape(rows, -1))
    back = R.rope(np.concatenate([dq.reshape(rows, H, d), dk.reshape(rows, Hk, d)], 1), pos, 32, "half", f, back=True)
    near(dev.get(DX), np.concatenate([back, dv.reshape(rows, Hk, d)], 1).reshape(rows, w))


PARTS = {
    "plain": {},
    "documents": dict(docs=1),
    "cap": dict(cap=6.0),
    "slopes": dict(slopes=True),
    "documents-cap": dict(docs=1, cap=6.0),
    "documents-slopes": dict(docs=1, slopes=True),
    "cap-slopes": dict(cap=6.0, slopes=True),
    "all": dict(docs=1, cap=6.0, slopes=True),
}


@pytest.mark.parametrize("d", [30, 64, 72, 104, 128])
@pytest.mark.parametrize("part", PARTS, ids=PARTS.keys())
def test_every_part_at_every_width(dev, part, d):
    kw = dict(PARTS[part])
    lq, lk = 130, 260
    if kw.pop("docs", 0):
        kw.update(qdoc=docs(1, lq, 5, 2), kdoc=docs(1, lk, 6, 2))
    both(Case(dev, 1, 4, 2, lq, lk, d, seed=31, causal=1, **kw))


@pytest.mark.parametrize("kw", [dict(causal=1, window=100), dict(window=70), dict(causal=1, window=50, prefix=[120]),
                                dict(causal=1, window=257, prefix=[3]), dict(causal=1, window=1), dict(causal=1, window=64, slopes=True)],
                         ids=str)
@pytest.mark.parametrize("s", [(1, 2, 1, 700, 700, 64), (1, 4, 1, 330, 901, 128), (1, 3, 3, 901, 330, 40), (1, 4, 1, 512, 512, 80)],
                         ids=str)
def test_windows_over_many_blocks(dev, s, kw):
    both(Case(dev, *s, seed=32, **kw))


@pytest.mark.parametrize("s", [(1, 2, 1, 16, 4000, 64), (1, 1, 1, 40, 2500, 128), (1, 4, 2, 30, 3000, 80),
                               (2, 6, 2, 1, 6000, 64), (8, 4, 4, 2, 1100, 64), (1, 8, 8, 7, 1500, 33)], ids=str)
@pytest.mark.parametrize("kw", [dict(causal=1, cap=7.0), dict(window=900, slopes=True)], ids=str)
def test_few_rows_over_many_keys(dev, s, kw):
    """dq's keys are cut into pieces, too."""
    c = Case(dev, *s, seed=38, **kw)
    both(c)
    want = c.reference()
    for got, ref, fl in zip(c.backward(acc=1, start=0.5), want[1:], (*c.floor(), 0.0)):
        near(got, ref + 0.5, floor=fl)


@pytest.mark.parametrize("lens", [(40, 16700), (16700, 40)], ids=str)
def test_more_blocks_than_are_listed(dev, lens):
    """Documents over more than 256 blocks of one side: those past the list are visited and masked key by key."""
    lq, lk = lens
    both(Case(dev, 1, 1, 1, lq, lk, 32, seed=33, qdoc=docs(1, lq, 7, 3), kdoc=docs(1, lk, 8, 3)))


@pytest.mark.parametrize("s", [(1, 4, 1, 300, 700, 64), (1, 4, 1, 300, 700, 96), (1, 8, 2, 300, 700, 128)], ids=str)
def test_accumulation_and_outputs_left_out_with_pieces(dev, s):
    """Sizes whose rows and keys are cut into pieces that a further launch joins."""
    c = Case(dev, *s, seed=34, causal=1, cap=9.0)
    want = c.reference()
    near(c.forward(), want[0])
    for got, ref, fl in zip(c.backward(acc=1, start=2.0), want[1:], (*c.floor(), 0.0)):
        near(got, ref + 2.0, floor=fl)
    for i in range(3):
        got = c.backward(want=[int(n == i) for n in range(3)])
        near(got[i], want[1 + i], floor=(*c.floor(), 0.0)[i])
        assert all((got[n] == 5.0).all() for n in range(3) if n != i)


@pytest.mark.parametrize("s", [(1, 4, 1, 300, 300, 32), (1, 4, 1, 300, 300, 96), (1, 4, 2, 600, 600, 128)], ids=str)
@pytest.mark.parametrize("ratio", [1e5, 1e12])
def test_values_of_very_different_size_at_every_width(dev, s, ratio):
    """As test_rows_of_very_different_size, in shared heads and over pieces; the larger ratio is summed row by row."""
    L = s[3]
    ids = (np.arange(L)[None] >= 150).astype(np.int32)
    c = Case(dev, *s, seed=35, causal=1, cap=12.0, qdoc=ids, kdoc=ids)
    c.v[:, 150:] *= np.float32(ratio)
    c.g[:, 150:] *= np.float32(1.0 / ratio)
    want = c.reference()
    for g, w, n in zip([c.forward()] + c.backward(), want, ("o", "dq", "dk", "dv")):
        for part in (slice(0, 150), slice(150, L)):
            near(g[:, part], w[:, part], what=(n, part))


@pytest.mark.parametrize("where", ["q", "k", "v", "g"])
def test_one_infinity_leaves_other_heads_alone(dev, where):
    """A value that the matrix products cannot hold sends its own head's rows to the plain sums, no other head's."""
    a = Case(dev, 1, 4, 2, 200, 200, 96, seed=36, causal=1)
    b = Case(dev, 1, 4, 2, 200, 200, 96, seed=36, causal=1)
    getattr(b, where)[0, 100, 0, 5] = np.inf
    want = a.reference()
    for g, w in zip([b.forward()] + b.backward(), want):
        n = g.shape[2] // 2  # the second key head and its query heads
        near(g[:, :, n:], w[:, :, n:], floor=max(a.floor()))
        assert np.isfinite(g[:, :, n:]).all()


def _drawn(n):
    r = rng_of(37, n)
    Hk, G, d = int(r.integers(1, 4)), int(r.integers(1, 5)), int(r.choice([8, 24, 32, 48, 64, 80, 96, 112, 128]))
    lq, lk = (int(np.exp(r.uniform(np.log(20), np.log(600)))) for _ in range(2))
    kw = dict(causal=int(r.integers(2)), cap=float(r.choice([0.0, 3.0, 30.0])), slopes=bool(r.integers(2)),
              window=int(r.choice([0, 0, 5, 60, 300])))
    if r.integers(2):
        kw["prefix"] = [int(r.integers(0, lk + 20))]
    if r.integers(2):
        kw.update(qdoc=docs(1, lq, n, 3), kdoc=docs(1, lk, n + 1, 3))
    return (1, Hk * G, Hk, lq, lk, d), kw


@pytest.mark.parametrize("n", range(30))
def test_drawn_rules(dev, n):
    s, kw = _drawn(n)
    print(s, {k: v for k, v in kw.items() if "doc" not in k}, flush=True)
    both(Case(dev, *s, seed=n, **kw))
