"""Every kernel of the 8-bit products and weight gradients by sizes that are known to reach it (packed8_shapes.py): values against
float64, infinities and NaN, the same bits twice, parts in scratch that two captured steps share, and contexts beside each other.

Tolerances are those that test_packed8_gpu.py derives."""
import ctypes as C

import numpy as np
import pytest

import packed8_ref as P
import packed8_shapes as S
from gpu_util import Dev
from test_packed8_gpu import EPS, Block, packed_buf, put_packed, sum_bound, wide

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return Dev()


def put_transposed(dev, x):
    """The packed transpose of x by the library, and its value laid out as x."""
    rows, cols = x.shape
    t = packed_buf(dev, cols, rows)
    dev.call("om_pack8", dev.put(x), cols, rows, cols, None, t)
    return t, np.ascontiguousarray(P.value(np.ascontiguousarray(x.T)).T)


@pytest.mark.parametrize("m,n,k", [s for s, _ in S.PRODUCTS])
def test_product(dev, m, n, k):
    rng = np.random.default_rng(m + n + k)
    (A, av), (B, bv) = put_packed(dev, wide(rng, (m, k), -3, 3)), put_packed(dev, wide(rng, (n, k), -3, 3))
    want, mag = av @ bv.T, np.abs(av) @ np.abs(bv).T
    bias, c0 = rng.normal(size=n).astype(np.float32), rng.normal(size=(m, n)).astype(np.float32)
    for use, acc in ((0, 0), (1, 1)):
        Y, Z = dev.put(c0), dev.put(c0)
        for to in (Y, Z):
            dev.call("om_gemm8", m, n, k, A, B, dev.put(bias) if use else None, to, n, acc)
        got = dev.get(Y)
        lim = sum_bound(k, mag) + 4 * EPS * (use * np.abs(bias) + acc * np.abs(c0))
        assert (np.abs(got - (want + use * bias + acc * c0)) <= lim).all()
        assert np.array_equal(got, dev.get(Z))  # the same bits twice


@pytest.mark.parametrize("m,n,k", [s for s, _ in S.SPECIAL_PRODUCTS])
def test_nan_stays_in_its_row_and_column(dev, m, n, k):
    rng = np.random.default_rng(m + n + k)
    a, b = rng.normal(size=(m, k)).astype(np.float32), rng.normal(size=(n, k)).astype(np.float32)
    r, c = min(m - 1, 3), min(n - 1, 11)
    clean = dev.empty((m, n))
    dev.call("om_gemm8", m, n, k, put_packed(dev, a)[0], put_packed(dev, b)[0], None, clean, n, 0)
    bad = np.zeros((m, n), bool)
    if m > 1:  # (of one row all would be)
        a[r, 17], bad[r] = np.inf, True
    if n > 1:
        b[c, k - 1], bad[:, c] = np.nan, True  # in the last block, which may be in a part of its own
    Y = dev.empty((m, n))
    dev.call("om_gemm8", m, n, k, put_packed(dev, a)[0], put_packed(dev, b)[0], None, Y, n, 0)
    got = dev.get(Y)
    assert np.array_equal(np.isnan(got), bad)
    assert np.array_equal(got[~bad], dev.get(clean)[~bad])


@pytest.mark.parametrize("rows,inp,out", [s for s, _ in S.WEIGHT_GRADIENTS])
def test_weight_gradient(dev, rows, inp, out):
    rng = np.random.default_rng(rows + inp + out)
    g = wide(rng, (rows, out), -4, 4)
    T, xv = put_transposed(dev, wide(rng, (rows, inp), -2, 3))
    gd = g.astype(np.float64)
    want, mag, db = gd.T @ xv, np.abs(gd).T @ np.abs(xv), gd.sum(0)
    G = dev.put(g)
    for acc in (0, 1):
        w0, b0 = rng.normal(size=(out, inp)).astype(np.float32), rng.normal(size=out).astype(np.float32)
        got = []
        for _ in range(2):
            A, B = dev.put(w0), dev.put(b0)
            dev.call("om_linear_bwd_x8", G, T, None, None, A, B, rows, inp, out, 0, acc, acc)
            got.append((dev.get(A), dev.get(B)))
        (dw, sums), again = got
        assert (np.abs(dw - (want + acc * w0)) <= 3 * sum_bound(rows, mag) + acc * 2 * EPS * np.abs(w0)).all()
        ref = db + acc * b0.astype(np.float64)
        assert (np.abs(sums - ref) <= EPS * (np.abs(ref) + acc * np.abs(db)) * 1.01 + 1e-14 * np.abs(gd).sum(0)).all()
        assert np.array_equal(dw, again[0]) and np.array_equal(sums, again[1])


@pytest.mark.parametrize("rows,inp,out", [s for s, _ in S.SPECIAL_WEIGHT_GRADIENTS])
def test_weight_gradient_of_infinities_and_extremes(dev, rows, inp, out):
    """Infinite and NaN gradients, in whole blocks and in the rows behind them, give what fp32 sums give, in their own row of dW
    alone; the largest and smallest g count; a NaN of x fills its column."""
    rng = np.random.default_rng(rows + out)
    g = rng.normal(size=(rows, out)).astype(np.float32)
    x = (1.0 + rng.random((rows, inp))).astype(np.float32)  # positive: an infinity stays one
    top, last = np.finfo(np.float32).max, rows - 1
    g[5, 3], g[7, 9] = np.inf, np.nan
    g[last, 4] = -np.inf
    g[6, 5], g[last, 5] = np.inf, -np.inf
    g[last, 6] = np.nan
    g[11, 20], g[last, 8] = top, -top  # round up to infinity in bf16
    g[:, 21] = 0.0
    g[13, 21] = 2.0 ** -126
    x[11], x[last] = 0.5, 0.5
    T, xv = put_transposed(dev, x)
    for column in (None, inp - 1):
        if column is not None:
            x[12, column] = np.nan
            T, xv = put_transposed(dev, x)
        A = dev.empty((out, inp))
        dev.call("om_linear_bwd_x8", dev.put(g), T, None, None, A, None, rows, inp, out, 0, 0, 0)
        got = dev.get(A)
        rest = [i for i in range(inp) if i != column]
        if column is not None:
            assert np.isnan(got[:, column]).all()
        if not rest:
            continue
        assert np.isposinf(got[3][rest]).all() and np.isneginf(got[4][rest]).all()
        assert np.isnan(got[np.ix_([5, 6, 9], rest)]).all()
        rows_left = [i for i in range(out) if i not in (3, 4, 5, 6, 9)]
        gd, xr = g[:, rows_left].astype(np.float64), np.ascontiguousarray(xv[:, rest])
        want, mag = gd.T @ xr, np.abs(gd).T @ np.abs(xr)
        # the fp32 instruction adds two products at a time: rows / 2 roundings
        lim = np.maximum(3 * sum_bound(rows, mag), rows * EPS * mag)
        assert (np.abs(got[np.ix_(rows_left, rest)] - want) <= lim).all()


@pytest.mark.parametrize("what,shape", [("gemm", s) for s, k in S.SPECIAL_PRODUCTS if k[-1] == "split"] +
                         [("dw", s) for s, k in S.SPECIAL_WEIGHT_GRADIENTS if k[-1] == "split"])
def test_split_calls_twice_have_the_same_bits(dev, what, shape):
    """Between the two another call leaves its own parts in the same scratch."""
    rng = np.random.default_rng(sum(shape))
    f = lambda *s: rng.normal(size=s).astype(np.float32)  # noqa: E731
    between = put_packed(dev, f(130, 9000))[0], put_packed(dev, f(260, 9000))[0], dev.empty((130, 260))
    if what == "gemm":
        m, n, k = shape
        A, B = put_packed(dev, f(m, k))[0], put_packed(dev, f(n, k))[0]
        outs = [[dev.empty((m, n))] for _ in range(2)]
        run = lambda o: dev.call("om_gemm8", m, n, k, A, B, None, o[0], n, 0)  # noqa: E731
    else:
        rows, inp, out = shape
        T, G = put_transposed(dev, f(rows, inp))[0], dev.put(f(rows, out))
        outs = [[dev.empty((out, inp)), dev.empty((out,))] for _ in range(2)]
        run = lambda o: dev.call("om_linear_bwd_x8", G, T, None, None, o[0], o[1], rows, inp, out, 0, 0, 0)  # noqa: E731
    run(outs[0])
    dev.call("om_gemm8", 130, 260, 9000, between[0], between[1], None, between[2], 260, 0)
    run(outs[1])
    for u, v in zip(*outs):
        assert np.array_equal(dev.get(u), dev.get(v))


def test_captured_steps_share_scratch(dev):
    """Two captured steps whose products and weight gradients leave parts in the context's scratch, replayed in turn with eager
    work between."""
    blocks = [Block(dev, *n, 11 + i) for i, n in enumerate(S.SPLIT_BLOCKS)]
    want = []
    for b in blocks:
        b.step()
        want.append(b.read())
    L, ctx, graphs = dev.ctx.L, dev.ctx, []
    for b in blocks:
        assert L.om_graph_capture_begin(ctx.h) == 0
        b.step()
        gr = C.c_void_p()
        assert L.om_graph_capture_end(ctx.h, C.byref(gr)) == 0
        graphs.append(gr)
    try:
        vals = (C.c_float * 3)()
        for turn in range(4):
            for b in blocks:
                for k in Block.NAMES:
                    dev.call("om_fill", b.t[k], float(turn + 3), int(np.prod(b.t[k].shape)))
            for gr in graphs if turn % 2 else graphs[::-1]:
                assert L.om_graph_launch(gr, vals) == 0
            ctx.sync()
            for b, w in zip(blocks, want):
                got = b.read()
                for k in Block.NAMES:
                    assert np.array_equal(got[k], w[k]), (turn, k)
            blocks[turn % 2].step()
    finally:
        for gr in graphs:
            L.om_graph_destroy(gr)


def test_two_contexts_beside_each_other():
    """Steps whose parts are in each context's own scratch, side by side, against each context alone."""
    devs = [Dev(), Dev()]
    blocks = [Block(d, *S.SPLIT_BLOCKS[0], 21 + i) for i, d in enumerate(devs)]
    want = []
    for d, b in zip(devs, blocks):
        b.step()
        d.ctx.sync()
        want.append(b.read())
    for turn in range(5):
        for b in blocks if turn % 2 else blocks[::-1]:
            b.step()
        for b in blocks:
            b.step()
        for b, w in zip(blocks, want):
            got = b.read()
            for k in Block.NAMES:
                assert np.array_equal(got[k], w[k]), (turn, k)


def test_a_block_whose_sums_are_split(dev):
    """Every stage of such a block against float64 from the values that the stage before left."""
    B = Block(dev, *S.SPLIT_BLOCKS[0], 31)
    B.step()
    r, p = B.read(), B.h
    f64 = {k: v.astype(np.float64) for k, v in {**p, **r}.items()}
    T = lambda v: P.value(np.ascontiguousarray(v.T)).T  # noqa: E731
    want = {"dw2": T(p["g"]).T @ T(r["a"]), "db2": f64["g"].sum(0), "dw1": f64["dh"].T @ T(r["y"]), "db1": f64["dh"].sum(0),
            "h": P.value(r["y"]) @ P.value(p["w1"]).T + f64["b1"], "da": P.value(p["g"]) @ T(p["w2"]), "dy": f64["dh"] @ f64["w1"]}
    for k, v in want.items():  # fp32 sums of random sign: 1e-6 in the 2-norm
        assert np.linalg.norm(r[k] - v) <= 1e-6 * np.linalg.norm(v), k
