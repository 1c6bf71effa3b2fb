"""8-bit tensors on the GPU: packing and unpacking against their definition byte for byte, the products of packed tensors,
a Linear's weight gradient from a packed input, GELU and LayerNorm that keep packed tensors, against float64.

Tolerances are derived at each check. EPS = 2^-24 is half a step of fp32 relative to the value."""
import ctypes as C

import numpy as np
import pytest

import packed8_ref as P
from gpu_util import Dev

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24


@pytest.fixture(scope="module")
def dev():
    return Dev()


def wide(rng, shape, lo=-40, hi=40):
    """Normal values over many binades."""
    return (rng.normal(size=shape) * np.exp2(rng.integers(lo, hi, shape).astype(np.float64))).astype(np.float32)


def packed_buf(dev, rows, cols, guard=64):
    return dev.empty((P.nbytes(rows, cols) + guard,), np.uint8, fill=0xA5)


def read_packed(dev, buf, rows, cols):
    raw = dev.get(buf)
    n = P.nbytes(rows, cols)
    assert (raw[n:] == 0xA5).all(), "bytes behind the packed tensor"
    return raw[:n]


def check_packed(raw, x):
    rows, cols = x.shape
    v, codes, scales = P.decode(raw, rows, cols)
    want, e = P.pack(x)
    assert np.array_equal(scales[:, :e.shape[1]].astype(int) - 127, e)
    assert not scales[:, e.shape[1]:].any() and not codes[:, cols:].any()
    assert np.array_equal(np.isnan(v), np.isnan(want))
    ok = ~np.isnan(want)
    assert np.array_equal(v[ok], want[ok])
    assert np.array_equal(np.signbit(v[ok]), np.signbit(x[ok]))


SHAPES = [(1, 1), (1, 128), (3, 5), (2, 129), (64, 256), (127, 127), (128, 128), (129, 130), (7, 512), (5, 513), (300, 77),
          (33, 1000), (640, 384), (4001, 1100), (1501, 1502), (20000, 130)]


@pytest.mark.parametrize("rows,cols", SHAPES)
def test_pack_and_unpack(dev, rows, cols):
    rng = np.random.default_rng(rows * 1009 + cols)
    for pad, make in ((0, lambda s: rng.normal(size=s).astype(np.float32)), (3, lambda s: wide(rng, s))):
        x = make((rows, cols + pad))
        X = dev.put(x)
        xs = x[:, :cols]
        for form in ("rows", "cols", "both"):
            a = packed_buf(dev, rows, cols) if form != "cols" else None
            t = packed_buf(dev, cols, rows) if form != "rows" else None
            dev.call("om_pack8", X, cols + pad, rows, cols, a, t)
            if a is not None:
                check_packed(read_packed(dev, a, rows, cols), xs)
            if t is not None:
                check_packed(read_packed(dev, t, cols, rows), np.ascontiguousarray(xs.T))
            if form == "rows":
                for acc in (0, 1):
                    y0 = rng.normal(size=(rows, cols + 2 * pad)).astype(np.float32)
                    Y = dev.put(y0)
                    dev.call("om_unpack8", a, Y, cols + 2 * pad, rows, cols, acc)
                    got, v = dev.get(Y), P.value(xs).astype(np.float32)
                    assert np.array_equal(got[:, :cols], y0[:, :cols] + v if acc else v)
                    assert np.array_equal(got[:, cols:], y0[:, cols:])


def test_pack_special_values(dev):
    """Zeros, subnormals, the largest values, ties, infinities and NaN, alone in a block and beside others."""
    tiny = np.float32(2.0) ** np.float32(-149)
    rows = [np.zeros(128), np.full(128, -0.0), np.full(128, tiny), np.full(128, np.finfo(np.float32).max),
            np.full(128, 448.0), np.full(128, np.nextafter(np.float32(448), np.float32(500))),
            np.full(128, np.nan), np.full(128, np.inf), np.linspace(-1, 1, 128) * 2.0 ** -140,
            np.concatenate([[np.inf, -np.inf, np.nan], np.linspace(-3, 3, 125)]),
            np.concatenate([[448.0], (np.arange(127) + 0.5) * 2.0 ** -9]),       # ties among the subnormal codes
            np.concatenate([[256.0], 16.0 + np.arange(127) * 0.5]),             # ties among the normal ones
            np.concatenate([[2.0 ** 127], np.full(127, 2.0 ** -126)])]
    x = np.stack(rows).astype(np.float32)
    X = dev.put(x)
    a, t = packed_buf(dev, *x.shape), packed_buf(dev, *x.shape[::-1])
    dev.call("om_pack8", X, 128, len(rows), 128, a, t)
    check_packed(read_packed(dev, a, *x.shape), x)
    check_packed(read_packed(dev, t, *x.shape[::-1]), np.ascontiguousarray(x.T))
    Y = dev.empty(x.shape)
    dev.call("om_unpack8", a, Y, 128, len(rows), 128, 0)
    assert np.array_equal(dev.get(Y), P.value(x).astype(np.float32), equal_nan=True)


def test_pack_every_code(dev):
    """Each finite code's value at every scale comes back as it is."""
    codes = np.array([c for c in range(256) if (c & 127) != 127], np.uint8)
    v = np.concatenate([P.CODES[codes], np.full(256 - len(codes), 448.0)])
    e = np.arange(-118, 119)
    x = (v[None] * np.exp2(e[:, None].astype(np.float64))).astype(np.float32)
    x[:, 128] = x[:, 255] = 448.0 * np.exp2(e.astype(np.float64))
    x[:, 0] = x[:, 127] = x[:, 255]
    a, Y = packed_buf(dev, *x.shape), dev.empty(x.shape)
    dev.call("om_pack8", dev.put(x), 256, len(e), 256, a, None)
    dev.call("om_unpack8", a, Y, 256, len(e), 256, 0)
    assert np.array_equal(dev.get(Y), x)


def test_packed_bytes(dev):
    L = dev.ctx.L
    for rows, cols in SHAPES + [(0, 5), (5, 0), (-1, 5), (2000000000, 2000000000)]:
        want = P.nbytes(rows, cols) if rows > 0 and cols > 0 else 0
        assert L.om_pack8_bytes(rows, cols) == want
    assert np.array_equal(P.encode(np.array([[1.0, -448.0]], np.float32))[:2], [0x38, 0xFE])


def test_empty_calls_do_nothing(dev):
    Y = dev.empty((4, 4), fill=7.0)
    B = dev.empty((64,), np.uint8, fill=0xA5)
    dev.call("om_pack8", None, 4, 0, 4, B, None)
    dev.call("om_pack8", None, 4, 4, 0, None, B)
    dev.call("om_unpack8", None, Y, 4, 0, 4, 1)
    dev.call("om_gelu_fwd_x8", None, Y, B, 0, 4)
    dev.call("om_gelu_bwd_x8", None, None, Y, 4, 0, 0)
    dev.call("om_layernorm_fwd_x8", None, None, None, Y, B, None, 0, 4, 1e-5)
    dev.call("om_gemm8", 0, 4, 8, None, None, None, Y, 4, 0)
    dev.call("om_gemm8", 4, 0, 8, None, None, None, Y, 4, 0)
    assert (dev.get(Y) == 7.0).all() and (dev.get(B) == 0xA5).all()


# ------------------------------------------------------------------------------------------------------------ products
def put_packed(dev, x):
    """x packed by the library, and its value."""
    rows, cols = x.shape
    buf = packed_buf(dev, rows, cols)
    dev.call("om_pack8", dev.put(x), cols, rows, cols, buf, None)
    return buf, P.value(x)


def sum_bound(k, mag, extra=4):
    """Products are exact. Every 16 of them enter an fp32 sum with one rounding, at most a step (2 EPS) of the largest partial
    sum, which the magnitudes' sum bounds; `extra`: joining parts, bias, C."""
    return (-(-k // 128) * 8 + 256 + extra) * 2 * EPS * mag


PRODUCTS = [(1, 1, 1), (3, 5, 7), (1, 300, 1000), (8, 70, 129), (16, 16, 4096), (17, 33, 640), (40, 100, 2000), (64, 64, 256),
            (65, 64, 128), (100, 130, 50), (128, 128, 128), (129, 257, 384), (300, 260, 1100), (512, 512, 513),
            (1536, 384, 4096), (700, 900, 300), (2100, 2050, 130), (4096, 4100, 128),
            # every tile with k in one part and in several
            (777, 1000, 100), (9, 40, 9000), (17, 20, 5000), (17, 20, 16500), (33, 1537, 16500), (500, 2050, 2600),
            (260, 1000, 9000), (70, 1000, 5000), (3503, 3501, 300), (6001, 2050, 300), (1537, 2050, 1300), (777, 1000, 9000),
            (1001, 4093, 100), (1001, 1000, 5000), (4099, 33, 16500), (4099, 33, 5000), (130, 1000, 9000), (130, 260, 9000),
            (4093, 4093, 520), (777, 333, 1000), (260, 500, 2000),
            # up to 48 rows, four and eight wavefronts, and past them
            (16, 4200, 300), (31, 257, 8192), (32, 5000, 200), (48, 4500, 700), (47, 30, 5000), (47, 30, 6100), (50, 300, 3000), (64, 4200, 130)]


@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_product(dev, m, n, k):
    rng = np.random.default_rng(m * 7 + n * 3 + k)
    a, b = wide(rng, (m, k), -3, 3), wide(rng, (n, k), -3, 3)
    bias = rng.normal(size=n).astype(np.float32)
    (A, av), (B, bv) = put_packed(dev, a), put_packed(dev, b)
    want, mag = av @ bv.T, np.abs(av) @ np.abs(bv).T
    for use_bias, acc, pad in ((False, 0, 0), (True, 1, 5)):
        c0 = rng.normal(size=(m, n + pad)).astype(np.float32)
        Cb = dev.put(c0)
        dev.call("om_gemm8", m, n, k, A, B, dev.put(bias) if use_bias else None, Cb, n + pad, acc)
        got = dev.get(Cb)
        ref = want + (bias if use_bias else 0) + (c0[:, :n] if acc else 0)
        lim = sum_bound(k, mag) + 4 * EPS * (np.abs(bias) * use_bias + acc * np.abs(c0[:, :n]))
        assert (np.abs(got[:, :n] - ref) <= lim + 1e-30).all(), float(np.abs(got[:, :n] - ref).max())
        assert np.array_equal(got[:, n:], c0[:, n:])
        # in the 2-norm a sum of k / 16 roundings of random sign stays far below the worst case
        assert np.linalg.norm(got[:, :n] - ref) <= 1e-6 * np.linalg.norm(np.sqrt(np.square(av) @ np.square(bv).T)) + 1e-6 * acc * np.linalg.norm(c0)


def test_product_of_wide_ranges(dev):
    """Scales far apart within a row, and operands whose products, not they themselves, are ordinary."""
    rng = np.random.default_rng(4)
    for la, lb in ((-30, 30), (-100, -90), (90, 100)):
        a, b = wide(rng, (70, 700), la, lb), wide(rng, (50, 700), -lb, -la)
        (A, av), (B, bv) = put_packed(dev, a), put_packed(dev, b)
        Y = dev.empty((70, 50))
        dev.call("om_gemm8", 70, 50, 700, A, B, None, Y, 50, 0)
        # values of a block that fall below bf16's smallest normal count as zero or as they are; none does here
        assert (np.abs(dev.get(Y) - av @ bv.T) <= sum_bound(700, np.abs(av) @ np.abs(bv).T)).all()


def test_product_of_the_smallest_scales(dev):
    """Blocks with the least exponents: values from 2^-126 on count in full."""
    x = np.zeros((33, 130), np.float32)
    x[:, :] = np.float32(2.0 ** -126) * (1 + np.arange(130) % 3)
    w = np.full((40, 130), 2.0 ** 100, np.float32)
    (A, av), (B, bv) = put_packed(dev, x), put_packed(dev, w)
    Y = dev.empty((33, 40))
    dev.call("om_gemm8", 33, 40, 130, A, B, None, Y, 40, 0)
    assert (np.abs(dev.get(Y) - av @ bv.T) <= sum_bound(130, np.abs(av) @ np.abs(bv).T)).all()


@pytest.mark.parametrize("m,n", [(5, 40), (150, 200)])
def test_nan_stays_in_its_row_and_column(dev, m, n):
    rng = np.random.default_rng(2)
    k = 300
    a, b = rng.normal(size=(m, k)).astype(np.float32), rng.normal(size=(n, k)).astype(np.float32)
    a[3, 17], b[11, 299] = np.inf, np.nan
    (A, av), (B, bv) = put_packed(dev, a), put_packed(dev, b)
    Y = dev.empty((m, n))
    dev.call("om_gemm8", m, n, k, A, B, None, Y, n, 0)
    bad = np.zeros((m, n), bool)
    bad[3], bad[:, 11] = True, True
    assert np.array_equal(np.isnan(dev.get(Y)), bad)


def test_product_over_nothing(dev):
    """k = 0: the bias, and C where it is kept."""
    rng = np.random.default_rng(6)
    for m, n in ((3, 5), (140, 150)):
        bias, c0 = rng.normal(size=n).astype(np.float32), rng.normal(size=(m, n)).astype(np.float32)
        for b, acc in ((None, 0), (bias, 0), (None, 1), (bias, 1)):
            Y = dev.put(c0)
            dev.call("om_gemm8", m, n, 0, None, None, dev.put(b) if b is not None else None, Y, n, acc)
            want = np.zeros((m, n), np.float32) + (b if b is not None else np.float32(0))
            assert np.array_equal(dev.get(Y), c0 + want if acc else want)


def test_the_same_product_twice_has_the_same_bits(dev):
    rng = np.random.default_rng(8)
    for m, n, k in ((4, 512, 4096), (384, 640, 4096), (1000, 300, 1000)):
        (A, _), (B, _) = put_packed(dev, rng.normal(size=(m, k)).astype(np.float32)), put_packed(
            dev, rng.normal(size=(n, k)).astype(np.float32))
        Y, Z = dev.empty((m, n)), dev.empty((m, n))
        dev.call("om_gemm8", m, n, k, A, B, None, Y, n, 0)
        dev.call("om_gemm8", m, n, k, A, B, None, Z, n, 0)
        assert np.array_equal(dev.get(Y), dev.get(Z))


# ----------------------------------------------------------------------------------------------------- weight gradient
def dw_case(dev, rng, rows, inp, out, g):
    x = wide(rng, (rows, inp), -2, 3)
    t = packed_buf(dev, inp, rows)
    dev.call("om_pack8", dev.put(x), inp, rows, inp, None, t)
    return t, P.value(np.ascontiguousarray(x.T)).T


DW = [(1, 1, 1), (2, 3, 5), (37, 20, 33), (127, 64, 64), (128, 128, 128), (129, 130, 257), (300, 77, 40), (1000, 384, 100),
      (4096, 384, 1536), (2500, 512, 2100), (640, 1000, 333), (64, 2048, 2304),
      # fewer than four columns of g, and rows just past whole blocks
      (129, 20, 1), (257, 40, 2), (384, 33, 3), (130, 7, 1), (131, 9, 2), (3, 5, 2), (512, 140, 1), (300, 50, 5), (640, 64, 70),
      # every tile with the rows in one part and in several, the last of them short
      (100, 1537, 1000), (2600, 260, 777), (5003, 777, 130), (9001, 130, 130), (5003, 1, 1), (9001, 260, 33), (9001, 33, 2),
      (2600, 1000, 260), (5003, 500, 1000), (9001, 1000, 500), (16390, 260, 500), (300, 300, 300), (1300, 33, 260), (16390, 20, 5)]


@pytest.mark.parametrize("rows,inp,out", DW)
def test_weight_gradient(dev, rows, inp, out):
    rng = np.random.default_rng(rows + 5 * inp + 11 * out)
    g = wide(rng, (rows, out), -4, 4)
    T, xv = dw_case(dev, rng, rows, inp, out, g)
    G = dev.put(g)
    want, mag = g.astype(np.float64).T @ xv, np.abs(g.astype(np.float64)).T @ np.abs(xv)
    db = g.astype(np.float64).sum(0)
    for acc in (0, 1):
        w0, b0 = rng.normal(size=(out, inp)).astype(np.float32), rng.normal(size=out).astype(np.float32)
        DW_, DB = dev.put(w0), dev.put(b0)
        dev.call("om_linear_bwd_x8", G, T, None, None, DW_, DB, rows, inp, out, 0, acc, acc)
        # g's three parts hold all its bits: three roundings where sum_bound counts one
        lim = 3 * sum_bound(rows, mag) + acc * 2 * EPS * np.abs(w0)
        got = dev.get(DW_)
        assert (np.abs(got - (want + acc * w0)) <= lim).all()
        assert np.linalg.norm(got - (want + acc * w0)) <= 1e-6 * np.linalg.norm(
            np.sqrt(np.square(g.astype(np.float64)).T @ np.square(xv))) + acc * 1e-6 * np.linalg.norm(w0)
        # the sum is double, rounded once; where it is kept, one more addition
        ref = db + acc * b0.astype(np.float64)
        assert (np.abs(dev.get(DB) - ref) <= EPS * (np.abs(ref) + acc * np.abs(db)) * 1.01 + 1e-14 * np.abs(g).sum(0)).all()


def test_weight_gradient_parts_and_dx(dev):
    """Each output alone; dx is om_linear_bwd's, bit for bit."""
    rng = np.random.default_rng(31)
    rows, inp, out = 300, 96, 160
    g, w = rng.normal(size=(rows, out)).astype(np.float32), rng.normal(size=(out, inp)).astype(np.float32)
    T, _ = dw_case(dev, rng, rows, inp, out, g)
    G, W = dev.put(g), dev.put(w)
    dx0 = rng.normal(size=(rows, inp)).astype(np.float32)
    for acc in (0, 1):
        X1, X2 = dev.put(dx0), dev.put(dx0)
        dev.call("om_linear_bwd", G, None, W, X1, None, None, rows, inp, out, acc, 0, 0)
        A, B = dev.empty((out, inp)), dev.empty((out,))
        dev.call("om_linear_bwd_x8", G, T, W, X2, A, B, rows, inp, out, acc, 0, 0)
        assert np.array_equal(dev.get(X1), dev.get(X2))
        A2, B2 = dev.empty((out, inp)), dev.empty((out,))
        dev.call("om_linear_bwd_x8", G, T, None, None, A2, None, rows, inp, out, 0, 0, 0)
        dev.call("om_linear_bwd_x8", G, None, None, None, None, B2, rows, inp, out, 0, 0, 0)
        assert np.array_equal(dev.get(A), dev.get(A2)) and np.array_equal(dev.get(B), dev.get(B2))
    dev.call("om_linear_bwd_x8", G, None, None, None, None, None, rows, inp, out, 0, 0, 0)


def test_weight_gradient_of_no_rows(dev):
    A, B = dev.empty((3, 4), fill=2.0), dev.empty((3,), fill=2.0)
    dev.call("om_linear_bwd_x8", None, None, None, None, A, B, 0, 4, 3, 0, 1, 1)
    assert (dev.get(A) == 2.0).all() and (dev.get(B) == 2.0).all()
    dev.call("om_linear_bwd_x8", None, None, None, None, A, B, 0, 4, 3, 0, 0, 0)
    assert not dev.get(A).any() and not dev.get(B).any()


@pytest.mark.parametrize("rows,inp,out", [(200, 64, 96), (3000, 300, 40)])
def test_weight_gradient_of_infinities_and_extremes(dev, rows, inp, out):
    """Infinite and NaN gradients give what fp32 sums give, in their own row of dW alone; the largest and smallest g count."""
    rng = np.random.default_rng(rows)
    g = rng.normal(size=(rows, out)).astype(np.float32)
    x = (1.0 + rng.random((rows, inp))).astype(np.float32)  # positive: an infinity stays one
    g[5, 3], g[7, 9] = np.inf, np.nan
    g[11, 20] = np.finfo(np.float32).max     # rounds up to infinity in bf16
    g[:, 21] = 0.0
    g[13, 21] = 2.0 ** -126
    x[11, :] = 0.5
    t = packed_buf(dev, inp, rows)
    dev.call("om_pack8", dev.put(x), inp, rows, inp, None, t)
    xv = P.value(np.ascontiguousarray(x.T)).T
    A = dev.empty((out, inp))
    dev.call("om_linear_bwd_x8", dev.put(g), t, None, None, A, None, rows, inp, out, 0, 0, 0)
    got = dev.get(A)
    assert np.isposinf(got[3]).all() and np.isnan(got[9]).all()
    rest = [i for i in range(out) if i not in (3, 9)]
    gd = g[:, rest].astype(np.float64)
    want, mag = gd.T @ xv, np.abs(gd).T @ np.abs(xv)
    # the fp32 instruction adds two products at a time: rows / 2 roundings
    lim = np.maximum(3 * sum_bound(rows, mag), rows * EPS * mag)
    assert (np.abs(got[rest] - want) <= lim).all()


# column sums in one launch and in two, by single columns and by four
@pytest.mark.parametrize("rows,cols", [(1, 1), (64, 300), (65, 17), (777, 333), (1024, 2048), (1025, 130), (1023, 2052), (64, 8193),
                                       (4097, 768), (70, 16001)])
def test_column_sums(dev, rows, cols):
    rng = np.random.default_rng(rows + cols)
    g, old = wide(rng, (rows, cols), -4, 4), rng.normal(size=cols).astype(np.float32)
    want, size = g.astype(np.float64).sum(0), np.abs(g.astype(np.float64)).sum(0)
    G = dev.put(g)
    for acc in (0, 1):
        B = dev.put(old)
        dev.call("om_colsum", G, B, rows, cols, acc)
        # a double sum rounded once, and one more addition where the old value is kept
        ref = want + acc * old.astype(np.float64)
        assert (np.abs(dev.get(B) - ref) <= EPS * (np.abs(ref) + acc * np.abs(want)) * 1.01 + 1e-14 * size).all()


# ------------------------------------------------------------------------------------------------- GELU and LayerNorm
@pytest.mark.parametrize("mode", [0, 1])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 130), (64, 256), (33, 1000), (700, 77), (5, 4096)])
def test_gelu(dev, mode, rows, cols):
    rng = np.random.default_rng(rows + cols)
    x = (3.0 * rng.normal(size=(rows, cols))).astype(np.float32)
    g = rng.normal(size=(rows, cols)).astype(np.float32)
    L = dev.ctx.L
    try:
        assert L.om_ctx_set_gelu(dev.ctx.h, mode) == 0
        X, Y, Q, G = dev.put(x), dev.empty(x.shape), packed_buf(dev, rows, cols), dev.put(g)
        Y0, D0 = dev.empty(x.shape), dev.empty(x.shape)
        dev.call("om_gelu_fwd_x8", X, Y, Q, rows, cols)
        check_packed(read_packed(dev, Q, rows, cols), x)
        dev.call("om_gelu_fwd", X, Y0, x.size)
        assert np.array_equal(dev.get(Y), dev.get(Y0))  # the bits of om_gelu_fwd
        h = P.value(x).astype(np.float32)
        H = dev.put(h)
        for acc in (0, 1):
            d0 = rng.normal(size=x.shape).astype(np.float32)
            D, E = dev.put(d0), dev.put(d0)
            dev.call("om_gelu_bwd_x8", G, Q, D, rows, cols, acc)
            dev.call("om_gelu_bwd", G, H, E, x.size, acc)  # the bits of om_gelu_bwd at the kept values
            assert np.array_equal(dev.get(D), dev.get(E))
            if not acc:  # the slope is within 2.2e-7, the product rounds once
                lim = np.abs(g) * (2.2e-7 + 4 * EPS)
                assert (np.abs(dev.get(D) - g.astype(np.float64) * P.gelu_slope(h)) <= lim).all()
        # in place
        dev.call("om_gelu_bwd_x8", G, Q, G, rows, cols, 0)
        dev.call("om_gelu_bwd", dev.put(g), H, D0, x.size, 0)
        assert np.array_equal(dev.get(G), dev.get(D0))
        dev.call("om_gelu_fwd_x8", X, X, Q, rows, cols)
        assert np.array_equal(dev.get(X), dev.get(Y0))
        check_packed(read_packed(dev, Q, rows, cols), x)
    finally:
        L.om_ctx_set_gelu(dev.ctx.h, 0)


def test_gelu_gradient_against_differences(dev):
    """At inputs that 8 bits hold exactly the backward is GELU's own derivative."""
    v = P.CODES[(np.abs(P.CODES) >= 2.0 ** -6) & (np.abs(P.CODES) <= 8.0)]
    x = np.zeros((1, 256), np.float32)
    x[0, :len(v)] = v
    Q, Y, D = packed_buf(dev, 1, 256), dev.empty(x.shape), dev.empty(x.shape)
    dev.call("om_gelu_fwd_x8", dev.put(x), Y, Q, 1, 256)
    dev.call("om_gelu_bwd_x8", dev.put(np.ones_like(x)), Q, D, 1, 256, 0)
    h = 1e-5
    diff = (P.gelu(x.astype(np.float64) + h) - P.gelu(x.astype(np.float64) - h)) / (2 * h)
    # the difference's own error: h^2 / 6 of the third derivative (below 2), and 1e-16 |x| / h
    assert np.abs(dev.get(D) - diff).max() <= 2.2e-7 + 4 * EPS + h * h + 1e-10


NORMS = [(1, 1), (1, 7), (3, 128), (5, 130), (64, 256), (33, 384), (130, 500), (70, 768), (9, 1023), (40, 1024), (21, 1025),
         (17, 2047), (12, 3000), (600, 4096), (5, 5000), (3, 8192), (4, 8200), (2, 16384), (3, 20000),
         # one workgroup, a few rows to each, and many
         (24, 384), (32, 512), (33, 100), (25, 640), (64, 1100), (300, 2048), (100, 5000), (3000, 130), (2100, 1030), (9000, 64)]


@pytest.mark.parametrize("rows,cols", NORMS)
def test_layernorm(dev, rows, cols):
    rng = np.random.default_rng(rows * 31 + cols)
    x = (rng.normal(size=(rows, cols)) * np.exp(rng.normal(size=cols)) + rng.normal(size=(rows, 1))).astype(np.float32)
    g = rng.normal(size=(rows, cols)).astype(np.float32)
    gamma, beta = (1 + 0.3 * rng.normal(size=cols)).astype(np.float32), rng.normal(size=cols).astype(np.float32)
    eps = 1e-5
    xh, rstd = P.layernorm(x, eps)
    X, GA, BE, Y, Q, R = dev.put(x), dev.put(gamma), dev.put(beta), dev.empty(x.shape), packed_buf(dev, rows, cols), dev.empty((rows,))
    dev.call("om_layernorm_fwd_x8", X, GA, BE, Y, Q, R, rows, cols, eps)
    # statistics are double, of relative error 1e-14, and rounded once: the same floats but where one lies that near to a tie
    assert np.array_equal(dev.get(R), rstd[:, 0])
    check_packed(read_packed(dev, Q, rows, cols), xh)
    y = xh * gamma + beta
    assert np.array_equal(dev.get(Y), y)
    h = P.value(xh)
    dx, dgamma, dbeta = P.layernorm_bwd(g, h, gamma, rstd)
    q = np.abs(g.astype(np.float64) * gamma)
    # q rounds once; a row's sums have at most cols / 256 + 16 roundings in sequence of up to its magnitudes' sum, joined in
    # six to nine more; then four operations
    n = cols / 256 + 32
    lim = rstd * EPS * (6 * q + n * q.mean(1, keepdims=True) + (n + 6) * np.abs(h) * (q * np.abs(h)).mean(1, keepdims=True))
    G = dev.put(g)
    for acc in (0, 1):
        d0, a0, b0 = (rng.normal(size=s).astype(np.float32) for s in (x.shape, cols, cols))
        D, A, B = dev.put(d0), dev.put(a0), dev.put(b0)
        dev.call("om_layernorm_bwd_x8", G, Q, GA, R, D, A, B, rows, cols, acc, acc)
        assert (np.abs(dev.get(D) - (dx + acc * d0)) <= lim + acc * 2 * EPS * (np.abs(d0) + np.abs(dx))).all()
        for got, want, old, size in ((dev.get(A), dgamma, a0, np.abs(g * h).sum(0)), (dev.get(B), dbeta, b0, np.abs(g).sum(0))):
            ref = want + acc * old.astype(np.float64)
            assert (np.abs(got - ref) <= 1.01 * EPS * (np.abs(ref) + acc * np.abs(want)) + 1e-14 * size).all()
    # each output alone has the same bits; in place
    D, A, B = dev.empty(x.shape), dev.empty((cols,)), dev.empty((cols,))
    D2, A2, B2 = dev.empty(x.shape), dev.empty((cols,)), dev.empty((cols,))
    dev.call("om_layernorm_bwd_x8", G, Q, GA, R, D, A, B, rows, cols, 0, 0)
    dev.call("om_layernorm_bwd_x8", G, Q, GA, R, D2, None, None, rows, cols, 0, 0)
    dev.call("om_layernorm_bwd_x8", G, Q, GA, R, None, A2, None, rows, cols, 0, 0)
    dev.call("om_layernorm_bwd_x8", G, Q, GA, R, None, None, B2, rows, cols, 0, 0)
    for u, v in ((D, D2), (A, A2), (B, B2)):
        assert np.array_equal(dev.get(u), dev.get(v))
    dev.call("om_layernorm_bwd_x8", G, Q, GA, R, G, A2, B2, rows, cols, 0, 0)
    assert np.array_equal(dev.get(G), dev.get(D)) and np.array_equal(dev.get(A2), dev.get(A))
    dev.call("om_layernorm_fwd_x8", X, GA, BE, X, Q, R, rows, cols, eps)
    assert np.array_equal(dev.get(X), y)


def test_layernorm_of_constant_and_broken_rows(dev):
    """A constant row gives zeros; a NaN or an infinity makes its own row NaN and no other."""
    x = np.random.default_rng(1).normal(size=(4, 200)).astype(np.float32)
    x[0] = 3.0
    x[1, 5], x[2, 7] = np.nan, np.inf
    ga, be = np.ones(200, np.float32), np.zeros(200, np.float32)
    Y, Q, R, D = dev.empty(x.shape), packed_buf(dev, 4, 200), dev.empty((4,)), dev.empty(x.shape)
    dev.call("om_layernorm_fwd_x8", dev.put(x), dev.put(ga), dev.put(be), Y, Q, R, 4, 200, 1e-5)
    got = dev.get(Y)
    assert not got[0].any() and np.isnan(got[1:3]).all() and np.isfinite(got[3]).all()
    dev.call("om_layernorm_bwd_x8", dev.put(np.ones_like(x)), Q, dev.put(ga), R, D, None, None, 4, 200, 0, 0)
    d = dev.get(D)
    assert np.isfinite(d[[0, 3]]).all() and np.isnan(d[1:3]).all()


def test_layernorm_backward_of_no_rows(dev):
    A, B = dev.empty((5,), fill=2.0), dev.empty((5,), fill=2.0)
    dev.call("om_layernorm_bwd_x8", None, None, None, None, None, A, B, 0, 5, 0, 1)
    assert (dev.get(A) == 2.0).all() and (dev.get(B) == 2.0).all()
    dev.call("om_layernorm_bwd_x8", None, None, None, None, None, A, B, 0, 5, 0, 0)
    assert not dev.get(A).any() and not dev.get(B).any()


# -------------------------------------------------------------------------------------------------------- used together
class Block:
    """A pre-norm feed-forward block, x + Linear(GELU(Linear(LayerNorm(x)))), that keeps its activations in 8 bits and
    multiplies packed tensors, as a training step calls it."""

    def __init__(self, dev, rows, width, hidden, seed):
        rng = np.random.default_rng(seed)
        f = lambda *s, std=1.0: (std * rng.normal(size=s)).astype(np.float32)  # noqa: E731
        self.d, self.n = dev, (rows, width, hidden)
        self.h = {"x": f(rows, width), "gamma": 1 + f(width, std=0.1), "beta": f(width, std=0.1),
                  "w1": f(hidden, width, std=width ** -0.5), "b1": f(hidden, std=0.1),
                  "w2": f(width, hidden, std=hidden ** -0.5), "b2": f(width, std=0.1), "g": f(rows, width, std=1 / rows)}
        self.t = {k: dev.put(v) for k, v in self.h.items()}
        e = dev.empty
        self.t.update(y=e((rows, width)), h=e((rows, hidden)), a=e((rows, hidden)), o=e((rows, width)), rstd=e((rows,)),
                      da=e((rows, hidden)), dh=e((rows, hidden)), dy=e((rows, width)), dx=e((rows, width)),
                      dw1=e((hidden, width)), db1=e((hidden,)), dw2=e((width, hidden)), db2=e((width,)),
                      dgamma=e((width,)), dbeta=e((width,)))
        for name, (r, c) in {"xh8": (rows, width), "y8": (rows, width), "yt8": (width, rows), "h8": (rows, hidden),
                             "a8": (rows, hidden), "at8": (hidden, rows), "w18": (hidden, width), "w1t8": (width, hidden),
                             "w28": (width, hidden), "w2t8": (hidden, width), "g8": (rows, width), "gt8": (width, rows),
                             "dh8": (rows, hidden), "dht8": (hidden, rows)}.items():
            self.t[name] = packed_buf(dev, r, c, 0)

    def step(self):
        rows, width, hidden = self.n
        t = self.t

        def call(name, *a):
            self.d.call(name, *[t[x] if isinstance(x, str) else x for x in a])

        call("om_layernorm_fwd_x8", "x", "gamma", "beta", "y", "xh8", "rstd", rows, width, 1e-5)
        call("om_pack8", "y", width, rows, width, "y8", "yt8")
        call("om_pack8", "w1", width, hidden, width, "w18", "w1t8")
        call("om_pack8", "w2", hidden, width, hidden, "w28", "w2t8")
        call("om_gemm8", rows, hidden, width, "y8", "w18", "b1", "h", hidden, 0)
        call("om_gelu_fwd_x8", "h", "a", "h8", rows, hidden)
        call("om_pack8", "a", hidden, rows, hidden, "a8", "at8")
        call("om_copy", "o", "x", 4 * rows * width)
        call("om_gemm8", rows, width, hidden, "a8", "w28", "b2", "o", width, 1)
        # backward: the second Linear with all products in 8 bits, the first with its weight gradient from the kept input
        call("om_pack8", "g", width, rows, width, "g8", "gt8")
        call("om_gemm8", rows, hidden, width, "g8", "w2t8", None, "da", hidden, 0)
        call("om_gemm8", width, hidden, rows, "gt8", "at8", None, "dw2", hidden, 0)
        call("om_colsum", "g", "db2", rows, width, 0)
        call("om_gelu_bwd_x8", "da", "h8", "dh", rows, hidden, 0)
        call("om_linear_bwd_x8", "dh", "yt8", "w1", "dy", "dw1", "db1", rows, width, hidden, 0, 0, 0)
        call("om_copy", "dx", "g", 4 * rows * width)
        call("om_layernorm_bwd_x8", "dy", "xh8", "gamma", "rstd", "dx", "dgamma", "dbeta", rows, width, 1, 0)

    NAMES = ("o", "dx", "dw1", "db1", "dw2", "db2", "dgamma", "dbeta", "y", "h", "a", "da", "dh", "dy", "rstd")

    def read(self):
        return {k: self.d.get(self.t[k]) for k in self.NAMES}


def test_a_block_trains_in_8_bits(dev):
    """Every stage of the block against float64 from the values that the stage before left."""
    B = Block(dev, 260, 96, 200, 5)
    B.step()
    r, p = B.read(), B.h
    T = lambda v: P.value(np.ascontiguousarray(v.T)).T  # noqa: E731  what the packed transpose holds
    V = P.value
    near = lambda got, want: float(np.linalg.norm(got - want) / np.linalg.norm(want))  # noqa: E731
    xh, rstd = P.layernorm(p["x"], 1e-5)
    f64 = {k: v.astype(np.float64) for k, v in {**p, **r}.items()}
    # each stage is a handful of fp32 roundings and sums of random sign: 1e-6 in the 2-norm
    want = {"y": xh * f64["gamma"] + f64["beta"], "h": V(r["y"]) @ V(p["w1"]).T + f64["b1"], "a": P.gelu(r["h"]),
            "o": f64["x"] + V(r["a"]) @ V(p["w2"]).T + f64["b2"], "da": V(p["g"]) @ T(p["w2"]), "dw2": T(p["g"]).T @ T(r["a"]),
            "db2": f64["g"].sum(0), "dh": f64["da"] * P.gelu_slope(V(r["h"])), "dy": f64["dh"] @ f64["w1"],
            "dw1": f64["dh"].T @ T(r["y"]), "db1": f64["dh"].sum(0)}
    dx, want["dgamma"], want["dbeta"] = P.layernorm_bwd(r["dy"], V(xh), p["gamma"], rstd)
    want["dx"] = f64["g"] + dx
    for k, v in want.items():
        assert near(r[k], v) <= 1e-6, (k, near(r[k], v))


def test_a_block_in_a_graph(dev):
    """Two captured steps that share the context's scratch, replayed in turn with eager work between."""
    blocks = [Block(dev, 260, 96, 200, 7), Block(dev, 1000, 64, 128, 8)]
    want = []
    for b in blocks:
        b.step()
        want.append(b.read())
    L, ctx = dev.ctx.L, dev.ctx
    graphs = []
    for b in blocks:
        assert L.om_graph_capture_begin(ctx.h) == 0
        b.step()
        gr = C.c_void_p()
        assert L.om_graph_capture_end(ctx.h, C.byref(gr)) == 0
        graphs.append(gr)
    try:
        vals = (C.c_float * 3)()
        for turn in range(3):
            for b in blocks:
                for k in Block.NAMES:
                    dev.call("om_fill", b.t[k], float(turn + 3), int(np.prod(b.t[k].shape)))
            for gr in graphs:
                assert L.om_graph_launch(gr, vals) == 0
            ctx.sync()
            for b, w in zip(blocks, want):
                got = b.read()
                for k in Block.NAMES:
                    assert np.array_equal(got[k], w[k]), (turn, k)
            blocks[0].step()
    finally:
        for gr in graphs:
            L.om_graph_destroy(gr)


def test_two_contexts_at_once():
    """Calls on two contexts run side by side, each with its own scratch."""
    a, b = Dev(), Dev()
    A, B = Block(a, 500, 96, 200, 5), Block(b, 500, 96, 200, 6)
    A.step(), B.step()
    wa, wb = A.read(), B.read()
    for _ in range(5):
        A.step(), B.step()
    ra, rb = A.read(), B.read()
    for k in Block.NAMES:
        assert np.array_equal(ra[k], wa[k]) and np.array_equal(rb[k], wb[k])


# -------------------------------------------------------------------------------------------------- past 32-bit offsets
class At:
    """A place inside a device buffer."""

    def __init__(self, buf, offset):
        self.p = buf.data_ptr() + offset

    def data_ptr(self):
        return self.p


def test_rows_far_apart(dev):
    """Leading dimensions whose rows start past 2^32 values: what lies between them is not touched."""
    rng = np.random.default_rng(12)
    rows, cols, ld = 5, 200, 1 << 30
    x = rng.normal(size=(rows, cols)).astype(np.float32)
    X = dev.empty(((rows - 1) * ld + cols + 8,))
    place = [At(X, 4 * r * ld) for r in range(rows)]
    line = dev.empty((cols + 8,))

    def row(r):
        dev.call("om_copy", line, place[r], 4 * (cols + 8))
        return dev.get(line)

    for r in range(rows):
        dev.call("om_fill", place[r], 9.0, cols + 8)
        dev.call("om_copy", place[r], dev.put(x[r]), 4 * cols)
    a, t = packed_buf(dev, rows, cols), packed_buf(dev, cols, rows)
    dev.call("om_pack8", X, ld, rows, cols, a, t)
    check_packed(read_packed(dev, a, rows, cols), x)
    check_packed(read_packed(dev, t, cols, rows), np.ascontiguousarray(x.T))
    dev.call("om_pack8", X, ld, rows, cols, a, None)
    check_packed(read_packed(dev, a, rows, cols), x)
    dev.call("om_unpack8", a, X, ld, rows, cols, 1)
    v = P.value(x)
    for r in range(rows):
        assert np.array_equal(row(r), np.concatenate([x[r] + v[r].astype(np.float32), np.full(8, 9.0, np.float32)]))
    B, bv = put_packed(dev, rng.normal(size=(cols, cols)).astype(np.float32))
    dev.call("om_gemm8", rows, cols, cols, a, B, None, X, ld, 0)
    for r in range(rows):
        got = row(r)
        assert (np.abs(got[:cols] - v[r] @ bv.T) <= sum_bound(cols, np.abs(v[r]) @ np.abs(bv).T)).all() and (got[cols:] == 9.0).all()


def test_tensors_past_32_bits(dev):
    """[66000, 65600]: more than 2^32 values, and codes past 2^32 bytes; the last rows are looked at."""
    rng = np.random.default_rng(13)
    rows, cols, n = 66000, 65600, 2
    X, Q = dev.empty((rows, cols)), dev.empty((P.nbytes(rows, cols),), np.uint8)
    x = rng.normal(size=(n, cols)).astype(np.float32)
    last = At(X, 4 * (rows - n) * cols)
    line = dev.empty((n, cols))

    def fresh():
        dev.call("om_fill", X, 1.0, rows * cols)
        dev.call("om_copy", last, dev.put(x), 4 * n * cols)

    def lines():
        dev.call("om_copy", line, last, 4 * n * cols)
        return dev.get(line)

    def check_last():
        S, T = P.strides(cols)
        raw = dev.empty((n * (S + T),), np.uint8)
        dev.call("om_copy", raw, At(Q, (rows - n) * S), n * S)
        dev.call("om_copy", At(raw, n * S), At(Q, rows * S + (rows - n) * T), n * T)
        return dev.get(raw)

    fresh()
    dev.call("om_pack8", X, cols, rows, cols, Q, None)
    check_packed(check_last(), x)
    dev.call("om_fill", X, 0.0, rows * cols)
    dev.call("om_unpack8", Q, X, cols, rows, cols, 0)
    v = P.value(x)
    assert np.array_equal(lines(), v.astype(np.float32))

    def beside(m, f=lambda u: u):  # m times rows of ones and then f of the last rows' values
        return np.concatenate([np.repeat(m.sum(1)[:, None], rows - n, 1), m @ f(v).T], 1)

    # as the second operand of a product, and as the packed input of a weight gradient
    a = rng.normal(size=(20, cols)).astype(np.float32)
    A, av = put_packed(dev, a)
    Y = dev.empty((20, rows))
    dev.call("om_gemm8", 20, rows, cols, A, Q, None, Y, rows, 0)
    assert (np.abs(dev.get(Y) - beside(av)) <= sum_bound(cols, beside(np.abs(av), np.abs))).all()
    g = rng.normal(size=(cols, 5)).astype(np.float32)
    D = dev.empty((5, rows))
    dev.call("om_linear_bwd_x8", dev.put(g), Q, None, None, D, None, cols, rows, 5, 0, 0, 0)
    gd = g.astype(np.float64).T
    assert (np.abs(dev.get(D) - beside(gd)) <= 3 * sum_bound(cols, beside(np.abs(gd), np.abs))).all()
    # as many rows of a product, far into C
    Z = dev.empty((rows, 70))
    dev.call("om_gemm8", rows, 20, cols, Q, A, None, Z, 70, 0)
    assert (np.abs(dev.get(Z)[:, :20].T - beside(av)) <= sum_bound(cols, beside(np.abs(av), np.abs))).all()
    # GELU, in place, there and back
    fresh()
    Y1, L1 = dev.empty((n, cols)), dev.put(x)
    dev.call("om_gelu_fwd", L1, Y1, n * cols)
    dev.call("om_gelu_fwd_x8", X, X, Q, rows, cols)
    assert np.array_equal(lines(), dev.get(Y1))
    check_packed(check_last(), x)
    fresh()
    dev.call("om_gelu_bwd", L1, dev.put(v.astype(np.float32)), Y1, n * cols, 0)
    dev.call("om_gelu_bwd_x8", X, Q, X, rows, cols, 0)
    assert np.array_equal(lines(), dev.get(Y1))
    # LayerNorm the same way: the last rows' bits are those of these rows alone
    fresh()
    ga, be = (rng.normal(size=cols).astype(np.float32) for _ in range(2))
    GA, BE, R, R1, Q1 = dev.put(ga), dev.put(be), dev.empty((rows,)), dev.empty((n,)), packed_buf(dev, n, cols, 0)
    dev.call("om_layernorm_fwd_x8", L1, GA, BE, Y1, Q1, R1, n, cols, 1e-5)
    dev.call("om_layernorm_fwd_x8", X, GA, BE, X, Q, R, rows, cols, 1e-5)
    assert np.array_equal(lines(), dev.get(Y1)) and np.array_equal(dev.get(R)[-n:], dev.get(R1))
    assert np.array_equal(check_last(), dev.get(Q1))
    fresh()
    dev.call("om_layernorm_bwd_x8", L1, Q1, GA, R1, Y1, None, None, n, cols, 0, 0)
    dev.call("om_layernorm_bwd_x8", X, Q, GA, R, X, None, None, rows, cols, 0, 0)
    assert np.array_equal(lines(), dev.get(Y1))
