"""Rotary positions (om_rope_fwd / om_rope_bwd) against the float64 definition.

Tolerance: cosine and sine are within 1.2e-7 (the reduced angle in fp32, 2^-24 of at most pi/4, the sums' roundings, and
the turns' double rounding, at most 2^-23 of a turn at 2^31 turns' scale, far below that at the positions here), times
the amplitude rounded once more; each output is two products and a sum of values up to |x|: 4 roundings of 2^-24, so an
error of at most 2 (1.2e-7 + 2 * 6e-8) + 6e-8 < 6e-7 of amp times the pair's larger value."""
import ctypes as C

import numpy as np
import pytest

import scored_ref as R
from gpu_util import Dev, load_pkg

pytestmark = pytest.mark.gpu
TOL = 6e-7


@pytest.fixture(scope="module")
def dev():
    return Dev()


def make(layout="half", scaling="plain", rot=32, amp=1.0, base=10000.0, factor=8.0, trained=4096.0, low=1.0, high=32.0):
    r = load_pkg().om_rope()
    r.layout = ("half", "interleaved").index(layout)
    r.scaling = ("plain", "linear", "ntk", "bands").index(scaling)
    r.rot, r.amplitude, r.base, r.factor, r.trained, r.low, r.high = rot, amp, base, factor, trained, low, high
    return r, R.rope_speeds(rot, scaling, base, factor, trained, low, high)


def check(got, want, x, amp):
    bound = TOL * max(1.0, abs(amp)) * float(np.abs(x).max())
    assert got.shape == want.shape and np.isfinite(got).all()
    assert float(np.abs(got - want).max()) <= bound, (float(np.abs(got - want).max()), bound)


CASES = [
    # rows, seq, heads, d, rot, layout, scaling, pad of the strides, far
    (1, 1, 1, 2, 2, "half", "plain", 0, 0),
    (8, 1, 16, 64, 64, "half", "linear", 0, 100000),
    (37, 37, 3, 32, 32, "interleaved", "plain", 4, 0),
    (50, 25, 2, 40, 40, "half", "ntk", 8, 5000),        # 16-byte slots
    (50, 25, 2, 40, 20, "half", "bands", 0, 5000),      # half of 20 pairs is no multiple of four: single pairs
    (50, 25, 2, 40, 20, "interleaved", "bands", 0, 5000),
    (33, 11, 5, 7, 6, "interleaved", "plain", 1, 300),  # odd width and stride
    (129, 43, 3, 256, 64, "half", "plain", 0, 2000000000),
    (64, 64, 2, 128, 128, "interleaved", "bands", 12, 1000000),
    (5, 5, 1, 256, 256, "half", "ntk", 0, 0),
]


@pytest.mark.parametrize("c", CASES, ids=[f"{c[3]}-{c[4]}-{c[5]}-{c[6]}" for c in CASES])
def test_forward_and_backward(dev, c):
    rows, seq, heads, d, rot, layout, scaling, pad, far = c
    rng = np.random.default_rng(rows * 7 + d)
    amp = 1.2 if scaling == "bands" else 1.0
    rp, f = make(layout, scaling, rot, amp)
    ld, ldy = heads * d + pad, heads * d + 2 * pad
    x = rng.normal(size=(rows, ld)).astype(np.float32)
    pos = rng.integers(-5 if far else 0, far + 50, rows).astype(np.int32)
    xh = x[:, :heads * d].reshape(rows, heads, d)
    X, P = dev.put(x), dev.put(pos)
    for name, back, acc in (("om_rope_fwd", False, 0), ("om_rope_bwd", True, 0), ("om_rope_bwd", True, 1)):
        y0 = rng.normal(size=(rows, ldy)).astype(np.float32)
        Y = dev.put(y0)
        dev.call(name, X, ld, P, 0, Y, ldy, rows, seq, heads, d, C.byref(rp), *([acc] if back else []))
        got = dev.get(Y)
        want = R.rope(xh, pos, rot, layout, f, float(np.float32(amp)), back).reshape(rows, -1)
        if acc:
            want = want + y0[:, :heads * d]
        check(got[:, :heads * d], want, np.abs(x).max() + (np.abs(y0).max() if acc else 0), amp)
        assert np.array_equal(got[:, heads * d:], y0[:, heads * d:])  # columns beside the heads stay
        if rot < d and not acc:
            assert np.array_equal(got[:, :heads * d].reshape(rows, heads, d)[..., rot:], xh[..., rot:])


def test_positions_from_the_row_number(dev):
    rng = np.random.default_rng(3)
    rp, f = make(rot=8)
    x = rng.normal(size=(12, 2, 8)).astype(np.float32)
    Y = dev.empty((12, 16))
    dev.call("om_rope_fwd", dev.put(x), 16, None, 70, Y, 16, 12, 5, 2, 8, C.byref(rp))
    want = R.rope(x, 70 + np.arange(12) % 5, 8, "half", f)
    check(dev.get(Y).reshape(x.shape), want, x, 1.0)


def test_in_place_on_the_q_and_k_columns_of_a_packed_projection(dev):
    rng = np.random.default_rng(4)
    rows, H, Hk, d = 30, 4, 2, 16
    w = (H + 2 * Hk) * d
    x = rng.normal(size=(rows, w)).astype(np.float32)
    rp, f = make("interleaved", rot=16)
    X = dev.put(x)
    dev.call("om_rope_fwd", X, w, None, 0, X, w, rows, rows, H + Hk, d, C.byref(rp))
    got = dev.get(X)
    want = R.rope(x[:, :(H + Hk) * d].reshape(rows, H + Hk, d), np.arange(rows), 16, "interleaved", f)
    check(got[:, :(H + Hk) * d], want.reshape(rows, -1), x, 1.0)
    assert np.array_equal(got[:, (H + Hk) * d:], x[:, (H + Hk) * d:])
    # turned back, the rows are what they were
    dev.call("om_rope_bwd", X, w, None, 0, X, w, rows, rows, H + Hk, d, C.byref(rp), 0)
    assert float(np.abs(dev.get(X) - x).max()) <= 2 * TOL * float(np.abs(x).max())


def test_nan_and_infinity_stay_in_their_pair(dev):
    rp, f = make(rot=4)
    x = np.ones((2, 1, 6), np.float32)
    x[0, 0, 1], x[1, 0, 5] = np.nan, np.inf
    Y = dev.empty((2, 6))
    dev.call("om_rope_fwd", dev.put(x), 6, None, 1, Y, 6, 2, 2, 1, 6, C.byref(rp))
    got = dev.get(Y)
    assert np.isnan(got[0, [1, 3]]).all() and np.isfinite(got[0, [0, 2, 4, 5]]).all()
    assert np.isinf(got[1, 5]) and np.isfinite(got[1, :5]).all()


def test_empty_calls_do_nothing(dev):
    rp, _ = make(rot=4)
    Y = dev.empty((2, 4), fill=7.0)
    dev.call("om_rope_fwd", None, 4, None, 0, Y, 4, 0, 1, 1, 4, C.byref(rp))
    dev.call("om_rope_bwd", None, 4, None, 0, Y, 4, 2, 1, 0, 4, C.byref(rp), 1)
    assert (dev.get(Y) == 7.0).all()


def test_more_work_than_one_grid(dev):
    """Past 64 workgroups per CU a thread takes several slots."""
    rng = np.random.default_rng(9)
    rows, heads, d = 40000, 16, 32
    rp, f = make(rot=32)
    x = rng.normal(size=(rows, heads, d)).astype(np.float32)
    Y = dev.empty((rows, heads * d))
    dev.call("om_rope_fwd", dev.put(x), heads * d, None, 0, Y, heads * d, rows, 1000, heads, d, C.byref(rp))
    check(dev.get(Y).reshape(x.shape), R.rope(x, np.arange(rows) % 1000, 32, "half", f), x, 1.0)
