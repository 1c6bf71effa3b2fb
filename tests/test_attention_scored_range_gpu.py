"""Scored attention where values or scores leave the ordinary range, against the float64 definition.

Tolerances: as in test_attention_scored_gpu.py (1e-5 of the largest value) where nothing else is said."""
import numpy as np
import pytest

from gpu_util import Dev
from test_attention_scored_gpu import TOL, Case, near

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return Dev()


def winners(c, size):
    """Each query points at one key that it sees: that key's score is about size * sqrt(d), the others' a few times less."""
    B, H, Hk, lq, lk, d = c.dims
    for t in range(lq):
        c.q[:, t] = np.float32(size) * np.repeat(c.k[:, (t + lk - lq) // 2], H // Hk, 1)


@pytest.mark.parametrize("s", [(1, 4, 2, 200, 200, 64), (2, 2, 1, 60, 300, 96), (1, 2, 2, 150, 150, 128), (1, 4, 1, 90, 90, 20),
                               (4, 4, 4, 100, 120, 32), (2, 2, 1, 160, 300, 96), (1, 4, 2, 260, 260, 128)], ids=str)
@pytest.mark.parametrize("size", [10.0, 1e3, 1e5, 1e8])
def test_scores_of_any_size_with_clear_winners(dev, s, size):
    """Weights are one for the winner. A recomputed score of the matrix products is within 2^-22 of itself, and so is the
    weight that the backward takes from it: their scores are kept below 2^10, beyond it sums round equally both ways. dq and dk
    are nothing but what rounding leaves of g . v - g . o: 2^-20 of the sum of magnitudes, times the row or key it goes with."""
    c = Case(dev, *s, causal=1, seed=41)
    winners(c, size)
    want = c.reference()
    near(c.forward(), want[0], what="o")
    dq, dk, dv = c.backward()
    near(dv, want[3], TOL + min(2.0 ** 10, 2 * size * s[5] ** 0.5) * 2.0 ** -22, what="dv")
    left = 2.0 ** -20 * np.abs(c.g).sum(3).max() * np.abs(c.v).max() * s[5] ** -0.5
    near(dq, want[1], what="dq", floor=left * np.abs(c.k).max())
    near(dk, want[2], what="dk", floor=left * np.abs(c.q).max() * s[3])


@pytest.mark.parametrize("cap", [0.0, 20.0])
def test_queries_of_very_different_size_in_one_block(dev, cap):
    """Every other query 2^32 times as large with a gradient as much smaller: the small ones' scores keep their bits."""
    c = Case(dev, 1, 4, 2, 190, 190, 64, causal=1, seed=42, cap=cap)
    c.q[:, ::2] *= np.float32(2.0 ** 32)
    c.g[:, ::2] *= np.float32(2.0 ** -32)
    want = c.reference()
    o, (dq, dk, dv) = c.forward(), c.backward()
    near(o[:, 1::2], want[0][:, 1::2], what="o")
    near(dq[:, 1::2], want[1][:, 1::2], what="dq")
    near(dv, want[3], what="dv")
    near(dk, want[2], what="dk", floor=c.floor()[1] * 2.0 ** -32)  # the large queries' part: their gradients are as small


@pytest.mark.parametrize("kw", [dict(scale=1e-43), dict(scale=-1e-20), dict(scale=1e-30, cap=1e-9), dict(cap=1e36), dict(cap=1e25, scale=1e-5),
                                dict(scale=1e20)], ids=str)
def test_scale_and_cap_far_from_one(dev, kw):
    c = Case(dev, 1, 4, 2, 150, 150, 64, causal=1, seed=43, **kw)
    if kw.get("scale") == 1e20:
        winners(c, 1.0)
    want = c.reference()
    near(c.forward(), want[0], what="o")
    dq, dk, dv = c.backward()
    near(dv, want[3], what="dv")
    if kw.get("scale") != 1e20:  # dq and dk are zero there: see test_scores_of_any_size_with_clear_winners
        near(dq, want[1], what="dq", floor=c.floor()[0])
        near(dk, want[2], what="dk", floor=c.floor()[1])


@pytest.mark.parametrize("s", [(1, 4, 2, 200, 200, 64), (1, 4, 4, 260, 300, 32), (1, 8, 2, 130, 140, 96), (1, 4, 2, 260, 260, 128)], ids=str)
def test_gradient_rows_of_very_different_size(dev, s):
    """A row's dq scales with its gradient, bit for bit by powers of two: no neighbour's size sends it to other sums."""
    a, b = (Case(dev, *s, causal=1, cap=12.0, seed=44) for _ in range(2))
    by = np.where(np.arange(s[3]) % 5 == 2, 20, 0)
    b.g = np.ldexp(b.g, by[None, :, None, None]).astype(np.float32)
    a.forward(), b.forward()
    plain, spread, want = a.backward()[0], b.backward(), b.reference()[1:]
    assert np.array_equal(spread[0], np.ldexp(plain, by[None, :, None, None]))
    for got, ref, n in zip(spread, want, ("dq", "dk", "dv")):
        near(got, ref, what=n, floor=b.floor()[0] if n == "dq" else 0.0)


COLUMN_SHAPES = [(1, 4, 2, 200, 200, 64), (1, 4, 4, 260, 300, 32), (1, 8, 2, 130, 140, 96), (1, 4, 2, 260, 260, 128), (1, 4, 2, 193, 193, 40)]


@pytest.mark.parametrize("s", COLUMN_SHAPES, ids=str)
@pytest.mark.parametrize("power", [-20, -28, -36])
@pytest.mark.parametrize("which", ["q", "k", "v", "g"])
def test_columns_of_very_different_size(dev, which, power, s):
    """A column of one operand 2^power times as large: the column that it makes of an output keeps its own precision."""
    c = Case(dev, *s, causal=1, seed=45)
    getattr(c, which)[..., 7] *= np.float32(2.0 ** power)
    want = c.reference()
    got = [c.forward()] + c.backward()
    out = {"v": 0, "k": 1, "q": 2, "g": 3}[which]
    floors = [0.0, c.floor()[0], 0.0, 0.0]
    near(got[out][..., 7], want[out][..., 7], what=which, floor=floors[out] * 2.0 ** power)
    for g, w, n, f in zip(got, want, ("o", "dq", "dk", "dv"), floors):
        near(g, w, what=n, floor=f)


@pytest.mark.parametrize("s", COLUMN_SHAPES, ids=str)
def test_a_small_column_of_v_beside_a_large_one_of_g(dev, s):
    """Values and gradients whose columns' sizes cancel: g . v keeps its bits."""
    c = Case(dev, *s, causal=1, seed=46)
    want = c.reference()
    c.v[..., 7] *= np.float32(2.0 ** -28)
    c.g[..., 7] *= np.float32(2.0 ** 28)
    near(c.forward()[..., :7], want[0][..., :7], what="o")
    dq, dk, dv = c.backward()
    near(dq, want[1], what="dq", floor=2.0 ** -22 * 64 * 8 * s[5] ** -0.5)  # sums of up to d products below 8, four roundings
    near(dk, want[2], what="dk")
    near(dv[..., :7], want[3][..., :7], what="dv")


def test_columns_of_one_live_row(dev):
    """A last block of one key or query: its columns are single values, and stay on the matrix cores down to 2^-22 of the largest."""
    c = Case(dev, 1, 4, 2, 193, 193, 64, causal=1, seed=47)
    for x in (c.q, c.k, c.v, c.g):
        x[:, 192, :, 3] *= np.float32(2.0 ** -19)
        x[:, 192, :, 9] = 0.0
    want = c.reference()
    for g, w, n, f in zip([c.forward()] + c.backward(), want, ("o", "dq", "dk", "dv"), (0.0, *c.floor(), 0.0)):
        near(g, w, what=n, floor=f)
    near(c.backward()[2][:, 192], want[3][:, 192], what="dv of the last key")


@pytest.mark.parametrize("s", [(1, 4, 2, 200, 200, 64), (1, 4, 4, 200, 200, 32), (2, 4, 2, 200, 200, 96), (2, 4, 1, 200, 200, 128)], ids=str)
@pytest.mark.parametrize("slopes", [(0.5, 3.0, 50.0, 800.0), (2e4, 1e6, 3e9, -40.0)], ids=str)
def test_distance_bias_where_only_far_keys_are_seen(dev, s, slopes):
    """Half of the queries see only the keys of the other half: their scores are all bias, the nearest key (the furthest, where a
    slope is negative) has the weight. Rounded the same way in both directions, it is one."""
    ids = np.repeat([[1, 0]], s[3] // 2, 1).repeat(s[0], 0)
    c = Case(dev, *s, seed=48, slopes=True, qdoc=ids, kdoc=1 - ids)
    c.sl[:] = slopes
    buf = dev.put(c.sl)
    c.keep.append(buf)
    c.form.slopes = buf.data_ptr()
    want = c.reference()
    near(c.forward(), want[0], what="o")
    dq, dk, dv = c.backward()
    near(dv, want[3], what="dv")
    near(dq, want[1], what="dq", floor=c.floor()[0])
    near(dk, want[2], what="dk", floor=c.floor()[1])


@pytest.mark.parametrize("s", [(1, 4, 2, 200, 200, 64), (1, 4, 4, 260, 260, 32), (1, 8, 2, 140, 140, 96), (1, 4, 2, 300, 300, 128)], ids=str)
@pytest.mark.parametrize("by", [16, 40, -40])
def test_gradients_of_one_document_leave_the_others_bits(dev, s, by):
    """Rows of one document with gradients 2^by times as large: dk and dv of its keys scale by it, the other document's keep their
    bits, though rows of both share blocks."""
    ids = (np.arange(s[3])[None] >= 100).astype(np.int32)
    a, b = (Case(dev, *s, causal=1, cap=12.0, seed=49, qdoc=ids, kdoc=ids) for _ in range(2))
    b.g[:, :100] = np.ldexp(b.g[:, :100], by)
    a.forward(), b.forward()
    for x, y in zip(a.backward(), b.backward()):
        assert np.array_equal(y[:, 100:], x[:, 100:])
        assert np.array_equal(y[:, :100], np.ldexp(x[:, :100], by))


@pytest.mark.parametrize("s", [(1, 4, 2, 400, 400, 64), (1, 4, 4, 260, 300, 32), (1, 8, 2, 333, 333, 96), (1, 4, 2, 300, 300, 128)], ids=str)
@pytest.mark.parametrize("width", [1.0, 3.0, 8.0])
def test_peaked_and_flat_rows_with_gradients_of_many_sizes(dev, s, width):
    """One row in ten peaked (its sum near one), the others flat, gradients log-normal over the rows."""
    c = Case(dev, *s, causal=1, seed=50)
    r = np.random.default_rng(50)
    c.q *= np.where(r.random((s[0], s[3], 1, 1)) < 0.1, 6.0, 0.2).astype(np.float32)
    c.g *= np.exp(width * r.normal(size=(s[0], s[3], 1, 1))).astype(np.float32)
    want = c.reference()
    near(c.forward(), want[0], what="o")
    for g, w, n, f in zip(c.backward(), want[1:], ("dq", "dk", "dv"), (2 * c.floor()[0], 0.0, 0.0)):
        near(g, w, what=n, floor=f)


@pytest.mark.parametrize("which", ["q", "k", "v", "g"])
def test_one_small_value_in_a_single_row_changes_no_other_rows_sums(dev, which):
    """A last block of one row: a value 2^-19 of its largest leaves the rows and keys that share workgroups with it on the matrix
    cores, so with their bits (q and g of the last row aside, what it gives to the keys is taken out)."""
    a, b = (Case(dev, 1, 2, 2, 193, 193, 64, causal=1, seed=53) for _ in range(2))
    for c in (a, b):
        c.g[:, 192] *= np.float32(2.0 ** -60)
    getattr(b, which)[:, 192, :, 3] = getattr(b, which)[:, 192].max(-1) * np.float32(2.0 ** -19)
    x, y = [a.forward()] + a.backward(), [b.forward()] + b.backward()
    for n, (p, q) in enumerate(zip(x, y)):
        assert np.array_equal(p[:, :192], q[:, :192]) or n >= 2 and which in "qg", n
