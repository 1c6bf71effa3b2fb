"""Column sums: whichever kernels a size is given to, a column's sum has the same additions in the same order. Columns of one wide
matrix, summed beside all the others and among few, have to come out with the same bits."""
import numpy as np
import pytest

from gpu_util import Dev

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return Dev()


# up to 1024 rows in one launch; past them in two: partials by one column a lane and by four, chunks by 16 columns to a workgroup
# and by a wavefront a column
@pytest.mark.parametrize("rows", [1, 65, 1000, 1025, 5000, 20001, 70000])
def test_the_same_bits_among_few_columns_and_many(dev, rows):
    rng = np.random.default_rng(rows)
    cols = 300 if rows < 70000 else 64
    # sums that depend on the order of their additions even in double: 2^-40 .. 2^40 of either sign
    g = (rng.normal(size=(rows, cols)) * np.exp2(rng.integers(-40, 40, (rows, cols)).astype(np.float64))).astype(np.float32)
    want, size = g.astype(np.float64).sum(0), np.abs(g.astype(np.float64)).sum(0)
    old = rng.normal(size=cols).astype(np.float32)

    def total(n, acc):
        B = dev.put(old[:n])
        dev.call("om_colsum", dev.put(np.ascontiguousarray(g[:, :n])), B, rows, n, acc)
        return dev.get(B)

    for acc in (0, 1):
        full = total(cols, acc)
        # rows additions in double of up to the magnitudes' sum, one rounding to float, one more addition where the old is kept
        ref = want + acc * old.astype(np.float64)
        assert (np.abs(full - ref) <= 2.0 ** -24 * (np.abs(ref) + acc * np.abs(want)) * 1.01 + rows * 2.0 ** -53 * size).all()
        for n in (1, 2, 15, 16, 17, 20, 21, 33, 256):
            if n <= cols:
                assert np.array_equal(total(n, acc), full[:n]), (n, acc)


@pytest.mark.parametrize("rows,cols", [(3000, 1), (3000, 12), (40000, 8), (3000, 18), (3000, 40)])
def test_layernorm_parameter_gradients_of_few_columns(dev, rows, cols):
    """Both sums of one last stage, alone and together."""
    rng = np.random.default_rng(cols)
    x, g = (rng.normal(size=(rows, cols)).astype(np.float32) for _ in range(2))
    ga, be = np.ones(cols, np.float32), np.zeros(cols, np.float32)
    X, G, GA, M, R = dev.put(x), dev.put(g), dev.put(ga), dev.empty((rows,)), dev.empty((rows,))
    dev.call("om_layernorm_fwd", X, GA, dev.put(be), dev.empty(x.shape), M, R, rows, cols, 1e-5)
    A, B, A1, B1 = (dev.empty((cols,)) for _ in range(4))
    dev.call("om_layernorm_bwd", G, X, GA, M, R, None, A, B, rows, cols, 0, 0)
    dev.call("om_layernorm_bwd", G, X, GA, M, R, None, A1, None, rows, cols, 0, 0)
    dev.call("om_layernorm_bwd", G, X, GA, M, R, None, None, B1, rows, cols, 0, 0)
    assert np.array_equal(dev.get(A), dev.get(A1)) and np.array_equal(dev.get(B), dev.get(B1))
    xh = (x - dev.get(M)[:, None]).astype(np.float64) * dev.get(R)[:, None]
    g64 = g.astype(np.float64)
    # xh within two roundings of its own; sums in double
    assert (np.abs(dev.get(A) - (g64 * xh).sum(0)) <= 2.0 ** -24 * (np.abs((g64 * xh).sum(0)) + 4 * np.abs(g64 * xh).sum(0))).all()
    assert (np.abs(dev.get(B) - g64.sum(0)) <= 2.0 ** -24 * 1.01 * np.abs(g64.sum(0)) + 1e-13 * np.abs(g64).sum(0)).all()
