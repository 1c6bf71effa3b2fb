"""Scored attention's gradients held closely: dq and dk at the sizes that reach the matrix kernels' pieces.

Tolerance: 1e-5 of the largest value, as for the outputs, and beside it only what the cancellation in ds = p (g . v - delta)
leaves of a row or key, formed from the float64 weights: g . v and delta are each within 2^-22 of their sums of magnitudes (22-bit
operands, fp32 sums), so dq_i is off by at most 2^-22 scale sum_j p_ij t_ij (sum_c |g_ic v_jc| + sum_c |g_ic o_ic|) |k_j| more,
t the cap's slope, and dk_j by the same sum over its rows with |q_i|. Where one key is seen that is all there is."""
import numpy as np
import pytest

import scored_ref as R
from gpu_util import Dev
from test_attention_scored_gpu import TOL, Case, docs

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return Dev()


def floors(c, o):
    """What rounding of g . v - delta may leave of each value of dq and dk (o: float64)."""
    B, H, Hk, lq, lk, d = c.dims
    rule = {n: v for n, v in c.rule.items() if n in ("causal", "window", "prefix", "qdoc", "kdoc")}
    scale = c.form.scale if c.form.scale else d ** -0.5
    fq, fk = np.zeros(c.q.shape), np.zeros(c.k.shape)
    dist = np.abs(np.arange(lq)[:, None] + (lk - lq) - np.arange(lk)[None, :])
    for b in range(B):
        see = R.visible(lq, lk, b=b, **rule)
        for h in range(H):
            hk = h // (H // Hk)
            q, g, k, v = (np.asarray(a, np.float64) for a in (c.q[b, :, h], c.g[b, :, h], c.k[b, :, hk], c.v[b, :, hk]))
            x, t = (q @ k.T) * scale, 0.0
            if c.form.cap:
                t = np.tanh(x / c.form.cap)
                x = t * c.form.cap
            if c.sl is not None:
                x = x - np.float64(c.sl[h]) * dist
            x = np.where(see, x, -np.inf)
            m = x.max(1, keepdims=True)
            e = np.where(see, np.exp(x - np.where(m == -np.inf, 0.0, m)), 0.0)
            p = e / np.maximum(e.sum(1, keepdims=True), 1e-300)
            a = np.abs(g) @ np.abs(v).T + np.abs(g * o[b, :, h]).sum(1, keepdims=True)
            w = 2.0 ** -22 * abs(scale) * p * (1.0 - t * t) * a
            fq[b, :, h] = w @ np.abs(k)
            fk[b, :, hk] += w.T @ np.abs(q)
    return fq, fk


def close(c):
    want = c.reference()
    o = c.forward()
    assert np.abs(o - want[0]).max() <= TOL * np.abs(want[0]).max(), "o"
    got = c.backward()
    for g, w, f, n in zip(got, want[1:], (*floors(c, want[0]), 0.0), ("dq", "dk", "dv")):
        over = np.abs(g - w) - (TOL * np.abs(w).max() + f)
        print(n, "error %.2g of the largest, floor up to %.2g" % (np.abs(g - w).max() / np.abs(w).max(), np.max(f) / np.abs(w).max()),
              flush=True)
        assert np.isfinite(g).all() and over.max() <= 0, (n, over.max(), np.abs(w).max())


CASES = {
    "causal-700": ((1, 2, 1, 700, 700, 64), dict(causal=1, cap=20.0)),
    "chunk-96": ((1, 4, 1, 515, 1300, 96), dict(causal=1, cap=20.0)),
    "narrow": ((2, 2, 2, 600, 600, 32), dict(causal=1)),
    "five-over-5000": ((1, 1, 1, 5, 5000, 128), dict(causal=1, cap=20.0)),
    "window-slopes": ((1, 2, 2, 1025, 1025, 64), dict(window=130, slopes=True)),
    "prefix-80": ((1, 3, 1, 777, 777, 80), dict(causal=1, prefix=[333])),
    "pieces-80": ((1, 4, 2, 30, 3000, 80), dict(causal=1, cap=7.0)),
    "pieces-window": ((1, 1, 1, 40, 2500, 128), dict(window=900, slopes=True)),
    "shared-128": ((1, 8, 2, 300, 700, 128), dict(causal=1, cap=9.0)),
    "one-key-each": ((1, 4, 2, 300, 300, 64), dict(window=1)),
    "two-keys-each": ((1, 4, 2, 300, 300, 96), dict(causal=1, window=2)),
    "wide-heads": ((1, 2, 1, 90, 120, 200), dict(causal=1, cap=9.0)),
}


@pytest.mark.parametrize("name", CASES)
def test_gradients_closely(dev, name):
    s, kw = CASES[name]
    close(Case(dev, *s, seed=51, **kw))


@pytest.mark.parametrize("d", [32, 64, 96, 128])
def test_gradients_closely_in_documents(dev, d):
    close(Case(dev, 2, 4, 2, 330, 330, d, seed=52, causal=1, slopes=True, qdoc=docs(2, 330, 3, 4), kdoc=docs(2, 330, 3, 4)))
