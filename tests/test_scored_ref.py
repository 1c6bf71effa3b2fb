"""The plain definitions the GPU tests compare with, checked on the CPU: gradients against central differences, and the
rules' corners by hand."""
import numpy as np
import pytest

import scored_ref as R

RULES = [
    dict(),
    dict(causal=1, cap=2.0),
    dict(window=3, slopes=[0.5, 0.125]),
    dict(causal=1, window=2, prefix=[2, 0]),
    dict(qdoc=[[0, 0, 1, -1], [3, 5, 5, 5]], kdoc=[[0, 1, 1, -1, 0], [5, 3, -1, 5, 2]], cap=1.5),
]


@pytest.mark.parametrize("rule", RULES, ids=range(len(RULES)))
def test_gradients_against_differences(rule):
    r = np.random.default_rng(5)
    B, lq, lk, H, Hk, d = 2, 4, 5, 2, 1, 3
    x = [r.normal(size=s) for s in ((B, lq, H, d), (B, lk, Hk, d), (B, lk, Hk, d))]
    g = r.normal(size=(B, lq, H, d))
    grads = R.attention(*x, g=g, **rule)[1:]
    eps = 1e-5
    for n in range(3):
        for _ in range(12):
            at = tuple(r.integers(0, s) for s in x[n].shape)
            up, dn = [a.copy() for a in x], [a.copy() for a in x]
            up[n][at] += eps
            dn[n][at] -= eps
            diff = ((R.attention(*up, **rule) - R.attention(*dn, **rule)) * g).sum() / (2 * eps)
            # central differences in float64: eps^2 third derivatives and 2^-52 / eps of rounding
            assert abs(diff - grads[n][at]) <= 1e-8, (n, at, diff, grads[n][at])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rope_backward_against_differences_and_length(layout):
    r = np.random.default_rng(6)
    x, g, pos = r.normal(size=(3, 2, 6)), r.normal(size=(3, 2, 6)), np.array([0, 7, -3])
    f = R.rope_speeds(4, "linear", factor=2.0)
    y = R.rope(x, pos, 4, layout, f)
    assert np.allclose((y ** 2).sum(-1), (x ** 2).sum(-1)) and np.array_equal(y[..., 4:], x[..., 4:])
    dx = R.rope(g, pos, 4, layout, f, amp=1.5, back=True)
    for at in np.ndindex(x.shape):
        e = np.zeros_like(x)
        e[at] = 1.0
        assert abs((R.rope(e, pos, 4, layout, f, amp=1.5) * g).sum() - dx[at]) < 1e-12


def test_rope_scaling_corners():
    f = R.rope_speeds(8)
    assert np.allclose(R.rope_speeds(8, "linear", factor=4.0), f / 4)
    ntk = R.rope_speeds(8, "ntk", factor=4.0)
    assert ntk[0] == f[0] and np.isclose(ntk[-1], f[-1] / 4)
    bands = R.rope_speeds(8, "bands", factor=4.0, trained=64.0, low=0.5, high=8.0)
    turns = f * 64.0 / (2 * np.pi)
    assert np.allclose(bands[turns >= 8.0], f[turns >= 8.0]) and np.allclose(bands[turns <= 0.5], f[turns <= 0.5] / 4)


def test_rules_by_hand():
    assert R.visible(2, 3, causal=1).tolist() == [[True, True, False], [True, True, True]]
    assert not R.visible(3, 1, causal=1)[:2].any()  # queries before the first key see nothing
    assert R.visible(3, 3, causal=1, window=1, prefix=[2]).tolist() == [[True, True, False], [True, True, False], [True, True, True]]
    see = R.visible(2, 2, qdoc=[[0, -1]], kdoc=[[0, -1]])
    assert see.tolist() == [[True, False], [False, False]]
