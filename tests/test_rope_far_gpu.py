"""Rotary angles at positions up to 2^31 - 1 against a 60-digit reference, where a float64 one is off by as much as the bound.

Tolerance: 4e-7, the bound that include/om.h states. A pair (1, 0) turns into the cosine and sine themselves, each within 1.2e-7
of its angle's (1.7e-7 together); what is left is the angle's."""
import ctypes as C
from decimal import Decimal as D
from decimal import getcontext

import numpy as np
import pytest

from gpu_util import Dev
from test_rope_gpu import make

pytestmark = pytest.mark.gpu
getcontext().prec = 60
TWO_PI = 2 * D("3.14159265358979323846264338327950288419716939937510582097494")


@pytest.fixture(scope="module")
def dev():
    return Dev()


def speeds(rot, scaling, base, factor, trained, low, high):
    base, factor = D(base), D(factor)
    if scaling == "ntk":
        base *= (factor.ln() * rot / (rot - 2)).exp()
    out = []
    for i in range(rot // 2):
        f = (-base.ln() * 2 * i / rot).exp()
        if scaling == "linear":
            f /= factor
        if scaling == "bands":
            keep = min(D(1), max(D(0), (f * D(trained) / TWO_PI - D(low)) / (D(high) - D(low))))
            f *= keep + (1 - keep) / factor
        out.append(f)
    return out


@pytest.mark.parametrize("scaling", ["plain", "linear", "ntk", "bands"])
@pytest.mark.parametrize("rot,base", [(256, 1e6), (64, 1e4), (32, 500.0)])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_angles_of_far_positions(dev, layout, rot, base, scaling):
    r = np.random.default_rng(rot)
    pos = np.concatenate([[2147398138, 2 ** 31 - 1, -2 ** 31, 2 ** 31 - 100, 0, 1, -1], 2 ** 31 - r.integers(1, 2 ** 20, 60),
                          r.integers(-2 ** 31, 2 ** 31, 30)]).astype(np.int64)
    kw = dict(factor=7.3, trained=4097.0, low=1.0, high=31.0)
    rp, _ = make(layout, scaling, rot, 1.0, base, **kw)
    i = np.arange(rot // 2)
    a, b = (i, i + rot // 2) if layout == "half" else (2 * i, 2 * i + 1)
    x = np.zeros((len(pos), rot), np.float32)
    x[:, a] = 1.0
    Y = dev.empty(x.shape)
    dev.call("om_rope_fwd", dev.put(x), rot, dev.put(pos.astype(np.int32)), 0, Y, rot, len(pos), 1, 1, rot, C.byref(rp))
    y = dev.get(Y).astype(np.float64)
    f = speeds(rot, scaling, base, **kw)
    ang = np.array([[float((int(p) * s) % TWO_PI) for s in f] for p in pos])
    off = np.hypot(y[:, a] - np.cos(ang), y[:, b] - np.sin(ang))
    assert off.max() <= 4e-7, (off.max(), pos[off.max(1).argmax()], off.max(0).argmax())
