"""Calls of more workgroups than a launch takes are refused before anything runs (their pointers are never read)."""
import ctypes as C

import pytest

from gpu_util import Dev

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return Dev()


@pytest.mark.parametrize("B,lq,d", [(1 << 24, 1, 1), (1 << 24, 8, 1), (1 << 24, 1, 200), (1 << 25, 9, 96), (1 << 23, 2, 256)], ids=str)
def test_too_many_workgroups(dev, B, lq, d):
    x = dev.empty((1024,), fill=1.0)
    f = dev.pkg.om_attention_scores()
    f.heads = f.kv_heads = 1
    assert dev.status("om_attention_fwd_scored", x, d, x, x, d, x, d, None, B, lq, 1, d, C.byref(f)) == 1
    assert b"too many row blocks" in dev.ctx.L.om_last_error(dev.ctx.h)
    assert dev.status("om_attention_bwd_scored", x, d, x, x, d, x, d, x, x, d, x, d, x, x, d, B, lq, 1, d, C.byref(f), 0) == 1
    assert b"too many row blocks" in dev.ctx.L.om_last_error(dev.ctx.h)
    assert (dev.get(x) == 1.0).all()
