"""Context scratch that outgrows its buffer while step graphs are about: the graphs keep the buffer that their launches name,
and it is given back with the last of them."""
import ctypes as C

import numpy as np
import pytest

from gpu_util import Dev, hip
from test_attention_scored_gpu import Case, _graph, _Values

pytestmark = pytest.mark.gpu
MIB = 1 << 20


@pytest.fixture()
def dev():
    return Dev()


def free():
    a, b = C.c_size_t(), C.c_size_t()
    hip().hipDeviceSynchronize()
    assert hip().hipMemGetInfo(C.byref(a), C.byref(b)) == 0
    return a.value


class Forward:
    """A forward whose scratch for the matrix cores is about 128 bytes a key: 64 keys a head in, `mib` of scratch out."""

    def __init__(self, dev, mib):
        self.dev, self.L = dev, mib * MIB // (8 * 4 * 64 * 2)
        f = self.form = dev.pkg.om_attention_scores()
        f.heads = f.kv_heads = 8
        self.q, self.o = dev.empty((16, 8 * 64), fill=0.5), dev.empty((16, 8 * 64))
        self.k, self.v = (dev.empty((self.L, 8 * 64), fill=0.25) for _ in range(2))

    def __call__(self):
        self.dev.call("om_attention_fwd_scored", self.q, 512, self.k, self.v, 512, self.o, 512, None, 1, 16, self.L, 64,
                      C.byref(self.form))


def test_outgrown_scratch_goes_with_the_last_graph(dev):
    small, large, larger = (Forward(dev, m) for m in (20, 150, 300))
    small()
    dev.ctx.sync()
    calls = [small, large]
    # a capture that is given up keeps nothing
    dev.ctx.call("om_graph_capture_begin")
    small()
    dev.ctx.call("om_graph_capture_abort")
    before = free()
    large()
    dev.ctx.sync()
    taken = before - free()  # the new buffer less the old one of 64 MiB
    graphs = [_graph(dev, c) for c in calls]
    mid = free()
    larger()
    dev.ctx.sync()
    kept = mid - free()
    vals = _Values(0.0, 0.0, 0.0)
    for _ in range(2):  # the first buffer of these graphs is still theirs
        for h, c in zip(graphs, calls):
            dev.call("om_fill", c.o, C.c_float(np.nan), 16 * 512)
            assert dev.ctx.L.om_graph_launch(h, C.byref(vals)) == 0
            assert np.abs(dev.get(c.o) - 0.25).max() < 1e-6
        larger()
    assert dev.ctx.L.om_graph_destroy(graphs[0]) == 0
    one = free()
    assert dev.ctx.L.om_graph_destroy(graphs[1]) == 0
    back = free() - one
    print("MiB:", taken / MIB, kept / MIB, back / MIB, flush=True)
    # the outgrown 64 MiB went at once without a graph, the next one (150 MiB and a quarter more) with the second graph
    assert 150 * MIB <= taken + 64 * MIB <= 215 * MIB
    assert taken + 64 * MIB - 8 * MIB <= back


def test_a_graph_keeps_its_results_when_another_goes(dev):
    """Two graphs, growth, one destroyed: the other's replays are those of the eager call."""
    c = Case(dev, 2, 4, 2, 150, 150, 64, causal=1, cap=8.0)
    eager = c.forward()
    o = dev.empty((2, 150, 4, 64))

    def call():
        dev.call("om_attention_fwd_scored", *c.ins, o, 256, c.st, 2, 150, 150, 64, C.byref(c.form))
    a, b = _graph(dev, call), _graph(dev, call)
    Forward(dev, 200)()
    vals = _Values(0.0, 0.0, 0.0)
    for n in range(3):
        dev.call("om_fill", o, C.c_float(np.nan), 2 * 150 * 256)
        assert dev.ctx.L.om_graph_launch(a, C.byref(vals)) == 0
        assert np.array_equal(dev.get(o).view(np.uint32), eager.view(np.uint32))
        if n == 1:
            assert dev.ctx.L.om_graph_destroy(b) == 0
    assert dev.ctx.L.om_graph_destroy(a) == 0
