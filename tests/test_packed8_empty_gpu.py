"""Backward passes of the 8-bit tensors over no rows, on a context of its own that has no scratch yet: what they leave does not
depend on what ran before."""
import pytest

from gpu_util import Dev

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cols", [5, 3000, 9000])
@pytest.mark.parametrize("both", [True, False])
def test_layernorm_backward_of_no_rows_on_a_fresh_context(cols, both):
    dev = Dev()
    A, B = dev.empty((cols,), fill=2.0), dev.empty((cols,), fill=2.0)
    dev.call("om_layernorm_bwd_x8", None, None, None, None, None, A if both else None, B, 0, cols, 0, 1)
    assert (dev.get(A) == 2.0).all() and (dev.get(B) == 2.0).all()
    dev.call("om_layernorm_bwd_x8", None, None, None, None, None, A if both else None, B, 0, cols, 0, 0)
    assert not dev.get(B).any()
    assert (dev.get(A) == (0.0 if both else 2.0)).all()


def test_linear_backward_of_no_rows_on_a_fresh_context():
    dev = Dev()
    A, B = dev.empty((7, 300), fill=2.0), dev.empty((7,), fill=2.0)
    dev.call("om_linear_bwd_x8", None, None, None, None, A, B, 0, 300, 7, 0, 1, 1)
    assert (dev.get(A) == 2.0).all() and (dev.get(B) == 2.0).all()
    dev.call("om_linear_bwd_x8", None, None, None, None, A, B, 0, 300, 7, 0, 0, 0)
    assert not dev.get(A).any() and not dev.get(B).any()
