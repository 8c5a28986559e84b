"""A call that the device has no memory for is refused alone: the next one's launch does not report its error."""
import numpy as np
import pytest

from glint_amd import _lib
from glint_amd._lib import GlaError

pytestmark = pytest.mark.gpu


def refused(what):
    with pytest.raises(GlaError) as e:
        what()
    assert e.value.code == _lib.GLA_ERR_BUFFER


@pytest.mark.parametrize("first", ["scratch", "storage", "buffer"])
def test_the_call_after_a_refused_allocation(backend, first):
    """Sizes of terabytes, which the allocator refuses before anything is launched."""
    be = backend
    cols = 1 << 22
    wide = be.create_q4_weights(np.zeros(cols // 32 * 18, np.uint8), 1, cols)
    w = be.create_q4_weights(np.zeros((16, 18), np.uint8), 16, 32)
    x, y = be.buffer(np.ones((20, 32), np.float32)), be.buffer(np.full((20, 16), 5.0, np.float32))
    if first == "scratch":  # 4.4 TB of pieces
        refused(lambda: be.matvec_q4(wide, x, 262128, y))
    elif first == "storage":  # 8.8 TB
        refused(lambda: be.create_page_pool(1 << 27, 8, 128, "f32"))
    elif first == "buffer":
        refused(lambda: be.empty(1 << 43))
    be.matvec_q4(w, x, 20, y)
    be.sync()
    assert np.all(y.download((20, 16)) == 0)
    if first == "storage":
        be.create_page_pool(2, 8, 128, "f32").destroy()
    plan = be.create_rope_plan(32)
    be.rope_rows(plan, x, 20, 1, be.buffer(np.zeros(20, np.int32)))
    be.sync()
    wide.destroy(), w.destroy()
