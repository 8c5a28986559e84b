"""The bound of tests/q4_structured.py on the CPU: it passes the product in pieces, and fails it with a mistake planted, at every
width that the GPU test takes."""
import numpy as np
import pytest

import q4_structured as st
from test_gpu_matvec_q4 import ggml, parts
from test_gpu_q4_edges import STRUCTURED


@pytest.mark.parametrize("fmt, rows, cols", STRUCTURED)
def test_planted_mistakes_are_found(fmt, rows, cols):
    rng = np.random.default_rng(cols)
    rows = min(rows, 64)
    wd, wm = parts(ggml(rng, fmt, rows, cols), fmt)
    for n in (1, 6, 40):
        x = st.vectors(rng, n, cols)
        assert st.holds(st.in_pieces(x, wd, wm), x, wd, wm)
        for mistake in ("lost", "shifted"):
            assert not st.holds(st.in_pieces(x, wd, wm, mistake), x, wd, wm), mistake
    if cols > 16384:
        x = st.vectors(rng, 40, cols, first=16384)
        assert st.holds(st.in_pieces(x, wd, wm), x, wd, wm)
        assert not st.holds(st.in_pieces(x, wd, wm, "tail"), x, wd, wm)
