"""Refusals of 4-bit weights before the library reads them: no device needed."""
import subprocess
import sys

import pytest

CODE = """
import numpy as np
from glint_amd.attn import GpuBackend
be = object.__new__(GpuBackend)  # no context: the bytes are counted first
be.ctx = None
for n, rows, cols, fmt in ((18, 2, 32, "q4_0"), (17, 1, 32, "q4_0"), (144, 1, 512, "q4_k"), (0, 1, 256, "q4_k")):
    try:
        be.create_q4_weights(np.zeros(n, np.uint8), rows, cols, fmt)
    except ValueError as e:
        assert "no %d x %d matrix" % (rows, cols) in str(e)
    else:
        raise SystemExit("taken: %s" % ((n, rows, cols, fmt),))
"""


@pytest.mark.parametrize("flags", [[], ["-O"]], ids=["", "optimised"])
def test_bytes_that_are_not_the_matrix_are_refused(hip_lib, flags):
    """Also where assertions are off: the library would read past the array."""
    proc = subprocess.run([sys.executable, *flags, "-c", CODE], capture_output=True, text=True, timeout=120)
    assert proc.returncode == 0, proc.stdout + proc.stderr
