"""gla_kv_append at the edges of what its documentation allows."""
import ctypes as C

import numpy as np
import pytest

from glint_amd import _lib

pytestmark = pytest.mark.gpu


def test_more_sequences_than_a_launch_has_are_refused(backend):
    """The count of workgroups along z is made of n_seqs: neither its sum nor the launch may overflow. (No array of that length
    is behind the pointers: the host has to refuse.)"""
    be, lib = backend, _lib.lib()
    cache = be.create_kv_cache(1, 16, 2, 64)
    buf, ints = be.buffer(np.zeros(256, np.float32)), be.buffer(np.zeros(8, np.int32))
    a = _lib.AppendArgs()
    a.kv, a.max_q_len = cache.handle, 1
    a.k = a.v = buf.ptr
    a.q_start = a.pos_offset = ints.ptr
    for n in ((1 << 31) - 1, 65535 * 32768 + 1):
        a.n_seqs = n
        assert lib.gla_kv_append(be.ctx, C.byref(a)) == _lib.GLA_ERR_INVALID and "n_seqs" in _lib.last_error()
    a.n_seqs = 1
    assert lib.gla_kv_append(be.ctx, C.byref(a)) == _lib.GLA_OK
    be.sync()
