"""Rows, storages and weights whose offsets pass 32 bits: rotation, append, rows read back and 4-bit projections."""
import ctypes as C

import numpy as np
import pytest

import q4_structured as st
import rope_ref
from glint_amd import _lib
from glint_amd.attn import HipStream, _hip
from test_gpu_append import PAGE, check_f32, q8_values
from test_gpu_matvec_q4 import ggml, parts

pytestmark = pytest.mark.gpu


class At:
    """A device address: `floats` behind a buffer's start."""

    def __init__(self, buf, floats=0):
        self.buf, self.ptr = buf, C.c_void_p(buf.ptr.value + 4 * floats)

    def put(self, x):
        x = np.ascontiguousarray(x, np.float32)
        _lib.check(_lib.lib().gla_memcpy_htod(self.buf.backend.ctx, self.ptr, x.ctypes.data_as(C.c_void_p), x.nbytes))

    def get(self, shape):
        x = np.empty(shape, np.float32)
        _lib.check(_lib.lib().gla_memcpy_dtoh(self.buf.backend.ctx, x.ctypes.data_as(C.c_void_p), self.ptr, x.nbytes))
        return x


@pytest.mark.parametrize("dtype", ["f32", "q8"])
def test_the_last_pages_of_a_large_pool(backend, dtype):
    """A pool of more than 5 GB: rows appended at far positions into its last pages, through a table of 40,000 pages a sequence,
    by rows and by pages of V, and read back."""
    be, n_kv, d = backend, 8, 128
    pages = 41000 if dtype == "f32" else 155000
    pool = be.create_page_pool(pages, n_kv, d, dtype)
    rng = np.random.default_rng(41)
    stride = 40000
    table = np.full((2, stride), -1, np.int32)
    plan = be.create_rope_plan(d, layout="half")
    for lens in ([3, 5], [40, 17]):
        past = [stride * PAGE - lens[0], 16 * 33000 + 9]
        for b in range(2):
            for lp in range(past[b] // PAGE, (past[b] + lens[b] - 1) // PAGE + 1):
                table[b, lp] = pages - 1 - (b * 8 + lp - past[b] // PAGE)
        n = sum(lens)
        k, v = (rng.standard_normal((n, n_kv, d)).astype(np.float32) for _ in "kv")
        be.append(pool, be.buffer(k), be.buffer(v), be.buffer(np.array([0, lens[0], n], np.int32)), be.buffer(np.array(past, np.int32)),
                  2, max(lens), rope=plan, page_table=be.buffer(table), page_table_stride=stride)
        pos = np.concatenate([np.arange(p, p + m) for p, m in zip(past, lens)])
        owner = np.repeat([0, 1], lens)
        rows = table[owner, pos // PAGE].astype(np.int64) * PAGE + pos % PAGE
        out = [be.empty(n * n_kv * d * 4) for _ in "kv"]
        pool.read_rows_device(be.buffer(rows), *out, n)
        be.sync()
        gk, gv = (t.download((n, n_kv * d)) for t in out)
        if dtype == "f32":
            check_f32(gk, k, pos, dict(layout="half"))
            assert np.array_equal(gv, v.reshape(n, -1))
        else:
            turned = rope_ref.rotate(k, pos, layout="half")[0].astype(np.float32)
            assert np.array_equal(gk, q8_values(turned.reshape(n, -1))[1]) and np.array_equal(gv, q8_values(v.reshape(n, -1))[1])
    pool.destroy()


def test_rows_far_apart(backend):
    """Rows 2^30 floats apart, rotated into rows beside them and, with the same strides, appended."""
    be, heads, d, n, apart = backend, 4, 64, 3, 1 << 30
    rng = np.random.default_rng(42)
    x = rng.standard_normal((n, heads, d)).astype(np.float32)
    buf = be.empty(4 * (apart * (n - 1) + 4 * heads * d))
    width = heads * d
    for i in range(n):
        At(buf, i * apart).put(x[i])
    pos = np.array([5, 70000, 131071], np.int32)
    plan = be.create_rope_plan(d, layout="half")
    be.rope_rows(plan, At(buf), n, heads, be.buffer(pos), out=At(buf, 2 * width), x_stride=apart, out_stride=apart)
    be.sync()
    got = np.stack([At(buf, i * apart + 2 * width).get((heads, d)) for i in range(n)])
    check_f32(got, x, pos, dict(layout="half"))
    cache = be.create_kv_cache(1, 16, 2, d, "f32", 1)
    q_out, out = be.empty(n * 2 * d * 4), [be.empty(n * 2 * d * 4) for _ in "kv"]
    be.append(cache, At(buf), At(buf, 2 * d), be.buffer(np.array([0, n], np.int32)), be.buffer(np.array([4], np.int32)), 1, n, rope=plan,
              q=At(buf), q_out=q_out, n_heads=2, k_stride=apart, v_stride=apart, q_stride=apart)
    cache.read_rows_device(be.buffer(np.arange(4, 4 + n, dtype=np.int64)), *out, n)
    be.sync()
    check_f32(q_out.download((n, 2, d)), x[:, :2], np.arange(4, 4 + n), dict(layout="half"))
    check_f32(out[0].download((n, 2 * d)), x[:, :2], np.arange(4, 4 + n), dict(layout="half"))
    assert np.array_equal(out[1].download((n, 2, d)), x[:, 2:])
    buf.free()


def zeros(be, nbytes):
    buf = be.empty(nbytes)
    assert _hip().hipMemset(buf.ptr, 0, C.c_size_t(nbytes)) == 0 and _hip().hipDeviceSynchronize() == 0
    return buf


@pytest.mark.parametrize("fmt", ["q4_0", "q4_k"])
@pytest.mark.parametrize("rows, n", [(33, 32768), (33, 40000), (1040, 40000)])
def test_vectors_past_32_bits(backend, fmt, rows, n):
    """2^31 elements of x and more, whose pieces take as many bytes again: vectors at both ends and in between are products of
    theirs, the others 0."""
    be, cols = backend, 65536
    rng = np.random.default_rng(43)
    raw = ggml(rng, fmt, rows, cols)
    w = be.create_q4_weights(raw, rows, cols, fmt)
    wd, wm = parts(raw, fmt)
    at = [0, 1, 8191, 16384, 32700, n - 2, n - 1]
    x = st.vectors(rng, len(at), cols, 30000)
    s = HipStream()
    try:
        be.set_stream(s)
        bx, by = zeros(be, n * cols * 4), be.empty(n * rows * 4)
        for i, v in zip(at, x):
            At(bx, i * cols).put(v)
        be.matvec_q4(w, bx, n, by)
        be.sync()
        y = by.download((n, rows))
        assert st.holds(y[at], x, wd, wm)
        assert not np.delete(y, at, 0).any()
        bx.free(), by.free()
    finally:
        be.set_stream(None)
        s.destroy()


@pytest.mark.parametrize("fmt", ["q4_0", "q4_k"])
@pytest.mark.parametrize("unit, again, cols, ns", [(64, 2048, 65536, (1, 3, 8, 16, 130)), (16, 256, 1 << 21, (1, 5, 16, 33))])
def test_weights_past_32_bits(backend, fmt, unit, again, cols, ns):
    """8.6 * 10^9 weights, 4.8 GB, tall and wide: the same rows again and again give the same outputs again and again, from each
    kernel, and five rows of their own behind them."""
    be = backend
    rng = np.random.default_rng(44)
    raw, tail = ggml(rng, fmt, unit, cols), ggml(rng, fmt, 5, cols)
    rows = unit * again + 5
    w = be.create_q4_weights(np.concatenate([np.broadcast_to(raw.reshape(1, -1), (again, raw.size)).reshape(-1), tail.reshape(-1)]), rows, cols, fmt)
    wd, wm = (np.concatenate(t) for t in zip(parts(raw, fmt), parts(tail, fmt)))
    s = HipStream()
    try:
        be.set_stream(s)
        for n in ns:
            x = st.vectors(rng, n, cols, cols - 700)
            bx, by = be.buffer(x), be.empty(n * rows * 4)
            be.matvec_q4(w, bx, n, by)
            be.sync()
            y = by.download((n, rows))
            block = y[:, :-5].reshape(n, again, unit)
            assert np.array_equal(block, np.broadcast_to(block[:, :1], block.shape)), n
            assert st.holds(np.concatenate([block[:, -1], y[:, -5:]], 1), x, wd, wm), n
            bx.free(), by.free()
        w.destroy()
    finally:
        be.set_stream(None)
        s.destroy()
