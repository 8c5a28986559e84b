"""gla_kv_append at the edges of what its documentation allows."""
import ctypes as C

import numpy as np
import pytest

from glint_amd import _lib
from glint_amd.attn import HipStream
from test_gpu_append import View

pytestmark = pytest.mark.gpu

PAGE = 16


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


@pytest.mark.parametrize("dtype", ["f32", "q8"])
@pytest.mark.parametrize("n", [1, 5, 40])
def test_rows_that_meet_at_one_place(backend, dtype, n):
    """Three sequences whose tables share their pages: every stored byte is one of the three rows' at its place (which one, the
    call does not say), and the rest of the pool stays. The same for row ids that are repeated."""
    be, n_kv, d, pages = backend, 2, 128, 8
    rng = np.random.default_rng(n)
    k, v = (rng.standard_normal((3 * n, n_kv * d)).astype(np.float32) for _ in "kv")
    shared = np.array([5, 2, 7], np.int32)
    rows = np.array([shared[(3 + i) // PAGE] * PAGE + (3 + i) % PAGE for i in range(n)])
    every = np.arange(pages * PAGE)
    rest = np.setdiff1d(every, rows)
    old = rng.standard_normal((len(every), n_kv * d)).astype(np.float32)

    def pool():
        p = be.create_page_pool(pages, n_kv, d, dtype)
        p.write_rows(every, old, -old)
        return p

    want = []
    for i in range(3):
        p = pool()
        p.write_rows(rows, k[i * n:(i + 1) * n], v[i * n:(i + 1) * n])
        want.append(p.export_rows(every))
    by_append, by_ids = pool(), pool()
    be.append(by_append, be.buffer(k), be.buffer(v), be.buffer(np.arange(0, 3 * n + 1, n, dtype=np.int32)),
              be.buffer(np.full(3, 3, np.int32)), 3, n, page_table=be.buffer(np.tile(shared, (3, 1))), page_table_stride=3)
    by_ids.write_rows(np.tile(rows, 3), k, v)
    be.sync()
    for p in (by_append, by_ids):
        for which, got in enumerate(p.export_rows(every)):
            got = np.asarray(got).view(np.uint8).reshape(len(every), -1)
            each = [np.asarray(t[which]).view(np.uint8).reshape(len(every), -1) for t in want]
            assert np.array_equal(got[rest], each[0][rest])
            assert np.all((got == each[0]) | (got == each[1]) | (got == each[2]))


@pytest.mark.parametrize("dtype", ["f32", "q8"])
@pytest.mark.parametrize("lens", [[1, 1, 1, 1], [40, 0, 17, 1]])
def test_captured_rotation_append_and_reading(backend, dtype, lens):
    """gla_rope_rows, gla_kv_append into a page pool and gla_kv_read_rows in one graph, replayed on another stream than the plan
    was made on, with new rows, positions and pages in between and eager calls beside: every replay has the eager bits."""
    be, heads, n_kv, d, n = backend, 4, 2, 128, sum(lens)
    rng = np.random.default_rng(n)
    plan = be.create_rope_plan(d, layout="half", rot_dim=96)
    s = HipStream()
    try:
        be.set_stream(s)
        pages, stride, width = 40, 8, (heads + 2 * n_kv) * d
        pools = [be.create_page_pool(pages, n_kv, d, dtype) for _ in range(2)]
        starts = be.buffer(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32))
        row, table, past, pos, rows = (be.empty(4 * k) for k in (n * width, 4 * stride, 4, n, 2 * n))
        outs = [[be.empty(4 * n * w) for w in (heads * d, heads * d, n_kv * d, n_kv * d)] for _ in range(2)]

        def step(i):
            turned, q, k, v = outs[i]
            be.rope_rows(plan, row, n, heads, pos, out=turned, x_stride=width)
            be.append(pools[i], View(row, heads * d), View(row, (heads + n_kv) * d), starts, past, 4, max(lens), rope=plan, q=row,
                      q_out=q, n_heads=heads, k_stride=width, v_stride=width, q_stride=width, page_table=table, page_table_stride=stride)
            pools[i].read_rows_device(rows, k, v, n)

        def inputs():
            t = rng.permutation(pages)[:4 * stride].astype(np.int32).reshape(4, stride)
            p = rng.integers(0, stride * PAGE - max(lens) + 1, 4)
            at = np.concatenate([np.arange(a, a + m) for a, m in zip(p, lens)])
            owner = np.repeat(np.arange(4), lens)
            row.upload(rng.standard_normal((n, width)).astype(np.float32))
            table.upload(t), past.upload(p.astype(np.int32)), pos.upload(at.astype(np.int32))
            rows.upload(t[owner, at // PAGE].astype(np.int64) * PAGE + at % PAGE)

        inputs()
        g = be.capture(lambda: step(1))
        for rep in range(5):
            inputs()
            step(0)
            g.replay()
            be.sync()
            for a, b, w in zip(*outs, (heads * d, heads * d, n_kv * d, n_kv * d)):
                a, b = a.download((n, w)), b.download((n, w))
                assert np.isfinite(a).all() and np.array_equal(a.view(np.uint32), b.view(np.uint32)), rep
            assert np.array_equal(outs[0][0].download((n, heads * d)), outs[0][1].download((n, heads * d)))
            for a, b in zip(*(p.export_rows(np.arange(pages * PAGE)) for p in pools)):
                assert np.array_equal(a, b), rep
        g.destroy()
    finally:
        be.set_stream(None)
        s.destroy()
