"""Windows with sinks, shared prefixes and norms at positions, pages and rows whose offsets pass 32 bits."""
import numpy as np
import pytest

from helpers import assert_close, attention_f64
from seen_ref import PAGE, held, seen
from test_gpu_block_norm import formula
from test_gpu_far_addresses import At

pytestmark = pytest.mark.gpu

H, HKV, D, SCALE = 16, 8, 128, 0.09


class Far:
    """K and V of a few positions in the last pages of a pool of more than 5 GB, through a table of 40,000 pages a sequence."""

    def __init__(self, be, dtype, held_positions, common=0):
        self.be, self.dtype, self.stride = be, dtype, 40000
        self.pages = 41000 if dtype == "f32" else 155000
        self.pool = be.create_page_pool(self.pages, HKV, D, dtype)
        self.table = np.full((len(held_positions), self.stride), -1, np.int32)
        at = self.pages
        for b, pos in enumerate(held_positions):
            for page in np.unique(pos // PAGE):
                if b and page < common // PAGE:
                    self.table[b, page] = self.table[0, page]
                else:
                    at -= 1
                    self.table[b, page] = at
        rng = np.random.default_rng(self.pages)
        self.rows = np.arange(at * PAGE, self.pages * PAGE, dtype=np.int64)
        self.k, self.v = (rng.standard_normal((len(self.rows), HKV * D)).astype(np.float32) for _ in "kv")
        self.pool.write_rows_device(be.buffer(self.rows), be.buffer(self.k), be.buffer(self.v), len(self.rows))
        self.where = dict(page_table=be.buffer(self.table), page_table_stride=self.stride)
        self.q = lambda n: rng.standard_normal((n, H, D)).astype(np.float32)

    def attend(self, b, q, pos):
        i = self.table[b, pos // PAGE].astype(np.int64) * PAGE + pos % PAGE - self.rows[0]
        k, v = (held(t[i], self.dtype).reshape(-1, HKV, D) for t in (self.k, self.v))
        return np.stack([attention_f64(q[h], k[:, h * HKV // H], v[:, h * HKV // H], SCALE) for h in range(H)])


@pytest.mark.parametrize("dtype", ["f32", "q8"])
def test_windows_with_sinks(backend, dtype):
    be, window, sinks = backend, 90, 21
    ends = np.array([40000 * PAGE, 16 * 33000 + 9])
    n = 40  # rows of the prefill, the last one the decode's
    f = Far(be, dtype, [seen(e - n - window, e, sinks) for e in ends])
    q = f.q(2 * n)
    start = (ends - window).astype(np.int32)
    last = q[[n - 1, 2 * n - 1]]
    out, rows = be.empty(last.nbytes), be.empty(q.nbytes)
    be.decode(f.pool, be.buffer(last), out, be.buffer(start), be.buffer(np.full(2, window, np.int32)), 2, window, H, SCALE, n_sinks=sinks,
              **f.where)
    be.prefill(f.pool, be.buffer(q), rows, be.buffer(np.array([0, n, 2 * n], np.int32)), be.buffer((ends - n).astype(np.int32)), 2, n, H,
               SCALE, sliding_window=window, n_sinks=sinks, **f.where)
    be.sync()
    out, rows = out.download(last.shape), rows.download(q.shape)
    for b, e in enumerate(ends):
        assert_close(out[b], f.attend(b, last[b], seen(e - window, e, sinks)))
        for r in (0, 17, n - 1):
            p = e - n + r
            assert_close(rows[b * n + r], f.attend(b, q[b * n + r], seen(p - window + 1, p + 1, sinks)))
    f.pool.destroy()


@pytest.mark.parametrize("dtype", ["f32", "q8"])
def test_a_shared_prefix(backend, dtype, monkeypatch):
    monkeypatch.setenv("GLA_DECODE_PREFIX", "1")
    be, prefix = backend, 600
    ends = np.array([prefix + 40, prefix + 1, prefix + 300], np.int32)
    f = Far(be, dtype, [np.arange(e) for e in ends], common=prefix)
    q = f.q(3)
    out = be.empty(q.nbytes)
    be.decode_shared(f.pool, be.buffer(q), out, be.buffer(np.zeros(3, np.int32)), be.buffer(ends), 3, int(ends.max()), H, SCALE,
                     be.buffer(np.array([0, 3], np.int32)), be.buffer(np.array([prefix // PAGE * PAGE], np.int32)), 1, 3, prefix, 340,
                     **f.where)
    be.sync()
    for b, row in enumerate(out.download(q.shape)):
        assert_close(row, f.attend(b, q[b], np.arange(ends[b])))
    f.pool.destroy()


def test_norms_of_rows_far_apart(backend):
    be, n, dim, apart = backend, 3, 1000, 1 << 30
    rng = np.random.default_rng(7)
    x, y, gate = (rng.standard_normal((n, dim)).astype(np.float32) for _ in range(3))
    post, pre = (rng.standard_normal(dim).astype(np.float32) for _ in range(2))
    buf = be.empty(4 * (apart * (n - 1) + 5 * dim))
    for i in range(n):
        for j, t in enumerate((x, y, gate)):
            At(buf, i * apart + j * dim).put(t[i])
    be.block_norm(At(buf), n, dim, 1e-5, y=At(buf, dim), post=be.buffer(post), gate=At(buf, 2 * dim), scale=0.5, x_out=At(buf, 3 * dim),
                  pre=be.buffer(pre), norm_out=At(buf, 4 * dim), x_stride=apart, y_stride=apart, gate_stride=apart, x_out_stride=apart,
                  norm_out_stride=apart)
    be.sync()
    want, dx, norm, dh = formula(x, y, post, gate, 0.5, pre, 1e-5)
    got, h = (np.stack([At(buf, i * apart + j * dim).get((dim,)) for i in range(n)]) for j in (3, 4))
    assert np.all(np.abs(got - want) <= dx) and np.all(np.abs(h - norm) <= dh)
    buf.free()
