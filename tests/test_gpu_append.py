"""gla_kv_append and gla_kv_read_rows: rotated rows in the places that prefill and decode read, and nothing else touched."""
import ctypes as C

import numpy as np
import pytest

import oracle as orc
import rope_ref
from glint_amd import _lib

pytestmark = pytest.mark.gpu

PAGE = 16


class View:
    """A device buffer from `floats` on."""

    def __init__(self, buf, floats):
        self.buf, self.ptr = buf, C.c_void_p(buf.ptr.value + 4 * floats)


def q8_values(x):
    """f32 rows [n][kv_dim] as Q8_0 holds them: exported bytes, and the values."""
    raw = orc.q8_quantize_rows(np.ascontiguousarray(x, np.float32))
    raw = raw.reshape(len(x), -1, 34)
    d = raw[..., :2].copy().view(np.float16).astype(np.float32)
    return raw.reshape(len(x), -1), (raw[..., 2:].view(np.int8).astype(np.float32) * d).reshape(len(x), -1)


def rows_of(lens, past, table=None, seq=None, layers=1, layer=0, ppl=0):
    """Storage rows of a batch's new positions."""
    out = []
    for b, (n, p) in enumerate(zip(lens, past)):
        for pos in range(p, p + n):
            page = table[b, pos // PAGE] if table is not None else ((seq[b] if seq is not None else b) * layers + layer) * ppl + pos // PAGE
            out.append(int(page) * PAGE + pos % PAGE)
    return np.array(out, np.int64)


def batch(rng, n_heads, n_kv, d, lens, fused, pad=0):
    n = int(sum(lens))
    q, k, v = (rng.standard_normal((n, h, d)).astype(np.float32) for h in (n_heads, n_kv, n_kv))
    if not fused:
        return q, k, v, None
    row = np.concatenate([q.reshape(n, -1), k.reshape(n, -1), v.reshape(n, -1), np.full((n, pad), 3.25, np.float32)], 1)
    return q, k, v, row


def append(be, kv, q, k, v, fused, lens, past, plan, with_q=True, max_len=None, tail=0, **where):
    """The call; returns the rotated q with `tail` rows behind the last sequence's."""
    n = int(sum(lens))
    n_heads, n_kv, d = q.shape[1], k.shape[1], k.shape[2]
    qs = be.buffer(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32))
    off = be.buffer(np.asarray(past, np.int32))
    out = be.buffer(np.full(((n + tail), n_heads * d), -9.0, np.float32))
    kw = dict(where)
    if fused is not None:
        buf = be.buffer(fused if n else np.zeros((1, 4), np.float32))
        stride = fused.shape[1]
        bq, bk, bv = View(buf, 0), View(buf, n_heads * d), View(buf, (n_heads + n_kv) * d)
        kw.update(q_stride=stride, k_stride=stride, v_stride=stride)
    else:
        bq, bk, bv = (be.buffer(t) for t in (q, k, v))
    if with_q:
        kw.update(q=bq, q_out=out, n_heads=n_heads)
    else:
        kw.pop("q_stride", None)
    be.append(kv, bk, bv, qs, off, len(lens), max(lens) if max_len is None else max_len, rope=plan, **kw)
    be.sync()
    return out.download((n + tail, n_heads, d))


def read(be, kv, rows):
    n, kv_dim = len(rows), kv.kv_dim
    k, v = be.empty(n * kv_dim * 4), be.empty(n * kv_dim * 4)
    kv.read_rows_device(be.buffer(np.asarray(rows, np.int64)), k, v, n)
    be.sync()
    return k.download((n, kv_dim)), v.download((n, kv_dim))


def check_f32(got, x, pos, spec):
    want, tol = rope_ref.rotate(x, pos, **spec)
    assert np.all(np.abs(got.reshape(x.shape).astype(np.float64) - want) <= tol)


SPECS = {
    "adjacent": dict(layout="interleaved"),
    "half": dict(layout="half", freq_base=500000.0, scaling="bands", factor=8.0, original_ctx=8192, low=1.0, high=4.0),
    "part": dict(layout="half", rot_dim=48, scaling="linear", factor=2.0),
    "odd": dict(layout="half", rot_dim=22),
    "odd-adjacent": dict(layout="interleaved", rot_dim=22, scaling="yarn", factor=4.0, original_ctx=2048),
    "none": None,
}


@pytest.mark.parametrize("spec", SPECS)
@pytest.mark.parametrize("dtype", ["f32", "q8"])
@pytest.mark.parametrize("n_heads, n_kv, d", [(9, 3, 64), (32, 8, 128), (4, 2, 256), (1, 1, 64)])
def test_pool_rows(backend, spec, dtype, n_heads, n_kv, d):
    """Ragged chunks that begin and end inside pages, an empty one among them; a decode step; every byte elsewhere stays."""
    be, spec = backend, SPECS[spec]
    rng = np.random.default_rng(d + n_heads)
    for lens, past in (([1, 1, 1], [0, 15, 70]), ([37, 0, 16, 5, 1], [3, 8, 16, 14, 31]), ([70], [0])):
        need = [(p + n + PAGE - 1) // PAGE for p, n in zip(past, lens)]
        pages = sum(need) + 2
        perm = rng.permutation(pages)
        table = np.full((len(lens), max(need) + 1), -1, np.int32)
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = perm[at:at + n]
            at += n
        pool = be.create_page_pool(pages, n_kv, d, dtype)
        every = np.arange(pages * PAGE, dtype=np.int64)
        old_k, old_v = (rng.standard_normal((len(every), n_kv * d)).astype(np.float32) for _ in "kv")
        pool.write_rows(every, old_k, old_v)
        before = [t.copy() for t in pool.export_rows(every)]
        plan = be.create_rope_plan(d, **spec) if spec else None
        fused = len(lens) != 3
        q, k, v, row = batch(rng, n_heads, n_kv, d, lens, fused)
        got_q = append(be, pool, q, k, v, row, lens, past, plan, tail=2, page_table=be.buffer(table),
                       page_table_stride=table.shape[1])
        pos = np.concatenate([np.arange(p, p + n) for p, n in zip(past, lens)])
        rows = rows_of(lens, past, table=table)
        assert np.all(got_q[len(pos):] == -9.0)
        if spec:
            check_f32(got_q[:len(pos)], q, pos, spec)
            k_turned = rope_ref.rotate(k, pos, **spec)[0].astype(np.float32).reshape(len(pos), -1)
        else:
            assert np.array_equal(got_q[:len(pos)], q)
            k_turned = k.reshape(len(pos), -1)
        v_flat = v.reshape(len(pos), -1)
        after = pool.export_rows(every)
        rest = np.setdiff1d(every, rows)
        assert all(np.array_equal(a[rest], b[rest]) for a, b in zip(after, before))
        rk, rv = read(be, pool, rows)
        if dtype == "f32":
            if spec:
                check_f32(rk, k, pos, spec)
            else:
                assert np.array_equal(rk, k_turned)
            assert np.array_equal(rv, v_flat)
        else:
            # the quantiser's own rules on the value rounded once: bit for bit
            for x, raw, values in ((k_turned, after[0], rk), (v_flat, after[1], rv)):
                want, want_values = q8_values(x)
                assert np.array_equal(raw[rows], want)
                assert np.array_equal(values, want_values)


@pytest.mark.parametrize("dtype", ["f32", "q8"])
def test_cache_rows_by_layer_and_slot(backend, dtype):
    be = backend
    n_seqs, layers, max_seq, n_kv, d = 4, 3, 50, 2, 64
    cache = be.create_kv_cache(layers, max_seq, n_kv, d, dtype, n_seqs)
    ppl = (max_seq + PAGE - 1) // PAGE
    rng = np.random.default_rng(8)
    lens, past, seq = [5, 1, 20], [45, 0, 17], [3, 0, 1]
    plan = be.create_rope_plan(d, layout="half")
    q, k, v, row = batch(rng, 4, n_kv, d, lens, True, pad=4)
    got_q = append(be, cache, q, k, v, row, lens, past, plan, layer=1, seq_slot=be.buffer(np.array(seq, np.int32)))
    pos = np.concatenate([np.arange(p, p + n) for p, n in zip(past, lens)])
    check_f32(got_q, q, pos, dict(layout="half"))
    rows = rows_of(lens, past, seq=seq, layers=layers, layer=1, ppl=ppl)
    assert rows[0] == cache.row_id(3, 1, 45)
    rk, rv = read(be, cache, rows)
    turned = rope_ref.rotate(k, pos, layout="half")[0].astype(np.float32).reshape(len(pos), -1)
    if dtype == "q8":
        assert np.array_equal(rk, q8_values(turned)[1]) and np.array_equal(rv, q8_values(v.reshape(len(pos), -1))[1])
    else:
        check_f32(rk, k, pos, dict(layout="half"))
    every = np.arange(n_seqs * layers * ppl * PAGE, dtype=np.int64)
    rest = np.setdiff1d(every, rows)
    assert not any(t.any() for t in read(be, cache, rest))


@pytest.mark.parametrize("dtype", ["f32", "q8"])
def test_rows_without_a_place_are_not_stored(backend, dtype):
    """Positions past the storage or below 0, slots and pages that do not exist: nothing is written for them, and their
    queries are rotated all the same."""
    be = backend
    n_kv, d = 2, 64
    rng = np.random.default_rng(9)
    plan = be.create_rope_plan(d)
    # positions -2 .. 3 of sequence 0; 30 .. 34 of sequence 1, whose table ends at 32; a table of nonsense pages
    lens, past = [6, 5, 3], [-2, 30, 0]
    pos = np.concatenate([np.arange(p, p + n) for p, n in zip(past, lens)])
    q, k, v, row = batch(rng, 2, n_kv, d, lens, True)
    table = np.array([[0, 1], [2, 3], [-1, 99]], np.int32)
    pool = be.create_page_pool(5, n_kv, d, dtype)
    got_q = append(be, pool, q, k, v, row, lens, past, plan, page_table=be.buffer(table), page_table_stride=2)
    check_f32(got_q, q, pos, {})
    stored = np.array([0, 1, 2, 3, 2 * 0 + 3 * PAGE + 14, 3 * PAGE + 15])
    rk, rv = read(be, pool, np.arange(5 * PAGE))
    kept = np.abs(rv).sum(1) > 0
    assert np.array_equal(np.flatnonzero(kept), stored)
    cache = be.create_kv_cache(1, 32, n_kv, d, dtype, 2)
    got_q = append(be, cache, q, k, v, row, lens, past, plan, seq_slot=be.buffer(np.array([1, 0, 2], np.int32)))
    check_f32(got_q, q, pos, {})
    rk, rv = read(be, cache, np.arange(2 * 32))
    assert np.array_equal(np.flatnonzero(np.abs(rv).sum(1) > 0), [30, 31, 32, 33, 34, 35])


def test_without_q_and_in_place(backend):
    be = backend
    n_kv, d, lens, past = 2, 128, [3, 4], [0, 9]
    rng = np.random.default_rng(10)
    plan = be.create_rope_plan(d, layout="half")
    q, k, v, _ = batch(rng, 4, n_kv, d, lens, False)
    cache = be.create_kv_cache(1, 16, n_kv, d, "f32", 2)
    pos = np.concatenate([np.arange(p, p + n) for p, n in zip(past, lens)])
    untouched = append(be, cache, q, k, v, None, lens, past, plan, with_q=False)
    assert np.all(untouched == -9.0)
    rk, _ = read(be, cache, rows_of(lens, past, ppl=1))
    check_f32(rk, k, pos, dict(layout="half"))
    bq = be.buffer(q)
    be.append(cache, be.buffer(k), be.buffer(v), be.buffer(np.array([0, 3, 7], np.int32)), be.buffer(np.array(past, np.int32)),
              2, 4, rope=plan, q=bq, n_heads=4)
    be.sync()
    check_f32(bq.download(q.shape), q, pos, dict(layout="half"))


def test_rows_past_max_q_len_and_misaligned_rows(backend):
    """Rows of a sequence past max_q_len are left alone; rows 4 bytes off 16-byte addresses take the element loads."""
    be = backend
    n_kv, d = 2, 64
    rng = np.random.default_rng(11)
    q, k, v, _ = batch(rng, 2, n_kv, d, [5], False)
    plan = be.create_rope_plan(d, layout="half", rot_dim=20)
    spec = dict(layout="half", rot_dim=20)
    for dtype in ("f32", "q8"):
        cache = be.create_kv_cache(1, 16, n_kv, d, dtype, 1)
        width = 4 * 64 + 64 * 2 + 3
        row = np.zeros((5, width), np.float32)
        row[:, 1:129], row[:, 130:258], row[:, 259:387] = (t.reshape(5, -1) for t in (q, k, v))
        buf = be.buffer(row)
        out = be.buffer(np.full((5, 128), -9.0, np.float32))
        be.append(cache, View(buf, 130), View(buf, 259), be.buffer(np.array([0, 5], np.int32)), be.buffer(np.array([2], np.int32)),
                  1, 3, rope=plan, q=View(buf, 1), q_out=out, n_heads=2, k_stride=width, v_stride=width, q_stride=width)
        be.sync()
        got = out.download((5, 2, d))
        check_f32(got[:3], q[:3], [2, 3, 4], spec)
        assert np.all(got[3:] == -9.0)
        rk, rv = read(be, cache, np.arange(16))
        assert np.array_equal(np.flatnonzero(np.abs(rv).sum(1) > 0), [2, 3, 4])
        turned = rope_ref.rotate(k[:3], [2, 3, 4], **spec)[0].astype(np.float32).reshape(3, -1)
        if dtype == "q8":
            assert np.array_equal(rk[2:5], q8_values(turned)[1])
        else:
            check_f32(rk[2:5], k[:3], [2, 3, 4], spec)


def test_read_rows_out_of_range_and_repeated(backend):
    be = backend
    for dtype in ("f32", "q8"):
        pool = be.create_page_pool(2, 2, 64, dtype)
        x = np.random.default_rng(12).standard_normal((32, 128)).astype(np.float32)
        pool.write_rows(np.arange(32), x, -x)
        rows = np.array([5, -1, 5, 32, 31, 1 << 40], np.int64)
        k, v = be.buffer(np.full((6, 128), 2.5, np.float32)), be.buffer(np.full((6, 128), 2.5, np.float32))
        pool.read_rows_device(be.buffer(rows), k, v, 6)
        be.sync()
        gk, gv = k.download((6, 128)), v.download((6, 128))
        want = x if dtype == "f32" else q8_values(x)[1]
        assert np.array_equal(gk[[0, 2, 4]], want[[5, 5, 31]]) and np.array_equal(gv[[0, 2, 4]], -want[[5, 5, 31]])
        assert np.all(gk[[1, 3, 5]] == 2.5) and np.all(gv[[1, 3, 5]] == 2.5)


def test_refusals(backend):
    be, lib = backend, _lib.lib()
    pool, cache = be.create_page_pool(2, 2, 64), be.create_kv_cache(2, 16, 2, 64)
    plan, wide = be.create_rope_plan(64), be.create_rope_plan(128)
    buf = be.buffer(np.zeros(4096, np.float32))
    ints = be.buffer(np.zeros(8, np.int32))

    def call(**kw):
        a = _lib.AppendArgs()
        a.kv, a.n_seqs, a.max_q_len, a.rope = cache.handle, 1, 1, plan.handle
        a.k = a.v = a.q = a.q_out = buf.ptr
        a.q_start = a.pos_offset = ints.ptr
        a.n_heads = 2
        for key, val in kw.items():
            setattr(a, key, val)
        return lib.gla_kv_append(be.ctx, C.byref(a))

    assert call() == _lib.GLA_OK  # an empty sequence: q_start is 0, 0
    assert call(n_seqs=0, k=None) == _lib.GLA_OK and call(max_q_len=0, k=None) == _lib.GLA_OK
    for kw in (dict(kv=None), dict(n_seqs=-1), dict(max_q_len=-1), dict(rope=wide.handle), dict(k=None), dict(v=None),
               dict(q_start=None), dict(pos_offset=None), dict(q_out=None), dict(n_heads=3), dict(n_heads=0), dict(k_stride=127),
               dict(v_stride=-1), dict(q_stride=100), dict(q_stride=256), dict(layer=2), dict(layer=-1),
               dict(page_table=ints.ptr), dict(kv=pool.handle), dict(kv=pool.handle, page_table=ints.ptr),
               dict(kv=pool.handle, page_table=ints.ptr, page_table_stride=-1),
               dict(kv=pool.handle, page_table=ints.ptr, page_table_stride=1 << 28), dict(max_q_len=(1 << 31) - 1)):
        assert call(**kw) == _lib.GLA_ERR_INVALID, kw
    assert call(q=None, q_out=None, n_heads=0) == _lib.GLA_OK
    for args in ((None, buf.ptr, buf.ptr, 1), (ints.ptr, None, buf.ptr, 1), (ints.ptr, buf.ptr, None, 1),
                 (ints.ptr, buf.ptr, buf.ptr, -1), (ints.ptr, C.c_void_p(buf.ptr.value + 4), buf.ptr, 1)):
        assert lib.gla_kv_read_rows(be.ctx, cache.handle, *args) == _lib.GLA_ERR_INVALID
    be.sync()


@pytest.mark.parametrize("n", [3, 40])
def test_quants_of_every_magnitude(backend, n):
    """Blocks whose quotients fall on halves, blocks from the smallest subnormals to the largest floats, with zeros, infinities
    and NaN: the storage's bytes are the oracle's, row by row and page by page."""
    be = backend
    rng = np.random.default_rng(n)
    k = rng.integers(-254, 255, (n, 8, 32)).astype(np.float64) / 2 * 2.0 ** rng.integers(-149, 120, (n, 8, 1))
    k[..., 0] = np.where(rng.random((n, 8)) < 0.8, 127.0, 1.0) * np.abs(k).max(-1) / 127.0
    k[rng.random(k.shape) < 0.03] = 0.0
    odd = rng.random(k.shape) < 0.002
    k[odd] = rng.choice([np.inf, -np.inf, np.nan], odd.sum())
    k[0, 0] = 0.0
    k[1, 1] = 2.0 ** -149
    k = np.clip(k, -3.4e38, 3.4e38, where=np.isfinite(k), out=k).astype(np.float32).reshape(n, 256)
    v = k[:, ::-1].copy()
    cache = be.create_kv_cache(1, 48, 2, 128, "q8", 1)
    be.append(cache, be.buffer(k), be.buffer(v), be.buffer(np.array([0, n], np.int32)), be.buffer(np.array([5], np.int32)), 1, n)
    be.sync()
    for got, x in zip(cache.export_rows(np.arange(5, 5 + n)), (k, v)):
        assert np.array_equal(np.asarray(got, np.uint8).reshape(n, -1), q8_values(x)[0])


@pytest.mark.parametrize("n_heads, n_kv, d", [(4, 2, 64), (16, 8, 128), (2, 1, 256)])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_long_prompts_into_a_quantised_pool(backend, n_heads, n_kv, d, layout):
    """Prompts of several hundred rows beside short ones: the pool holds what write_rows stores of the rotated rows, every
    query is rotated, and rows outside the prompts stay as they were."""
    be = backend
    rng = np.random.default_rng(d)
    lens, past = [300, 5, 0, 131, 517], [3, 16, 9, 21, 0]
    q, k, v, row = batch(rng, n_heads, n_kv, d, lens, True)
    pages = sum(-(-(n + p) // PAGE) for n, p in zip(lens, past))
    order, table, at = rng.permutation(pages).astype(np.int32), np.full((5, 40), -1, np.int32), 0
    for b, (n, p) in enumerate(zip(lens, past)):
        m = -(-(n + p) // PAGE)
        table[b, :m] = order[at:at + m]
        at += m
    spec = dict(layout=layout, freq_base=500000.0)
    pools = [be.create_page_pool(pages, n_kv, d, "q8") for _ in range(2)]
    plan = be.create_rope_plan(d, **spec)
    got = append(be, pools[0], q, k, v, row, lens, past, plan, tail=2, page_table=be.buffer(table), page_table_stride=40)
    pos = np.concatenate([np.arange(p, p + n) for n, p in zip(lens, past)])
    check_f32(got[:len(pos)], q, pos, spec)
    assert np.all(got[len(pos):] == -9.0)
    # K as the library rotates it alone (one rounding, so the same f32), written row by row
    turned = be.buffer(k)
    be.rope_rows(plan, turned, len(pos), n_kv, be.buffer(pos.astype(np.int32)))
    be.sync()
    check_f32(turned.download(k.shape), k, pos, spec)
    pools[1].write_rows(rows_of(lens, past, table=table), turned.download((len(pos), n_kv * d)), v.reshape(len(pos), -1))
    every = np.arange(pages * PAGE)
    for a, b in zip(pools[0].export_rows(every), pools[1].export_rows(every)):
        assert np.array_equal(a, b)
