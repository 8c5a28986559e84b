"""The operators as a layer uses them: a fused 4-bit Q/K/V projection, the append that rotates and stores, attention and the
4-bit output projection, on a paged or contiguous cache; every stage against 64 bits from the stage's own input on the device.
Then the same steps captured into a graph, and on two streams."""
import ctypes as C

import numpy as np
import pytest

import rope_ref
import test_gpu_matvec_q4 as q4
from glint_amd import _lib
from glint_amd._lib import GlaError
from glint_amd.attn import HipStream
from helpers import assert_close, attention_f64
from test_gpu_append import PAGE, View, read, rows_of

pytestmark = pytest.mark.gpu

H, HKV, D, MODEL = 8, 2, 64, 512
WIDTH = (H + 2 * HKV) * D
SPEC = dict(layout="half", freq_base=10000.0, scaling="yarn", factor=4.0, original_ctx=64)
SCALE = D ** -0.5


class Layer:
    def __init__(self, be, qkv_fmt, seed, out_fmt="q4_0"):
        rng = np.random.default_rng(seed)
        raw, raw_o = q4.ggml(rng, qkv_fmt, WIDTH, MODEL), q4.ggml(rng, out_fmt, MODEL, H * D)
        self.qkv, self.out = be.create_q4_weights(raw, WIDTH, MODEL, qkv_fmt), be.create_q4_weights(raw_o, MODEL, H * D, out_fmt)
        self.qkv_parts, self.out_parts = q4.parts(raw, qkv_fmt), q4.parts(raw_o, out_fmt)


class Buffers:
    def __init__(self, be, n):
        self.x, self.row, self.q, self.att, self.y = (be.empty(n * w * 4) for w in (MODEL, WIDTH, H * D, H * D, MODEL))


def check_attention(att, q, K, V, past, lens):
    r = 0
    for b, n in enumerate(lens):
        for i in range(n):
            for h in range(H):
                g = h // (H // HKV)
                end = past[b] + i + 1
                assert_close(att[r, h], attention_f64(q[r, h], K[b][:end, g], V[b][:end, g], SCALE), what=f"seq {b} row {i}")
            r += 1


def check_stored(k, want, tol, dtype):
    """An f32 row is the rotated one; a Q8_0 value is half a step of its block's largest / 127 away at most, and that scale is
    rounded to f16."""
    if dtype == "q8":
        most = np.abs(want).reshape(len(want), -1, 32).max(-1)
        tol = np.repeat(most * (0.5 / 127 * (1 + 2.0 ** -10) + 2.0 ** -11) + 2.0 ** -24, 32, 1).reshape(want.shape) + tol
    assert np.all(np.abs(k - want) <= tol)


@pytest.mark.parametrize("fmt", ["q4_0", "q4_k"])
@pytest.mark.parametrize("dtype", ["f32", "q8"])
@pytest.mark.parametrize("paged", [False, True])
def test_prompts_then_single_tokens(backend, fmt, dtype, paged):
    be = backend
    layer = Layer(be, fmt, 5 + paged)
    plan = be.create_rope_plan(D, **SPEC)
    rng = np.random.default_rng(9)
    B, cap = 5, 80
    table = rng.permutation(B * cap // PAGE).astype(np.int32).reshape(B, -1)
    slots = np.array([3, 0, 4, 1, 2], np.int32)
    where, layer_id = {}, 0
    if paged:
        kv = be.create_page_pool(B * cap // PAGE, HKV, D, dtype)
        where = dict(page_table=be.buffer(table), page_table_stride=table.shape[1])
    else:
        kv, layer_id = be.create_kv_cache(2, cap, HKV, D, dtype, B), 1
        where = dict(seq_slot=be.buffer(slots), layer=1)
    past = [0, 0, 0, 0, 0]
    for lens in ([17, 0, 1, 33, 64], [1] * 5, [1] * 5, [4, 16, 15, 1, 3]):
        n = int(sum(lens))
        t = Buffers(be, n)
        x = rng.standard_normal((n, MODEL)).astype(np.float32)
        t.x.upload(x)
        starts = be.buffer(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32))
        offsets = be.buffer(np.array(past, np.int32))
        be.matvec_q4(layer.qkv, t.x, n, t.row)
        be.append(kv, View(t.row, H * D), View(t.row, (H + HKV) * D), starts, offsets, B, max(lens), rope=plan, q=t.row, q_out=t.q,
                  n_heads=H, k_stride=WIDTH, v_stride=WIDTH, q_stride=WIDTH, **where)
        if max(lens) == 1:
            ends = be.buffer(np.array(past, np.int32) + 1)
            be.decode(kv, t.q, t.att, be.buffer(np.zeros(B, np.int32)), ends, B, max(past) + 1, H, SCALE, **where)
        else:
            be.prefill(kv, t.q, t.att, starts, offsets, B, max(lens), H, SCALE, **where)
        be.matvec_q4(layer.out, t.att, n, t.y)
        be.sync()
        row, q, att, y = t.row.download((n, WIDTH)), t.q.download((n, H, D)), t.att.download((n, H, D)), t.y.download((n, MODEL))
        q4.check(row, x, *layer.qkv_parts)
        pos = np.concatenate([np.arange(p, p + m) for p, m in zip(past, lens)])
        want, tol = rope_ref.rotate(row[:, :H * D].reshape(n, H, D), pos, **SPEC)
        assert np.all(np.abs(q - want) <= tol)
        rows = lambda b, a, e: rows_of([e - a], [a], **(dict(table=table[b:b + 1]) if paged else dict(
            seq=slots[b:b + 1], layers=2, layer=layer_id, ppl=cap // PAGE)))
        K, V, r = [], [], 0
        for b, (p, m) in enumerate(zip(past, lens)):
            if p + m == 0:
                K.append(None), V.append(None)
                continue
            k, v = read(be, kv, rows(b, 0, p + m))
            if m:
                new = row[r:r + m, H * D:].reshape(m, 2, HKV, D).astype(np.float64)
                kw, kt = rope_ref.rotate(new[:, 0], pos[r:r + m], **SPEC)
                check_stored(k[p:], kw.reshape(m, -1), kt.reshape(m, -1), dtype)
                check_stored(v[p:], new[:, 1].reshape(m, -1), 0.0, dtype)
            K.append(k.reshape(-1, HKV, D)), V.append(v.reshape(-1, HKV, D))
            r += m
        check_attention(att, q, K, V, past, lens)
        q4.check(y, att.reshape(n, -1), *layer.out_parts)
        past = [p + m for p, m in zip(past, lens)]


@pytest.mark.parametrize("B", [3, 40, 150])
def test_captured_steps_equal_eager_ones(backend, B):
    """One decode step of B sequences as a graph (4-bit products of few, some and many vectors), replayed with new inputs and
    positions, eager steps and a larger product between the replays: rows, caches and outputs equal bit for bit."""
    be = backend
    layer, plan = Layer(be, "q4_k", 3), be.create_rope_plan(D, **SPEC)
    s = HipStream()
    try:
        be.set_stream(s)
        cap = 48
        kv = [be.create_kv_cache(1, cap, HKV, D, "q8", B) for _ in range(2)]
        t = [Buffers(be, 400) for _ in range(2)]
        starts, zeros = be.buffer(np.arange(B + 1, dtype=np.int32)), be.buffer(np.zeros(B, np.int32))
        offsets, ends = be.empty(B * 4), be.empty(B * 4)

        def step(i):
            be.matvec_q4(layer.qkv, t[0].x, B, t[i].row)
            be.append(kv[i], View(t[i].row, H * D), View(t[i].row, (H + HKV) * D), starts, offsets, B, 1, rope=plan, q=t[i].row,
                      q_out=t[i].q, n_heads=H, k_stride=WIDTH, v_stride=WIDTH, q_stride=WIDTH)
            be.decode(kv[i], t[i].q, t[i].att, zeros, ends, B, cap, H, SCALE)
            be.matvec_q4(layer.out, t[i].att, B, t[i].y)

        rng = np.random.default_rng(B)
        at = np.arange(B, dtype=np.int32) % 11

        def inputs():
            t[0].x.upload(rng.standard_normal((B, MODEL)).astype(np.float32))
            offsets.upload(at), ends.upload(at + 1)

        inputs()
        if B > 8:
            with pytest.raises(GlaError, match="sized before capture"):
                be.capture(lambda: be.matvec_q4(layer.qkv, t[0].x, B, t[1].row))
        step(0), step(1)
        be.sync()
        graph = be.capture(lambda: step(1))
        for rep in range(5):
            if rep == 3:  # the eager side takes larger scratch; the graph keeps its own
                be.matvec_q4(layer.qkv, t[0].x, 400, t[0].row)
            at += 1 + (np.arange(B, dtype=np.int32) + rep) % 3
            inputs()
            step(0)
            graph.replay()
            be.sync()
            got = [[getattr(b, k).download((B, w)) for k, w in (("row", WIDTH), ("q", H * D), ("att", H * D), ("y", MODEL))] for b in t]
            for a, b in zip(*got):
                assert np.isfinite(a).all() and np.array_equal(a.view(np.uint32), b.view(np.uint32)), rep
            every = np.arange(B * cap)
            for a, b in zip(read(be, kv[0], every), read(be, kv[1], every)):
                assert np.array_equal(a, b), rep
        graph.destroy()
    finally:
        be.set_stream(None)
        s.destroy()


def test_two_streams_at_once(backend):
    """Products that take scratch and counters, and appends, interleaved on two streams without a wait: the bits of one at a time."""
    be = backend
    layer, plan = Layer(be, "q4_0", 12, "q4_k"), be.create_rope_plan(D, **SPEC)
    rng = np.random.default_rng(13)
    sizes = [40, 300, 64, 129]
    x = [be.buffer(rng.standard_normal((n, MODEL)).astype(np.float32)) for n in sizes]
    zero = be.buffer(np.zeros(1, np.int32))

    def step(i, row, q, kv, starts):
        be.matvec_q4(layer.qkv, x[i], sizes[i], row)
        be.append(kv, View(row, H * D), View(row, (H + HKV) * D), starts, zero, 1, sizes[i], rope=plan, q=row, q_out=q, n_heads=H,
                  k_stride=WIDTH, v_stride=WIDTH, q_stride=WIDTH)

    def sets():
        return [(be.empty(n * WIDTH * 4), be.empty(n * H * D * 4), be.create_kv_cache(1, 304, HKV, D, "q8", 1),
                 be.buffer(np.array([0, n], np.int32))) for n in sizes]

    def results(state):
        return [(row.download((n, WIDTH)), q.download((n, H * D)), *read(be, kv, np.arange(304))) for n, (row, q, kv, _) in zip(sizes, state)]

    one = sets()
    for i in range(len(sizes)):
        step(i, *one[i])
        be.sync()
    want = results(one)
    streams = [HipStream(), HipStream()]
    try:
        for _ in range(3):
            two = sets()
            be.sync()
            for i in range(len(sizes)):
                be.set_stream(streams[i % 2])
                step(i, *two[i])
            for s in streams:
                s.synchronize()
            be.set_stream(None)
            for a, b in zip(want, results(two)):
                for m, g in zip(a, b):
                    assert np.array_equal(m.view(np.uint32), g.view(np.uint32))
    finally:
        be.set_stream(None)
        for s in streams:
            s.destroy()


@pytest.mark.parametrize("fmt, rows, cols, n", [("q4_0", 1027, 4096, 300), ("q4_k", 1027, 4096, 129), ("q4_0", 45, 8192, 65),
                                                ("q4_k", 30, 4096, 128), ("q4_0", 8200, 512, 128), ("q4_k", 4100, 256, 500)])
def test_products_of_odd_rows(backend, fmt, rows, cols, n):
    """Rows that no vector store fits, K in slices and not, tall matrices that leave the middle kernel early; y 4 bytes off."""
    rng = np.random.default_rng(rows + n)
    raw = q4.ggml(rng, fmt, rows, cols)
    w = backend.create_q4_weights(raw, rows, cols, fmt)
    x = rng.standard_normal((n, cols)).astype(np.float32)
    parts = q4.parts(raw, fmt)
    for shift in (0, 1):
        q4.check(q4.run(backend, w, x, shift=shift), x, *parts)


@pytest.mark.parametrize("dtype", ["f32", "q8"])
def test_many_rows_read(backend, dtype):
    """Enough rows that a thread takes four, some of them twice and some no row; the same rows a few at a time."""
    be = backend
    pool = be.create_page_pool(64, 8, 128, dtype)
    rng = np.random.default_rng(14)
    pool.write_rows(np.arange(1024), *(rng.standard_normal((1024, 1024)).astype(np.float32) for _ in range(2)))
    rows = rng.integers(-3, 1030, 9001)
    few = [np.concatenate(t) for t in zip(*(read(be, pool, np.arange(i, i + 128)) for i in range(0, 1024, 128)))]
    n = len(rows)
    k, v = (be.buffer(np.full((n, 1024), 7.5, np.float32)) for _ in range(2))
    pool.read_rows_device(be.buffer(rows.astype(np.int64)), k, v, n)
    be.sync()
    held = (rows >= 0) & (rows < 1024)
    for got, want in zip((k.download((n, 1024)), v.download((n, 1024))), few):
        assert np.array_equal(got[held], want[rows[held]]) and np.all(got[~held] == 7.5)


@pytest.mark.parametrize("dtype", ["f32", "q8"])
def test_very_many_sequences(backend, dtype):
    """More sequences than one dimension of a launch: 70,000 of one row, each a place of its own; one page id is none."""
    be = backend
    B, pages = 70000, 70000 // PAGE + 1
    pool = be.create_page_pool(pages, 1, 64, dtype)
    rng = np.random.default_rng(15)
    k, v = (rng.standard_normal((B, 64)).astype(np.float32) for _ in range(2))
    table = (np.arange(B, dtype=np.int32) // PAGE)[::-1].copy().reshape(B, 1)
    past = (np.arange(B, dtype=np.int32) % PAGE)[::-1].copy()
    table[B // 2] = pages
    be.append(pool, be.buffer(k), be.buffer(v), be.buffer(np.arange(B + 1, dtype=np.int32)), be.buffer(past), B, 1,
              page_table=be.buffer(table), page_table_stride=1)
    be.sync()
    gk, gv = read(be, pool, np.arange(B))
    wk, wv = k[::-1].copy(), v[::-1].copy()
    wk[B - 1 - B // 2] = wv[B - 1 - B // 2] = 0
    check_stored(gk, wk.astype(np.float64), 0.0, dtype), check_stored(gv, wv.astype(np.float64), 0.0, dtype)


@pytest.mark.parametrize("lo", [15, 16, 17])
def test_v_by_row_and_by_page_alike(backend, lo):
    """Prompts about the length at which V goes page by page: the storage's bits are those of write_rows, from any offset."""
    be = backend
    lens, past = [lo, lo - 1, 1, 0, lo], [0, 1, 15, 7, 13]
    rng = np.random.default_rng(lo)
    n = sum(lens)
    k, v = (rng.standard_normal((n, 256)).astype(np.float32) for _ in range(2))
    caches = [be.create_kv_cache(1, 40, 2, 128, "q8", 5) for _ in range(2)]
    be.append(caches[0], be.buffer(k), be.buffer(v), be.buffer(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)),
              be.buffer(np.array(past, np.int32)), 5, lo)
    be.sync()
    caches[1].write_rows(rows_of(lens, past, ppl=3), k, v)
    every = np.arange(5 * 48)
    for a, b in zip(caches[0].export_rows(every), caches[1].export_rows(every)):
        assert np.array_equal(a, b)


def test_too_many_rows_are_refused(backend):
    be = backend
    few, out = np.zeros(18, np.uint8), C.c_void_p()
    for fmt, rows, cols in ((0, (1 << 26) + 1, 32), (0, 1 << 24, 1 << 14), (1, 1 << 14, 1 << 24), (0, 1, (1 << 26) + 32)):
        assert _lib.lib().gla_q4w_create(be.ctx, fmt, few.ctypes.data, rows, cols, C.byref(out)) == _lib.GLA_ERR_INVALID
        assert not out.value
    plan, buf = be.create_rope_plan(4), be.buffer(np.zeros(64, np.float32))
    with pytest.raises(GlaError, match="too many"):
        be.rope_rows(plan, buf, 33554429, 1, buf)


@pytest.mark.parametrize("fmt", ["q4_0", "q4_k"])
@pytest.mark.parametrize("rows, cols, n", [(1027, 2048, 2500), (1028, 2048, 2500), (1027, 512, 8100), (48, 1024, 2000), (1027, 256, 4000)])
def test_products_of_many_vectors_and_odd_rows(backend, fmt, rows, cols, n):
    """Large tiles with K in two slices (rows that a vector store fits and not), in one, and 128 vectors wide; y 4 bytes off."""
    rng = np.random.default_rng(rows + n)
    raw = q4.ggml(rng, fmt, rows, cols)
    w = backend.create_q4_weights(raw, rows, cols, fmt)
    x = rng.standard_normal((n, cols)).astype(np.float32)
    parts = q4.parts(raw, fmt)
    for shift in (0, 1):
        q4.check(q4.run(backend, w, x, shift=shift), x, *parts)


def test_products_of_every_tile(backend):
    """Rows and vectors that take each of the middle kernel's tiles, cut short on both sides."""
    rng = np.random.default_rng(16)
    for fmt, cols in (("q4_0", 96), ("q4_k", 512)):
        for rows, n in ((1000, 33), (6001, 17), (6100, 30), (8100, 32), (6100, 63), (8100, 60), (14000, 61), (14300, 120)):
            raw = q4.ggml(rng, fmt, rows, cols)
            w = backend.create_q4_weights(raw, rows, cols, fmt)
            x = rng.standard_normal((n, cols)).astype(np.float32)
            q4.check(q4.run(backend, w, x, shift=rows // 100 % 2), x, *q4.parts(raw, fmt))


@pytest.mark.parametrize("fmt", ["q4_0", "q4_k"])
def test_slices_of_k_captured_and_on_two_streams(backend, fmt):
    """A product whose workgroups are two slices of K (the last to arrive adds them): a graph replayed between eager calls, and
    two streams at once; every result has the bits of a call by itself, and those are the product's."""
    be = backend
    rows, cols, n = 6144, 2048, 400
    rng = np.random.default_rng(17)
    raw = q4.ggml(rng, fmt, rows, cols)
    w = be.create_q4_weights(raw, rows, cols, fmt)
    xs = [rng.standard_normal((n, cols)).astype(np.float32) for _ in range(3)]
    x = [be.buffer(a) for a in xs]
    y = [be.empty(n * rows * 4) for _ in range(3)]
    want = []
    for i in range(3):
        be.matvec_q4(w, x[i], n, y[i])
        be.sync()
        want.append(y[i].download((n, rows)))
    q4.check(want[0], xs[0], *q4.parts(raw, fmt))
    s = [HipStream(), HipStream()]
    try:
        be.set_stream(s[0])
        inp, out = be.buffer(xs[0]), be.empty(n * rows * 4)
        be.matvec_q4(w, inp, n, y[0])
        be.sync()
        g = be.capture(lambda: be.matvec_q4(w, inp, n, out))
        for rep in range(4):
            inp.upload(xs[rep % 3])
            be.matvec_q4(w, x[2], n, y[2])
            g.replay()
            be.matvec_q4(w, x[1], n, y[1])
            be.sync()
            assert np.array_equal(out.download((n, rows)), want[rep % 3])
            assert np.array_equal(y[1].download((n, rows)), want[1]) and np.array_equal(y[2].download((n, rows)), want[2])
        g.destroy()
        for rep in range(3):
            for i in range(3):
                be.set_stream(s[i % 2])
                be.matvec_q4(w, x[i], n, y[i])
            for t in s:
                t.synchronize()
            be.set_stream(None)
            for i in range(3):
                assert np.array_equal(y[i].download((n, rows)), want[i]), (rep, i)
    finally:
        be.set_stream(None)
        for t in s:
            t.destroy()
