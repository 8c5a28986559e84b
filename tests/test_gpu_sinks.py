"""Windows with sinks: decode and prefill against 64-bit attention over the positions that each row sees."""
import numpy as np
import pytest

from glint_amd import _lib
from glint_amd.attn import HipStream
from helpers import BF16_ABS_TOL, BF16_REL_TOL, assert_close
from seen_ref import Batch, seen

pytestmark = pytest.mark.gpu

SHAPES = [(9, 3, 64), (32, 8, 128), (16, 8, 256), (5, 1, 128), (7, 7, 64)]


def decode(b, q, start, length, sinks, scale, cap=None, host=True, bound=None):
    be, n = b.be, len(q)
    out = be.buffer(np.full(q.shape, -7.0, np.float32))
    kw = dict(b.where)
    start, length = np.asarray(start, np.int32), np.asarray(length, np.int32)
    if host:
        kw.update(kv_start_host=start, kv_len_host=length)
    be.decode(b.kv, be.buffer(q), out, be.buffer(start), be.buffer(length), n, int(length.max()) if bound is None else bound,
              q.shape[1], scale, cap, n_sinks=sinks, **kw)
    be.sync()
    return out.download(q.shape)


def prefill(b, q, q_start, past, window, sinks, scale, cap=None, precision="f32"):
    be = b.be
    out = be.buffer(np.full((len(q) + 3,) + q.shape[1:], -7.0, np.float32))
    be.prefill(b.kv, be.buffer(q), out, be.buffer(np.asarray(q_start, np.int32)), be.buffer(np.asarray(past, np.int32)),
               len(past), int(np.diff(q_start).max()), q.shape[1], scale, cap, window, precision=precision, n_sinks=sinks, **b.where)
    be.sync()
    got = out.download((len(q) + 3,) + q.shape[1:])
    assert np.all(got[len(q):] == -7.0), "rows behind the last sequence"
    return got[:len(q)]


def want_prefill(b, q, q_start, past, window, sinks, scale, cap=None, rows=None):
    want = np.zeros(q.shape)
    for s, p0 in enumerate(past):
        for r in range(q_start[s], q_start[s + 1]):
            if rows is not None and r not in rows:
                continue
            p = p0 + r - q_start[s]
            want[r] = b.attend(s, q[r], seen(max(0, p - window + 1) if window else 0, p + 1, sinks), scale, cap)
    return want


# windows that end everywhere about the sinks' pages: behind them, meeting them, inside them, from the first position
STARTS_ENDS = [(0, 1), (0, 40), (1, 17), (3, 30), (4, 5), (15, 33), (16, 17), (17, 200), (47, 64), (64, 65), (100, 131), (256, 700),
               (701, 702), (500, 500)]


@pytest.mark.parametrize("paged", [True, False])
@pytest.mark.parametrize("dtype", ["f32", "q8"])
@pytest.mark.parametrize("H, n_kv, d", SHAPES)
@pytest.mark.parametrize("sinks", [1, 4, 16, 17, 33, 100, 100000])
def test_decode(backend, H, n_kv, d, dtype, paged, sinks):
    rng = np.random.default_rng(d + H + sinks)
    start, end = np.array(STARTS_ENDS).T
    b = Batch(backend, rng, dtype, paged, end, n_kv, d)
    q = rng.standard_normal((len(end), H, d)).astype(np.float32)
    cap = 30.0 if sinks == 16 else None
    got = decode(b, q, start, end - start, sinks, d ** -0.5, cap)
    want = np.stack([b.attend(i, q[i], seen(s, e, sinks), d ** -0.5, cap) for i, (s, e) in enumerate(zip(start, end))])
    assert_close(got, want)
    assert np.all(got[-1] == 0), "an empty window sees nothing"
    # sized by the bounds alone: the same bits
    assert np.array_equal(decode(b, q, start, end - start, sinks, d ** -0.5, cap, host=False).view(np.uint32), got.view(np.uint32))


@pytest.mark.parametrize("dtype", ["f32", "q8"])
@pytest.mark.parametrize("H, n_kv, d", SHAPES[:3])
def test_decode_long_windows(backend, H, n_kv, d, dtype):
    """Windows of many splits, merged by the last workgroup or by the second kernel, each row alone as in its batch."""
    rng = np.random.default_rng(7 * d)
    end = np.array([5000, 1025, 4096, 2900, 131])
    start = end - np.array([4096, 700, 1000, 2000, 100])
    b = Batch(backend, rng, dtype, True, end, n_kv, d)
    q = rng.standard_normal((len(end), H, d)).astype(np.float32)
    for sinks in (5, 512):
        got = decode(b, q, start, end - start, sinks, d ** -0.5)
        want = np.stack([b.attend(i, q[i], seen(s, e, sinks), d ** -0.5) for i, (s, e) in enumerate(zip(start, end))])
        assert_close(got, want)
        for i in (0, 4):
            one = Rows(b, i)
            alone = decode(one, q[i:i + 1], start[i:i + 1], (end - start)[i:i + 1], sinks, d ** -0.5)
            assert np.array_equal(alone[0].view(np.uint32), got[i].view(np.uint32))


class Rows:
    """One sequence of a paged Batch as a batch of its own."""

    def __init__(self, b, i):
        self.be, self.kv = b.be, b.kv
        self.where = {"page_table": b.be.buffer(b.table[i:i + 1]), "page_table_stride": b.table.shape[1]}


@pytest.mark.parametrize("dtype", ["f32", "q8"])
def test_without_sinks_or_a_window_it_is_decode(backend, dtype):
    rng = np.random.default_rng(3)
    end = np.array([1500, 40, 700])
    b = Batch(backend, rng, dtype, True, end, 2, 128)
    q = rng.standard_normal((3, 8, 128)).astype(np.float32)
    be, out = backend, backend.empty(q.nbytes)
    for start in (end * 0, end - 30):
        plain = decode(b, q, start, end - start, 0, 0.1)
        a = _lib.DecodeArgs()
        ds, dl, dq = be.buffer(start.astype(np.int32)), be.buffer((end - start).astype(np.int32)), be.buffer(q)
        a.kv, a.n_seqs, a.page_table, a.page_table_stride = b.kv.handle, 3, b.where["page_table"].ptr, b.where["page_table_stride"]
        a.kv_start, a.kv_len, a.max_kv_len, a.n_heads, a.scale = ds.ptr, dl.ptr, int((end - start).max()), 8, 0.1
        a.q, a.out = dq.ptr, out.ptr
        _lib.check(_lib.lib().gla_decode_sinks(be.ctx, a, 0))
        be.sync()
        assert np.array_equal(out.download(q.shape).view(np.uint32), plain.view(np.uint32))
    assert np.array_equal(decode(b, q, end * 0, end, 50, 0.1).view(np.uint32), decode(b, q, end * 0, end, 0, 0.1).view(np.uint32))


@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("dtype", ["f32", "q8"])
def test_decode_leaves_what_it_does_not_see(backend, dtype, bad):
    """Positions between the sinks and the window, behind the end and on other pages hold what must not count."""
    rng = np.random.default_rng(11)
    start, end, sinks = [9, 60, 200, 640], [30, 90, 333, 801], 5

    def fill(b):
        keep = np.concatenate([b.at(i, seen(s, e, sinks)) for i, (s, e) in enumerate(zip(start, end))])
        gone = np.setdiff1d(np.arange(len(b.k)), keep)
        b.k[gone], b.v[gone] = bad, bad

    b = Batch(backend, rng, dtype, True, end, 2, 64, fill=fill)
    q = rng.standard_normal((4, 8, 64)).astype(np.float32)
    got = decode(b, q, start, np.subtract(end, start), sinks, 0.125)
    assert_close(got, np.stack([b.attend(i, q[i], seen(s, e, sinks), 0.125) for i, (s, e) in enumerate(zip(start, end))]))


# (rows, position of the first, window): windows below, at and above a tile, rows that see the sinks' tiles and the window's
CHUNKS = [([40], [700], 256), ([1, 70, 33], [0, 5, 1000], 7), ([200], [0], 50), ([130, 3], [31, 64], 32), ([300, 0, 17], [0, 9, 470], 100),
          ([5], [3], 1), ([97], [2000], 1500)]


@pytest.mark.parametrize("rows, past, window", CHUNKS, ids=str)
@pytest.mark.parametrize("dtype", ["f32", "q8"])
@pytest.mark.parametrize("H, n_kv, d", SHAPES[:4])
@pytest.mark.parametrize("sinks", [1, 4, 33, 64])
def test_prefill(backend, H, n_kv, d, dtype, sinks, rows, past, window):
    rng = np.random.default_rng(d + H + sinks)
    paged = (sinks + len(rows)) % 2 == 0
    b = Batch(backend, rng, dtype, paged, [p + n for p, n in zip(past, rows)], n_kv, d)
    q_start = np.concatenate([[0], np.cumsum(rows)])
    q = rng.standard_normal((q_start[-1], H, d)).astype(np.float32)
    cap = 30.0 if sinks == 33 else None
    check = None if q_start[-1] <= 60 else set(rng.choice(q_start[-1], 40, replace=False).tolist()) | {0, int(q_start[-1]) - 1}
    pick = sorted(check) if check is not None else slice(None)
    want = want_prefill(b, q, q_start, past, window, sinks, d ** -0.5, cap, check)[pick]
    assert_close(prefill(b, q, q_start, past, window, sinks, d ** -0.5, cap)[pick], want)
    assert_close(prefill(b, q, q_start, past, window, sinks, d ** -0.5, cap, "bf16")[pick], want, BF16_ABS_TOL, BF16_REL_TOL)


@pytest.mark.parametrize("dtype", ["f32", "q8"])
def test_prefill_bf16_without_scratch(backend, dtype, monkeypatch):
    """Workgroups that convert their own tiles give the staged kernel's result."""
    rng = np.random.default_rng(5)
    b = Batch(backend, rng, dtype, True, [330, 90], 2, 128)
    q_start, past = [0, 130, 180], [200, 40]
    q = rng.standard_normal((180, 8, 128)).astype(np.float32)
    want = want_prefill(b, q, q_start, past, 60, 9, 0.09, None, set(range(0, 180, 7)))
    monkeypatch.setenv("GLA_BF16_UNSTAGED", "1")
    got = prefill(b, q, q_start, past, 60, 9, 0.09, None, "bf16")
    assert_close(got[::7], want[::7], BF16_ABS_TOL, BF16_REL_TOL)


@pytest.mark.parametrize("dtype", ["f32", "q8"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_prefill_rows_of_unlike_keys(backend, dtype, d):
    """Keys whose magnitudes differ by many binades, by tile and by key, infinities among V's values: a row's result is
    that of the positions it sees, and a row gives the same bits in any chunk."""
    rng = np.random.default_rng(21)
    window, sinks, n, past = 70, 6, 150, 200
    inf_at = 230

    def fill(b):
        at = b.at(0, np.arange(350))
        b.v[at] *= (2.0 ** rng.integers(-12, 12, (350, 1))).astype(np.float32)
        b.v[at[:6]] *= np.float32(2.0 ** 14)
        b.k[at[100:140]] *= np.float32(2.0 ** -10)
        b.v[at[inf_at], 3] = np.inf
        if dtype == "f32":
            b.v[at[260], 1], b.k[at[270], :8] = 1e-38, 1e-20

    b = Batch(backend, rng, dtype, True, [past + n], 1, d, fill=fill)
    q = rng.standard_normal((n, 2, d)).astype(np.float32)
    got = prefill(b, q, [0, n], [past], window, sinks, d ** -0.5)
    for r in range(0, n, 3):
        p = past + r
        pos = seen(p - window + 1, p + 1, sinks)
        with np.errstate(invalid="ignore"):
            want = b.attend(0, q[r], pos, d ** -0.5)
        ok = np.isfinite(want)
        if dtype == "f32":
            assert np.array_equal(np.isinf(want[:, 3]), [inf_at in pos] * 2)
            assert np.array_equal(np.isinf(got[r, :, 3]), np.isinf(want[:, 3]))
        # the values span 2^14: rounding counts against the largest that a row sees
        top = np.abs(np.where(np.isfinite(b.v[b.at(0, pos)]), b.v[b.at(0, pos)], 0)).max()
        assert np.all(np.abs(got[r] - want)[ok] <= 1e-4 * max(top, 1.0))
    for r in (0, 31, 77, 149):
        alone = prefill(b, q[r:r + 1], [0, 1], [past + r], window, sinks, d ** -0.5)
        assert np.array_equal(alone[0].view(np.uint32), got[r].view(np.uint32)), r


@pytest.mark.parametrize("precision", ["f32", "bf16"])
@pytest.mark.parametrize("dtype", ["f32", "q8"])
def test_prefill_leaves_what_it_does_not_see(backend, dtype, precision):
    rng = np.random.default_rng(12)
    window, sinks, past, n = 40, 3, 300, 70

    def fill(b):
        keep = b.at(0, np.concatenate([np.arange(sinks), np.arange(past - window + 1, past + n)]))
        gone = np.setdiff1d(np.arange(len(b.k)), keep)
        b.k[gone], b.v[gone] = np.nan, np.inf

    b = Batch(backend, rng, dtype, True, [past + n], 2, 64, fill=fill)
    q = rng.standard_normal((n, 4, 64)).astype(np.float32)
    want = want_prefill(b, q, [0, n], [past], window, sinks, 0.125)
    tol = (BF16_ABS_TOL, BF16_REL_TOL) if precision == "bf16" else (1e-4, 1e-3)
    assert_close(prefill(b, q, [0, n], [past], window, sinks, 0.125, None, precision), want, *tol)


def test_prefill_without_sinks_or_a_window_is_prefill(backend):
    rng = np.random.default_rng(3)
    b = Batch(backend, rng, "f32", True, [200, 90], 2, 128)
    q, q_start, past = rng.standard_normal((150, 8, 128)).astype(np.float32), [0, 100, 150], [100, 40]
    for window, sinks in ((30, 0), (0, 7)):
        for precision in ("f32", "bf16"):
            be, out = backend, backend.empty(q.nbytes)
            a = _lib.PrefillArgs()
            bufs = be.buffer(np.asarray(q_start, np.int32)), be.buffer(np.asarray(past, np.int32)), be.buffer(q)
            a.kv, a.n_seqs, a.page_table, a.page_table_stride = b.kv.handle, 2, b.where["page_table"].ptr, b.where["page_table_stride"]
            a.q_start, a.pos_offset, a.max_q_len, a.n_heads, a.scale = bufs[0].ptr, bufs[1].ptr, 100, 8, 0.1
            a.sliding_window, a.q, a.out = window, bufs[2].ptr, out.ptr
            a.precision = _lib.GLA_PREC_BF16 if precision == "bf16" else _lib.GLA_PREC_F32
            _lib.check(_lib.lib().gla_prefill_sinks(be.ctx, a, sinks))
            be.sync()
            plain = prefill(b, q, q_start, past, window, 0, 0.1, None, precision)
            assert np.array_equal(out.download(q.shape).view(np.uint32), plain.view(np.uint32))


@pytest.mark.parametrize("dtype", ["f32", "q8"])
def test_captured_replayed_and_on_another_stream(backend, dtype):
    """A step's two calls in a graph, replayed as the window moves on, beside the same calls on another stream."""
    be, rng = backend, np.random.default_rng(8)
    window, sinks, n, rows = 64, 5, 3, 20
    b = Batch(be, rng, dtype, True, [400] * n, 2, 128)
    q = be.buffer(rng.standard_normal((n, 8, 128)).astype(np.float32))
    qp = be.buffer(rng.standard_normal((n * rows, 8, 128)).astype(np.float32))
    starts = be.buffer(np.arange(0, n * rows + 1, rows).astype(np.int32))
    start, length, past = be.empty(4 * n), be.empty(4 * n), be.empty(4 * n)
    outs = [(be.empty(q.nbytes), be.empty(qp.nbytes)) for _ in range(3)]

    def at(end):
        start.upload(np.maximum(end - window, 0).astype(np.int32))
        length.upload(np.minimum(end, window).astype(np.int32))
        past.upload((end - rows).astype(np.int32))

    def step(out):
        be.decode(b.kv, q, out[0], start, length, n, window, 8, 0.1, n_sinks=sinks, **b.where)
        be.prefill(b.kv, qp, out[1], starts, past, n, rows, 8, 0.1, None, window, n_sinks=sinks, **b.where)

    at(np.array([50, 70, 300]))
    step(outs[0])
    graph = be.capture(lambda: step(outs[1]))
    other = HipStream()
    for move in (0, 7, 40, 100):
        at(np.array([50, 70, 300]) + move)
        graph.replay()
        be.sync()
        step(outs[0])
        be.sync()
        be.set_stream(other)
        step(outs[2])
        be.sync()
        be.set_stream(None)
        for i, shape in enumerate(((n, 8, 128), (n * rows, 8, 128))):
            a = [o[i].download(shape).view(np.uint32) for o in outs]
            assert np.array_equal(a[0], a[1]) and np.array_equal(a[0], a[2])
    graph.destroy()
    other.destroy()


def test_refusals(backend):
    rng = np.random.default_rng(0)
    b = Batch(backend, rng, "f32", True, [100], 2, 64)
    q = rng.standard_normal((1, 4, 64)).astype(np.float32)
    with pytest.raises(_lib.GlaError, match="n_sinks"):
        decode(b, q, [50], [50], -1, 0.1)
    with pytest.raises(_lib.GlaError, match="n_sinks"):
        prefill(b, q, [0, 1], [50], 10, -1, 0.1)
    with pytest.raises(_lib.GlaError, match="longer than"):
        decode(b, q, [50], [50], 4, 0.1, bound=40)
    with pytest.raises(ValueError, match="noalloc"):
        backend.decode(b.kv, None, None, None, None, 1, 1, 4, 0.1, noalloc=True, n_sinks=1)
    assert_close(decode(b, q, [50], [50], 4, 0.1), b.attend(0, q[0], seen(50, 100, 4), 0.1)[None])


def test_lengths_and_starts_past_the_storage_are_clamped(backend):
    """Device values that the host does not see: attention over what the storage has of them, and nothing outside."""
    rng = np.random.default_rng(2)
    for dtype in ("f32", "q8"):
        b = Batch(backend, rng, dtype, False, [100, 100, 100, 100], 2, 64)
        q = rng.standard_normal((4, 4, 64)).astype(np.float32)
        top = b.limit
        start, length = [-5, 90, 2 ** 31 - 1, 60], [40, 2 ** 31 - 1, 2 ** 31 - 1, -3]
        got = decode(b, q, start, length, 8, 0.1, host=False, bound=top)
        assert_close(got[0], b.attend(0, q[0], seen(0, 40, 8), 0.1))
        assert_close(got[1], b.attend(1, q[1], seen(90, top, 8), 0.1))
        assert np.all(got[2:] == 0)
