"""gla_block_norm against its formula in 64 bits, within what its roundings can make of it."""
import ctypes as C

import numpy as np
import pytest

from glint_amd import _lib
from glint_amd.attn import HipStream

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # half a step of f32, relative


class View:
    """A device buffer from `floats` on."""

    def __init__(self, buf, floats):
        self.buf, self.ptr = buf, C.c_void_p(buf.ptr.value + 4 * floats)


def formula(x, y, post, gate, scale, pre, eps):
    """x_out, norm_out in 64 bits and how far each may be off. A sum of squares is a chain of at most 16 products a thread,
    6 steps across its wave and 16 waves, all of one sign: 38 U; its half by the root, then mean, eps, root and reciprocal: 24 U
    for the factor. The products with y, scale, gate and weight, and the sum: 5 U of the part and U of the result."""
    x = np.asarray(x, np.float64)
    z = np.zeros_like(x)
    if y is not None:
        z = np.asarray(y, np.float64)
        if post is not None:
            z = z / np.sqrt((z * z).mean(-1, keepdims=True) + eps) * post
        z = scale * (z if gate is None else z * gate)
    s = x + z
    ds = 29 * U * np.abs(z) + U * np.abs(s)
    if pre is None:
        return s, ds, None, None
    r = np.sqrt((s * s).mean(-1, keepdims=True) + eps)
    h = s / r * pre
    # the factor's own 24 U, and what the sum's errors make of it
    rel = 24 * U + np.sqrt((ds * ds).mean(-1, keepdims=True)) / r
    return s, ds, h, np.abs(pre) * ds / r + np.abs(h) * (rel * 1.01 + 2 * U)


def inputs(rng, n, dim, post, gate, mul=1.0):
    f = lambda *shape: (mul * rng.standard_normal(shape)).astype(np.float32)
    return (f(n, dim), f(n, dim), f(dim) if post else None, {None: None, "vector": f(1, dim), "rows": f(n, dim)}[gate], f(dim))


def run(be, x, y, post, gate, scale, pre, eps, tail=1):
    n, dim = x.shape
    out, h = (be.buffer(np.full((n + tail, dim), -9.0, np.float32)) for _ in "xh")
    buf = lambda t: None if t is None else be.buffer(t)
    be.block_norm(be.buffer(x), n, dim, eps, y=buf(y), post=buf(post), gate=buf(gate),
                  gate_stride=dim if gate is not None and len(gate) > 1 else 0, scale=scale, x_out=out, pre=buf(pre),
                  norm_out=h if pre is not None else None)
    be.sync()
    out, h = out.download((n + tail, dim)), h.download((n + tail, dim))
    assert np.all(out[n:] == -9.0) and np.all(h[n:] == -9.0), "rows behind the last"
    return out[:n], h[:n]


def check(got, want, tol):
    assert np.all(np.abs(got.astype(np.float64) - want) <= tol), float((np.abs(got - want) / np.maximum(tol, 1e-300)).max())


DIMS = [1, 2, 3, 4, 31, 63, 64, 65, 255, 256, 257, 260, 576, 1000, 1023, 1024, 1025, 1028, 3584, 4095, 4096, 4097, 4100, 8192, 16383,
        16384]


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("post, gate", [(False, None), (True, None), (True, "vector"), (False, "rows"), (True, "rows")])
def test_the_formula(backend, dim, post, gate):
    rng = np.random.default_rng(dim)
    for n in (1, 2, 5, 9):
        x, y, w, g, pre = inputs(rng, n, dim, post, gate)
        if n == 1 and gate == "rows":
            continue
        out, h = run(backend, x, y, w, g, 0.75, pre, 1e-5)
        s, ds, hn, dh = formula(x, y, w, g, 0.75, pre, 1e-5)
        check(out, s, ds)
        check(h, hn, dh)


@pytest.mark.parametrize("dim", [576, 577, 4096])
def test_many_rows(backend, dim):
    rng = np.random.default_rng(1)
    x, y, w, g, pre = inputs(rng, 1999, dim, True, "rows")
    out, h = run(backend, x, y, w, g, 1.0, pre, 1e-6)
    s, ds, hn, dh = formula(x, y, w, g, 1.0, pre, 1e-6)
    check(out, s, ds)
    check(h, hn, dh)


def test_the_parts_alone(backend):
    """Only a norm, only a sum, only a normed sum."""
    be, rng = backend, np.random.default_rng(2)
    for dim in (64, 100, 2050):
        x, y, w, _, pre = inputs(rng, 7, dim, True, None)
        h = be.empty(x.nbytes)
        be.block_norm(be.buffer(x), 7, dim, 1e-6, pre=be.buffer(pre), norm_out=h)
        be.sync()
        _, _, want, tol = formula(x, None, None, None, 1.0, pre, 1e-6)
        check(h.download(x.shape), want, tol)
        out, _ = run(be, x, y, None, None, -2.0, None, 0.0)
        check(out, *formula(x, y, None, None, -2.0, None, 0.0)[:2])
        be.block_norm(be.buffer(x), 7, dim, 1e-6, y=be.buffer(y), post=be.buffer(w), pre=be.buffer(pre), norm_out=h)
        be.sync()
        check(h.download(x.shape), *formula(x, y, w, None, 1.0, pre, 1e-6)[2:])


def test_in_place_strides_and_columns(backend):
    """The stream kept in place, the norm over the block's output, both as columns of one wider row, odd addresses."""
    be, rng = backend, np.random.default_rng(3)
    for dim, width, ox, oy in ((64, 136, 0, 68), (65, 137, 1, 70), (576, 1200, 4, 600), (4096, 8200, 2, 4099), (4096, 8200, 4, 4104)):
        n = 6
        row = rng.standard_normal((n, width)).astype(np.float32)
        _, _, w, g, pre = inputs(rng, n, dim, True, "vector")
        x, y = row[:, ox:ox + dim].copy(), row[:, oy:oy + dim].copy()
        buf = be.buffer(row)
        bx, by = View(buf, ox), View(buf, oy)
        be.block_norm(bx, n, dim, 1e-6, y=by, post=be.buffer(w), gate=be.buffer(g), x_out=bx, pre=be.buffer(pre), norm_out=by,
                      x_stride=width, y_stride=width, x_out_stride=width, norm_out_stride=width)
        be.sync()
        got = buf.download(row.shape)
        s, ds, hn, dh = formula(x, y, w, g, 1.0, pre, 1e-6)
        check(got[:, ox:ox + dim], s, ds)
        check(got[:, oy:oy + dim], hn, dh)
        rest = np.ones(width, bool)
        rest[ox:ox + dim] = rest[oy:oy + dim] = False
        assert np.array_equal(got[:, rest], row[:, rest])
        # the gate's rows taken by the norm
        gates = be.buffer(rng.standard_normal((n, dim)).astype(np.float32))
        gv = gates.download((n, dim))
        be.block_norm(be.buffer(x), n, dim, 1e-6, y=be.buffer(y), gate=gates, gate_stride=dim, pre=be.buffer(pre), norm_out=gates)
        be.sync()
        check(gates.download((n, dim)), *formula(x, y, None, gv, 1.0, pre, 1e-6)[2:])


def test_magnitudes(backend):
    """Rows of large and small values side by side; zeros under eps."""
    rng = np.random.default_rng(4)
    x, y, w, g, pre = inputs(rng, 8, 1000, True, "rows")
    for r, m in enumerate((1e15, 1e-15, 1.0, 1e8, 0.0, 1e-3, 1e4, 1.0)):
        x[r] *= np.float32(m)
        y[r] *= np.float32(m)
    x[4] = 0
    out, h = run(backend, x, y, w, g, 1.0, pre, 1e-6)
    s, ds, hn, dh = formula(x, y, w, g, 1.0, pre, 1e-6)
    check(out, s, ds)
    check(h, hn, dh)
    assert np.all(out[4] == 0) and np.all(h[4] == 0)


@pytest.mark.parametrize("dim", [64, 300, 4096])
def test_non_finite_rows_stay_alone(backend, dim):
    rng = np.random.default_rng(5)
    x, y, w, g, pre = inputs(rng, 9, dim, True, "rows")
    clean = run(backend, x, y, w, g, 1.0, pre, 1e-6)
    y[2, 1], x[5, 3], y[7, 0] = np.nan, np.inf, np.inf
    got = run(backend, x, y, w, g, 1.0, pre, 1e-6)
    keep = [0, 1, 3, 4, 6, 8]
    for a, b in zip(clean, got):
        assert np.array_equal(a[keep], b[keep])
    assert np.isnan(got[0][2]).all() and np.isnan(got[1][2]).all()
    assert got[0][5, 3] == np.inf and np.isfinite(np.delete(got[0][5], 3)).all()
    assert np.isnan(got[1][5, 3]) and np.all(np.delete(got[1][5], 3) == 0)


def test_captured_and_on_two_streams(backend):
    be, rng = backend, np.random.default_rng(6)
    x, y, w, g, pre = inputs(rng, 33, 577, True, "vector")
    bufs = [be.buffer(t) for t in (x, y, w, g, pre)]
    outs = [(be.empty(x.nbytes), be.empty(x.nbytes)) for _ in range(3)]

    def call(o):
        be.block_norm(bufs[0], 33, 577, 1e-6, y=bufs[1], post=bufs[2], gate=bufs[3], x_out=o[0], pre=bufs[4], norm_out=o[1])

    graph = be.capture(lambda: call(outs[1]))
    other = HipStream()
    for _ in range(3):
        bufs[0].upload(rng.standard_normal(x.shape).astype(np.float32))
        graph.replay()
        be.set_stream(other)
        call(outs[2])
        be.sync()
        be.set_stream(None)
        call(outs[0])
        be.sync()
        for i in range(2):
            a = [o[i].download(x.shape).view(np.uint32) for o in outs]
            assert np.array_equal(a[0], a[1]) and np.array_equal(a[0], a[2])
    graph.destroy()
    other.destroy()


def test_refusals(backend):
    be = backend
    t, v = be.empty(4 * 4 * 200), be.empty(4 * 200)
    o = be.empty(4 * 4 * 200)
    ok = dict(x=t, n_rows=4, dim=100, eps=1e-6, x_out=o)
    be.block_norm(**ok)
    be.block_norm(**{**ok, "n_rows": 0})
    for bad in (dict(n_rows=-1), dict(dim=0), dict(dim=_lib.GLA_BLOCK_NORM_MAX_DIM + 1), dict(eps=-1.0), dict(eps=float("nan")),
                dict(eps=float("inf")), dict(x_out=None), dict(post=v), dict(gate=v), dict(pre=v), dict(norm_out=t), dict(x_stride=99),
                dict(x_out_stride=-100), dict(y=t, gate=t, gate_stride=50), dict(y=t, gate=t, gate_stride=-1),
                dict(x_out=View(t, 1)), dict(x_out=t, x_stride=200), dict(x_out=View(t, 100), x_stride=150, x_out_stride=150),
                dict(y=t, x=o, x_out=View(t, 4)), dict(pre=v, norm_out=o), dict(pre=v, norm_out=View(o, 100)),
                dict(pre=v, norm_out=v), dict(y=t, post=v, x_out=View(v, 50)), dict(y=t, gate=v, x_out=v), dict(x=None)):
        with pytest.raises(_lib.GlaError) as e:
            args = {**ok, **bad}
            if args["x"] is None:
                args["x"] = type("Null", (), {"ptr": None})()
            be.block_norm(**args)
        assert e.value.code == _lib.GLA_ERR_INVALID, bad
    be.block_norm(**{**ok, "x_out": View(t, 100), "x_stride": 200, "x_out_stride": 200})
    be.sync()


@pytest.mark.parametrize("n, dim, gate", [(90000, 256, None), (22000, 1000, "rows"), (4100, 5000, "vector")])
def test_more_than_the_caches_hold(backend, n, dim, gate):
    """Inputs that are read past the caches (more than 256 MB of rows), in every width's variant."""
    rng = np.random.default_rng(31)
    x, y, post, g, pre = inputs(rng, n, dim, True, gate)
    out, h = run(backend, x, y, post, g, 0.5, pre, 1e-5)
    at = np.concatenate([np.arange(50), rng.integers(0, n, 400), np.arange(n - 50, n)])
    want, dx, norm, dh = formula(x[at], y[at], post, g if gate != "rows" else g[at], 0.5, pre, 1e-5)
    assert np.all(np.abs(out[at] - want) <= dx) and np.all(np.abs(h[at] - norm) <= dh)


def test_more_rows_than_a_launch_takes(backend):
    rng = np.random.default_rng(32)
    n, dim = 4 * 2 ** 21 + 5, 4
    x, y, _, _, pre = inputs(rng, n, dim, False, None)
    out, h = run(backend, x, y, None, None, 1.0, pre, 1e-5)
    want, dx, norm, dh = formula(x, y, None, None, 1.0, pre, 1e-5)
    assert np.all(np.abs(out - want) <= dx) and np.all(np.abs(h - norm) <= dh)
