"""gla_matvec_q4 against the product of the dequantised rows in 64 bits."""
import ctypes as C

import numpy as np
import pytest

from glint_amd import _lib

pytestmark = pytest.mark.gpu


def ggml(rng, fmt, rows, cols):
    """Random blocks of the format with ordinary scales, the nibbles and 6-bit fields over their whole range."""
    if fmt == "q4_0":
        raw = rng.integers(0, 256, (rows, cols // 32, 18), dtype=np.uint8)
        raw[..., :2] = (rng.standard_normal((rows, cols // 32, 1)) * 0.02).astype(np.float16).view(np.uint8)
        return raw
    raw = rng.integers(0, 256, (rows, cols // 256, 144), dtype=np.uint8)
    raw[..., :4] = (np.abs(rng.standard_normal((rows, cols // 256, 2))) * [5e-4, 4e-3]).astype(np.float16).view(np.uint8)
    return raw


def parts(raw, fmt):
    """(d * q, minimum) of every value, f64 [rows][cols]; the weight is their difference."""
    rows = raw.shape[0]
    if fmt == "q4_0":
        d = raw[..., :2].copy().view(np.float16).astype(np.float64)
        q = np.concatenate([raw[..., 2:] & 15, raw[..., 2:] >> 4], -1).astype(np.float64) - 8
        w = (q * d).reshape(rows, -1)
        return w, np.zeros_like(w)
    d, dmin = (raw[..., i:i + 2].copy().view(np.float16).astype(np.float64) for i in (0, 2))
    b = raw[..., 4:16].astype(int)
    sc = np.concatenate([b[..., :4] & 63, (b[..., 8:] & 15) | (b[..., :4] >> 6 << 4)], -1)
    mn = np.concatenate([b[..., 4:8] & 63, (b[..., 8:] >> 4) | (b[..., 4:8] >> 6 << 4)], -1)
    qs = raw[..., 16:].reshape(*raw.shape[:2], 4, 1, 32)
    q = np.concatenate([qs & 15, qs >> 4], -2).reshape(*raw.shape[:2], 8, 32).astype(np.float64)
    return ((d * sc)[..., None] * q).reshape(rows, -1), np.repeat((dmin * mn)[..., None], 32, -1).reshape(rows, -1)


def run(be, w, x, shift=0):
    n, rows = len(x), w.rows
    bx = be.buffer(np.concatenate([np.zeros(shift, np.float32), np.asarray(x, np.float32).reshape(-1)]))
    by = be.buffer(np.full(shift + n * rows + 8, -3.5, np.float32))

    class At:
        def __init__(self, b):
            self.ptr = C.c_void_p(b.ptr.value + 4 * shift)

    be.matvec_q4(w, At(bx), n, At(by))
    be.sync()
    got = by.download(shift + n * rows + 8)
    assert np.all(got[:shift] == -3.5) and np.all(got[shift + n * rows:] == -3.5)
    return got[shift:shift + n * rows].reshape(n, rows)


def check(got, x, wd, wm):
    """Each output is a sum of cols products. x enters exactly or as two f16 pieces of a scaled value (2^-22 of the slice's
    largest |x| at most), a product or a group's sum is rounded to f32, and so is each of the cols / 32 + 64 additions
    (the longest chain: a group after the other, 32 products in a group, the slices and waves): every rounding is half a
    step of at most the sum of the magnitudes. As the roundings are of either sign, the error over all outputs is that
    bound's by the root of the number of additions: a lost piece (2^-12) would be far outside it."""
    x = np.asarray(x, np.float64)
    want = x @ (wd - wm).T
    size = np.abs(x) @ (np.abs(wd) + wm).T + np.abs(x).max(1, keepdims=True) * (np.abs(wd) + wm).sum(1)[None] * 2.0 ** -2
    steps = wd.shape[1] / 32 + 64
    err = np.abs(got - want)
    assert np.all(err <= size * (2.0 ** -22 + steps * 2.0 ** -24)), (err / size).max()
    rms = np.sqrt(np.mean((err / np.maximum(size, 1e-300)) ** 2))
    assert rms <= 2.0 ** -24 * np.sqrt(steps) + 2.0 ** -23, rms


SHAPES = [("q4_0", 16, 32), ("q4_0", 1, 96), ("q4_0", 47, 160), ("q4_0", 130, 576), ("q4_0", 96, 4128), ("q4_0", 33, 16384),
          ("q4_k", 16, 256), ("q4_k", 1, 512), ("q4_k", 77, 768), ("q4_k", 300, 4096), ("q4_k", 17, 16640)]


@pytest.mark.parametrize("fmt, rows, cols", SHAPES)
def test_matches_64_bits(backend, fmt, rows, cols):
    rng = np.random.default_rng(rows * 7 + cols)
    raw = ggml(rng, fmt, rows, cols)
    w = backend.create_q4_weights(raw, rows, cols, fmt)
    wd, wm = parts(raw, fmt)
    for n in (1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 33, 48, 64, 65, 100, 130):
        x = rng.standard_normal((n, cols)).astype(np.float32)
        check(run(backend, w, x, shift=n % 2), x, wd, wm)


@pytest.mark.parametrize("fmt, rows, cols, n", [("q4_0", 6144, 4096, 1), ("q4_k", 6144, 4096, 3), ("q4_k", 4096, 4096, 64),
                                                ("q4_0", 4096, 4096, 40), ("q4_0", 6144, 4096, 300), ("q4_k", 1024, 4096, 997),
                                                ("q4_k", 8192, 3584, 130), ("q4_0", 576, 576, 2048), ("q4_0", 960, 576, 7)])
def test_projection_sizes(backend, fmt, rows, cols, n):
    rng = np.random.default_rng(rows + cols + n)
    raw = ggml(rng, fmt, rows, cols)
    w = backend.create_q4_weights(raw, rows, cols, fmt)
    wd, wm = parts(raw, fmt)
    x = rng.standard_normal((n, cols)).astype(np.float32)
    check(run(backend, w, x), x, wd, wm)


@pytest.mark.parametrize("fmt, cols", [("q4_0", 96), ("q4_k", 512)])
def test_every_nibble_scale_and_minimum_counts_once(backend, fmt, cols):
    """Unit vectors read the matrix back, value by value: sums of one term, rounded once or twice."""
    rows = 20
    raw = ggml(np.random.default_rng(cols), fmt, rows, cols)
    w = backend.create_q4_weights(raw, rows, cols, fmt)
    wd, wm = parts(raw, fmt)
    for n in (cols, 1, 6):  # all at once; a few at a time
        cs = np.arange(cols) if n == cols else np.arange(n) * 37 % cols
        got = run(backend, w, np.eye(cols, dtype=np.float32)[cs])
        assert np.all(np.abs(got - (wd - wm).T[cs]) <= 3 * 2.0 ** -24 * (np.abs(wd) + wm).T[cs])


@pytest.mark.parametrize("fmt", ["q4_0", "q4_k"])
def test_magnitudes_far_apart(backend, fmt):
    """Vectors of other magnitudes in one call do not disturb each other: 1e-20 beside 1e20, and wide ranges within a row."""
    rows, cols = 40, 1024
    rng = np.random.default_rng(21)
    raw = ggml(rng, fmt, rows, cols)
    w = backend.create_q4_weights(raw, rows, cols, fmt)
    wd, wm = parts(raw, fmt)
    for n in (3, 6, 20, 70):
        x = (rng.standard_normal((n, cols)) * 10.0 ** rng.uniform(-20, 20, (n, 1))).astype(np.float32)
        check(run(backend, w, x), x, wd, wm)
        x = (rng.standard_normal((n, cols)) * 10.0 ** rng.uniform(-3, 3, (n, cols))).astype(np.float32)
        check(run(backend, w, x), x, wd, wm)
        x[:] = 0
        assert np.all(run(backend, w, x) == 0)


@pytest.mark.parametrize("fmt", ["q4_0", "q4_k"])
@pytest.mark.parametrize("n", [1, 3, 6, 20, 70])
def test_non_finite_vectors_keep_to_themselves(backend, fmt, n):
    rows, cols = 40, 1024
    rng = np.random.default_rng(22)
    raw = ggml(rng, fmt, rows, cols)
    w = backend.create_q4_weights(raw, rows, cols, fmt)
    x = rng.standard_normal((n, cols)).astype(np.float32)
    clean = run(backend, w, x)
    y = x.copy()
    y[n // 2, 5] = np.inf
    got = run(backend, w, y)
    assert not np.isfinite(got[n // 2]).any()
    y[n // 2, 5] = np.nan
    nan = run(backend, w, y)
    assert np.isnan(nan[n // 2]).all()
    rest = np.arange(n) != n // 2
    assert np.array_equal(got[rest], clean[rest]) and np.array_equal(nan[rest], clean[rest])


def test_refusals_and_lifetime(backend):
    be, lib = backend, _lib.lib()
    raw = np.zeros(144 * 16, np.uint8)
    out = C.c_void_p()
    p = raw.ctypes.data
    for args in ((0, p, 0, 32), (0, p, 1, 0), (0, p, 1, 33), (0, p, -1, 32), (1, p, 1, 128), (1, p, 1, 32), (2, p, 1, 256),
                 (0, None, 1, 32), (-1, p, 1, 32)):
        assert lib.gla_q4w_create(be.ctx, *args, C.byref(out)) == _lib.GLA_ERR_INVALID, args
        assert not out.value
    w = be.create_q4_weights(raw[:18 * 16], 16, 32)
    assert lib.gla_q4w_rows(w.handle) == 16 and lib.gla_q4w_cols(w.handle) == 32
    x, y = be.buffer(np.zeros((4, 32), np.float32)), be.buffer(np.zeros((4, 16), np.float32))
    assert lib.gla_matvec_q4(be.ctx, w.handle, None, 0, None) == _lib.GLA_OK
    for args in ((w.handle, x.ptr, -1, y.ptr), (w.handle, None, 1, y.ptr), (w.handle, x.ptr, 1, None), (None, x.ptr, 1, y.ptr),
                 (w.handle, x.ptr, 262129, y.ptr)):
        assert lib.gla_matvec_q4(be.ctx, *args) == _lib.GLA_ERR_INVALID, args
    from glint_amd.attn import GpuBackend
    other = GpuBackend(0)
    theirs = other.create_q4_weights(raw[:18 * 16], 16, 32)
    assert lib.gla_matvec_q4(be.ctx, theirs.handle, x.ptr, 1, y.ptr) == _lib.GLA_ERR_INVALID
    other.close()
    assert lib.gla_matvec_q4(be.ctx, theirs.handle, x.ptr, 1, y.ptr) == _lib.GLA_ERR_INVALID
    assert "destroyed" in _lib.last_error()
    theirs.destroy()
    w.destroy()
    be.sync()
