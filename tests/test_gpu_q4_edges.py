"""gla_matvec_q4 where it can go wrong beside its sizes."""
import numpy as np
import pytest

import q4_structured as st
from glint_amd.attn import HipStream
from test_gpu_matvec_q4 import check, ggml, parts, run

pytestmark = pytest.mark.gpu


def with_zero_weights(rng, fmt, rows, cols):
    """Random blocks, some of whose weights are 0: nibbles of 8 are (Q4_0); nibbles of 0 in blocks without minima (Q4_K)."""
    raw = ggml(rng, fmt, rows, cols)
    if fmt == "q4_k":
        raw[rng.random(raw.shape[:2]) < 0.3, 2:4] = 0
    return raw


def odd_vectors(rng, n, cols):
    """Ordinary vectors, and among them some with infinities: one, two of one sign, two that differ, beside a NaN, nothing but."""
    x = rng.standard_normal((n, cols)).astype(np.float32)
    for i in range(n):
        at = rng.permutation(cols)
        kind = i % 8 if n > 1 else 1
        if kind == 1:
            x[i, at[0]] = np.inf
        elif kind == 2:
            x[i, cols - 1] = -np.inf
        elif kind == 3:
            x[i, at[:2]] = np.inf
        elif kind == 4:
            c = at[0] // 32 * 32  # in one group
            x[i, [c + 3, c + 17]] = np.inf, -np.inf
        elif kind == 5:
            x[i, 0], x[i, at[0]] = np.inf, np.nan
        elif kind == 6:
            x[i] = -np.inf
    return x


@pytest.mark.parametrize("fmt", ["q4_0", "q4_k"])
@pytest.mark.parametrize("rows, cols, ns", [(40, 1024, (1, 2, 3, 5, 8, 9, 20, 70)), (300, 4096, (1, 2, 4, 7, 33)), (4113, 512, (2, 4, 8, 30)),
                                            (8209, 512, (1,)), (14000, 512, (61, 120)), (1027, 2048, (2500,)), (1028, 512, (8100,))])
def test_infinities_meet_the_whole_weight(backend, fmt, rows, cols, ns):
    """An infinite element times a weight is an infinity of the weight's sign, and NaN where the weight is 0; sums of them, and
    with finite products, are IEEE's. Both formats, every kernel: 64 bits say which outputs are NaN, +inf, -inf and finite."""
    rng = np.random.default_rng(rows + cols)
    raw = with_zero_weights(rng, fmt, rows, cols)
    w = backend.create_q4_weights(raw, rows, cols, fmt)
    wd, wm = parts(raw, fmt)
    whole = wd - wm  # exact: 21 bits against 17, within a few binades
    assert (whole == 0).any()
    sign = np.sign(whole)
    alike = (sign == sign[:, :1]).all(1) & (sign[:, 0] != 0)
    every = np.where(alike, np.copysign(np.inf, -sign[:, 0]), np.nan)  # all of x is -inf
    for n in ns:
        x = odd_vectors(rng, n, cols)
        got = run(backend, w, x, shift=n % 2)
        odd = ~np.isfinite(x).all(1)
        assert odd.any() and np.isfinite(got[~odd]).all()
        want = np.zeros((int(odd.sum()), rows))
        for i, v in enumerate(x[odd].astype(np.float64)):
            at = ~np.isfinite(v)
            if at.all():
                want[i] = every
            else:
                with np.errstate(invalid="ignore"):
                    want[i] = (whole[:, at] * v[at]).sum(1)
        assert not np.isfinite(want).any()
        assert np.array_equal(got[odd].astype(np.float64), want, equal_nan=True), n


@pytest.mark.parametrize("n", [1, 6, 20, 2500])
def test_infinities_leave_the_other_vectors_their_bits(backend, n):
    """An infinity in one vector of a call changes no bit of the others'."""
    rows, cols = (1027, 2048) if n > 70 else (40, 1024)
    rng = np.random.default_rng(n)
    raw = ggml(rng, "q4_k", rows, cols)
    w = backend.create_q4_weights(raw, rows, cols, "q4_k")
    x = rng.standard_normal((n, cols)).astype(np.float32)
    clean = run(backend, w, x)
    x[n // 2, 5] = np.inf
    got = run(backend, w, x)
    rest = np.arange(n) != n // 2
    assert np.array_equal(got[rest], clean[rest])
    wd, wm = parts(raw, "q4_k")
    with np.errstate(invalid="ignore"):
        assert np.array_equal(got[n // 2].astype(np.float64), (wd - wm)[:, 5] * np.inf, equal_nan=True)


@pytest.mark.parametrize("fmt", ["q4_0", "q4_k"])
@pytest.mark.parametrize("rows, n, larger", [(6144, 400, 2000), (1027, 2500, 4000)])
def test_slices_without_their_own_scratch(backend, fmt, rows, n, larger):
    """A product in two slices of K whose partial sums and counters would have to grow during a capture takes the slices one
    after the other: an earlier call of more vectors, which needs neither, is enough before the capture. The bits are those of
    two slices at once, replay by replay."""
    be, cols = backend, 2048
    rng = np.random.default_rng(rows)
    raw = ggml(rng, fmt, rows, cols)
    w = be.create_q4_weights(raw, rows, cols, fmt)
    xs = [rng.standard_normal((n, cols)).astype(np.float32) for _ in range(2)]
    xs[1][3, 100] = np.inf
    want = [run(be, w, x) for x in xs]
    assert np.isfinite(want[0]).all()
    s = HipStream()
    try:
        be.set_stream(s)
        inp, out = be.buffer(xs[0]), be.empty(n * rows * 4)
        big, y = be.buffer(rng.standard_normal((larger, cols)).astype(np.float32)), be.empty(larger * rows * 4)
        be.matvec_q4(w, big, larger, y)
        be.sync()
        g = be.capture(lambda: be.matvec_q4(w, inp, n, out))
        for rep in range(4):
            inp.upload(xs[rep % 2])
            be.matvec_q4(w, big, larger, y)
            g.replay()
            be.sync()
            assert np.array_equal(out.download((n, rows)), want[rep % 2], equal_nan=True), rep
        g.destroy()
    finally:
        be.set_stream(None)
        s.destroy()


@pytest.mark.parametrize("fmt, rows, cols", [("q4_0", 96, 4096), ("q4_k", 96, 4096), ("q4_0", 4113, 576), ("q4_k", 1027, 2048)])
def test_batches_agree_within_their_roundings(backend, fmt, rows, cols):
    """The first vectors in batches that take other kernels, tiles and slices. Each call is off by at most 2^-22 of |x| and
    2^-38 of the largest |x| for the pieces, and half a step of f32 for each of cols / 32 + 64 additions (the longest chain);
    two calls by twice that. The same call twice, and with other vectors behind, has the same bits."""
    rng = np.random.default_rng(rows)
    raw = ggml(rng, fmt, rows, cols)
    w = backend.create_q4_weights(raw, rows, cols, fmt)
    wd, wm = parts(raw, fmt)
    x = rng.standard_normal((2500, cols)).astype(np.float32)
    x[0, 7] = 3e4  # an outlier: the scale of its own vector alone
    a = np.abs(x[:2].astype(np.float64))
    size = a @ (np.abs(wd) + wm).T
    largest = a.max(1, keepdims=True) * (np.abs(wd) + wm).sum(1)[None]
    bound = 2 * (size * (2.0 ** -22 + (cols / 32 + 64) * 2.0 ** -24) + largest * 2.0 ** -38)
    base = run(backend, w, x[:2])
    for n in (4, 8, 9, 33, 64, 100, 130, 400, 2500):
        got = run(backend, w, x[:n])[:2]
        assert np.all(np.abs(got.astype(np.float64) - base) <= bound), n
        other = x[:n].copy()
        other[2:] = -other[2:] * 1e3
        assert np.array_equal(run(backend, w, other)[:2], got), n


# (format, rows, columns): short rows, rows that leave waves without a quad or end inside one, the widest that is kept in
# registers when x is split (16,384 columns) and wider ones, tall matrices (two row tiles a workgroup)
STRUCTURED = [("q4_0", 33, 96), ("q4_0", 40, 576), ("q4_0", 47, 2080), ("q4_0", 20, 4128), ("q4_0", 33, 16384), ("q4_0", 33, 16416),
              ("q4_0", 17, 20480), ("q4_0", 4113, 5152), ("q4_k", 33, 256), ("q4_k", 47, 768), ("q4_k", 300, 4096), ("q4_k", 17, 16384),
              ("q4_k", 17, 16640), ("q4_k", 20, 20480), ("q4_k", 4113, 5120)]


@pytest.mark.parametrize("fmt, rows, cols", STRUCTURED)
def test_low_pieces_count_at_every_width(backend, fmt, rows, cols):
    """Vectors of four elements that need both pieces, each column in turn: a low piece that is lost, or of another column, is far
    outside the bound (shown on the CPU with the mistakes planted)."""
    rng = np.random.default_rng(cols + rows)
    raw = ggml(rng, fmt, rows, cols)
    w = backend.create_q4_weights(raw, rows, cols, fmt)
    wd, wm = parts(raw, fmt)
    first = 0
    for n in (1, 2, 4, 7, 8, 9, 16, 40, 64, 65, 130, 400, 1100):
        x = st.vectors(rng, n, cols, first if n < 400 else 0)
        assert st.holds(run(backend, w, x, shift=n % 2), x, wd, wm), n
        if cols > 16384 and n > 8:
            x = st.vectors(rng, n, cols, 16384)
            assert st.holds(run(backend, w, x, shift=n % 2), x, wd, wm), (n, "tail")
        first += n


@pytest.mark.parametrize("fmt", ["q4_0", "q4_k"])
@pytest.mark.parametrize("outlier", [1e3, 1e6, 1e9])
def test_an_outlier_on_zero_weights(backend, fmt, outlier):
    """The largest |x| sets the scale of its vector's pieces. Where all its weights are 0 (nibbles of 8; a superblock without
    scale and minimum), what is left of the others shows: an element is off by 2^-22 of itself (two halves, half a step of 11
    bits each) or by 2^-38 of the largest (half a step of the smallest half, 2^-25, against 2^13), whichever is more."""
    rows, cols, at = 48, 4096, 1030
    rng = np.random.default_rng(23)
    raw = ggml(rng, fmt, rows, cols)
    if fmt == "q4_0":
        raw[:, at // 32, 2 + at % 16] = raw[:, at // 32, 2 + at % 16] & 0xF0 | 8  # column 1030 is value 6 of its block
    else:
        raw[:, at // 256, :4] = 0
    w = backend.create_q4_weights(raw, rows, cols, fmt)
    wd, wm = parts(raw, fmt)
    assert not wd[:, at].any() and not wm[:, at].any()
    for n in (1, 3, 8, 9, 70, 300):
        x = rng.standard_normal((n, cols)).astype(np.float32)
        x[:, at] = outlier
        rest = np.abs(x.astype(np.float64))
        rest[:, at] = 0
        mag = np.abs(wd) + wm
        bound = rest @ mag.T * (2.0 ** -22 + (cols / 32 + 64) * 2.0 ** -24) + outlier * mag.sum(1) * 2.0 ** -38
        got = run(backend, w, x).astype(np.float64)
        assert np.all(np.abs(got - x.astype(np.float64) @ (wd - wm).T) <= bound), n


@pytest.mark.parametrize("fmt, cols", [("q4_0", 576), ("q4_0", 2048), ("q4_0", 2080), ("q4_0", 5152), ("q4_k", 512), ("q4_k", 2048),
                                       ("q4_k", 2304), ("q4_k", 5120)])
@pytest.mark.parametrize("rows, ns", [(4113, (2, 3, 4, 5, 8)), (4129, (2, 4, 7)), (8209, (1, 6)), (8225, (1,))])
def test_tall_matrices_and_few_vectors(backend, fmt, cols, rows, ns):
    """More row tiles than compute units (258 and 259; for one vector 514 and 515): two tiles a workgroup, the second one missing
    at the end of an odd number. Rows shorter than a wave's chunk, rows that end inside one, and longer ones."""
    rng = np.random.default_rng(rows + cols)
    raw = ggml(rng, fmt, rows, cols)
    w = backend.create_q4_weights(raw, rows, cols, fmt)
    wd, wm = parts(raw, fmt)
    for n in ns:
        x = rng.standard_normal((n, cols)).astype(np.float32)
        check(run(backend, w, x, shift=n % 2), x, wd, wm)
        x = st.vectors(rng, n, cols, int(rng.integers(0, cols)))
        assert st.holds(run(backend, w, x), x, wd, wm), n


@pytest.mark.parametrize("fmt, cols", [("q4_0", 2080), ("q4_k", 2304)])
@pytest.mark.parametrize("rows, n", [(1000, 33), (6133, 16), (6001, 17), (8100, 32), (6100, 63), (8100, 60), (14000, 61), (14300, 120)],
                         ids=["1x1", "1x2", "1x3", "1x4", "2x3", "2x4", "4x4", "8x4"])
def test_tiles_with_quads_for_every_wave(backend, fmt, cols, rows, n):
    """The middle kernel's tiles (of 16 vectors x of 16 rows, as 256 compute units choose them) over rows long enough that the
    ranges of K that its waves merge have work, the last of them less."""
    rng = np.random.default_rng(rows + n)
    raw = ggml(rng, fmt, rows, cols)
    w = backend.create_q4_weights(raw, rows, cols, fmt)
    wd, wm = parts(raw, fmt)
    x = rng.standard_normal((n, cols)).astype(np.float32)
    check(run(backend, w, x, shift=n % 2), x, wd, wm)
    x = st.vectors(rng, n, cols, int(rng.integers(0, cols)))
    assert st.holds(run(backend, w, x), x, wd, wm)


def test_a_graph_launched_on_another_stream(backend):
    """Products captured on one stream and replayed on another, between that one's own calls and without a wait: the graph has the
    scratch and counters of the first stream, the calls those of the second."""
    be, rows, cols = backend, 6144, 2048
    rng = np.random.default_rng(31)
    raw = ggml(rng, "q4_k", rows, cols)
    w = be.create_q4_weights(raw, rows, cols, "q4_k")
    sizes = (40, 400)  # pieces; pieces, partial sums and counters
    xs = [[rng.standard_normal((n, cols)).astype(np.float32) for n in sizes] for _ in range(2)]
    want = [[run(be, w, x) for x in pair] for pair in xs]
    x = [[be.buffer(a) for a in pair] for pair in xs]
    y = [[be.empty(n * rows * 4) for n in sizes] for _ in range(2)]

    def step(i):
        for a, b, n in zip(x[i], y[i], sizes):
            be.matvec_q4(w, a, n, b)

    streams = [HipStream(), HipStream()]
    try:
        be.set_stream(streams[0])
        step(0)
        be.sync()
        g = be.capture(lambda: step(0))
        be.set_stream(streams[1])
        for rep in range(4):
            step(1)
            g.replay()
            step(1)
            be.sync()
            for i in range(2):
                for b, n, right in zip(y[i], sizes, want[i]):
                    assert np.array_equal(b.download((n, rows)), right), (rep, i, n)
                    b.upload(np.zeros((n, rows), np.float32))
        g.destroy()
    finally:
        be.set_stream(None)
        for s in streams:
            s.destroy()
