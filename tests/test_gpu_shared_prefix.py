"""gla_decode_shared: a batch whose groups of rows begin with the same pages, against 64-bit attention row by row."""
import numpy as np
import pytest

from glint_amd import _lib
from glint_amd.attn import HipStream
from helpers import assert_close
from seen_ref import PAGE, Batch, seen

pytestmark = pytest.mark.gpu

SHAPES = [(9, 3, 64), (32, 8, 128), (16, 8, 256), (5, 1, 128), (7, 7, 64), (24, 2, 64), (2, 2, 256)]


def shared(b, q, groups, prefix, start, length, scale, cap=None, host="all", slack=0, n_groups=None, bounds=None):
    """The call, with host copies of everything, of the windows ("windows") or of nothing ("none")."""
    be, n = b.be, len(q)
    out = be.buffer(np.full(q.shape, -7.0, np.float32))
    groups, prefix, start, length = (np.asarray(a, np.int32) for a in (groups, prefix, start, length))
    kw = dict(b.where)
    if host != "none":
        kw.update(kv_start_host=start, kv_len_host=length)
    if host == "all":
        kw.update(group_start_host=groups, prefix_len_host=prefix)
    mine = np.zeros(n, np.int64)
    for r in range(n):
        g = np.searchsorted(groups, r, side="right") - 1
        mine[r] = int(start[r]) + int(length[r]) - (int(prefix[g]) if 0 <= g < len(prefix) else 0)
    if bounds is None:
        bounds = (int(np.diff(groups).max(initial=0)) + slack, int(prefix.max(initial=0)) + slack, max(int(mine.max()), 0) + slack)
    be.decode_shared(b.kv, be.buffer(q), out, be.buffer(start), be.buffer(length), n,
                     min(int(length.max()) + slack, b.limit), q.shape[1], scale,
                     be.buffer(groups), be.buffer(prefix if len(prefix) else np.zeros(1, np.int32)),
                     len(prefix) if n_groups is None else n_groups, *bounds, softcap=cap, **kw)
    be.sync()
    return out.download(q.shape)


def make(be, rng, dtype, H, n_kv, d, sizes, prefix, own, paged=True, lead=0, trail=0, **kw):
    """Groups of `sizes` rows after `lead` rows of no group and before `trail` more; own(row) positions past the prefix."""
    groups = lead + np.concatenate([[0], np.cumsum(sizes)])
    n = groups[-1] + trail
    lens, common, of = [], [], []
    for r in range(n):
        g = int(np.searchsorted(groups, r, side="right")) - 1
        inside = 0 <= g < len(sizes)
        lens.append((prefix[g] if inside else 0) + own(r))
        common.append(prefix[g] // PAGE * PAGE if inside and r > groups[g] and lens[-1] >= prefix[g] else 0)
        of.append(groups[g] if inside else r)
    if not paged:  # every sequence has its own copy of the prefix
        def fill(b, more=kw.pop("fill", None)):
            for r in range(n):
                if common[r]:
                    src, dst = (b.at(i, np.arange(common[r])) for i in (of[r], r))
                    b.k[dst], b.v[dst] = b.k[src], b.v[src]
            if more:
                more(b)
        b = Batch(be, rng, dtype, False, lens, n_kv, d, fill=fill, **kw)
    else:
        b = Batch(be, rng, dtype, True, lens, n_kv, d, common=common, common_of=of, **kw)
    q = rng.standard_normal((n, H, d)).astype(np.float32)
    return b, q, groups, np.array(lens)


def want(b, q, start, end, scale, cap=None):
    return np.stack([b.attend(r, q[r], seen(int(s), int(e), 0), scale, cap) for r, (s, e) in enumerate(zip(start, end))])


# (rows of each group, prefixes, own positions by row)
GROUPS = [
    ([2], [16], lambda r: 1 + r),
    ([5], [100], lambda r: [1, 16, 40, 7, 300][r]),
    ([1, 4, 9], [33, 700, 48], lambda r: 1 + 13 * r),
    ([40], [321], lambda r: 1 + (7 * r) % 50),
    ([3, 70], [2100, 1], lambda r: 1 + r % 5),
    ([2, 2], [5, 0], lambda r: 20 + r),
]


@pytest.mark.parametrize("sizes, prefix, own", GROUPS, ids=lambda v: str(v) if isinstance(v, list) else "")
@pytest.mark.parametrize("dtype", ["f32", "q8"])
@pytest.mark.parametrize("H, n_kv, d", SHAPES)
def test_rows_of_groups(backend, H, n_kv, d, dtype, sizes, prefix, own):
    rng = np.random.default_rng(d + H + sum(sizes))
    b, q, groups, end = make(backend, rng, dtype, H, n_kv, d, sizes, prefix, own)
    cap = 30.0 if len(sizes) == 3 else None
    ref = want(b, q, end * 0, end, d ** -0.5, cap)
    assert_close(shared(b, q, groups, prefix, end * 0, end, d ** -0.5, cap), ref)
    assert_close(shared(b, q, groups, prefix, end * 0, end, d ** -0.5, cap, host="none", slack=37), ref)


@pytest.mark.parametrize("dtype", ["f32", "q8"])
@pytest.mark.parametrize("H, n_kv, d", SHAPES[:3])
def test_long_prefixes_and_long_rows(backend, H, n_kv, d, dtype):
    rng = np.random.default_rng(d)
    own = lambda r: [1, 2000, 17, 900, 130, 64][r % 6]
    b, q, groups, end = make(backend, rng, dtype, H, n_kv, d, [3, 14], [4097, 5000], own)
    ref = want(b, q, end * 0, end, d ** -0.5)
    for host in ("all", "windows", "none"):
        assert_close(shared(b, q, groups, [4097, 5000], end * 0, end, d ** -0.5, host=host), ref)


@pytest.mark.parametrize("dtype", ["f32", "q8"])
def test_rows_outside_groups_and_caches(backend, dtype):
    """Rows before the first group and behind the last; contiguous caches, whose sequences hold copies of the prefix."""
    rng = np.random.default_rng(4)
    for paged in (True, False):
        b, q, groups, end = make(backend, rng, dtype, 8, 2, 128, [4, 3], [200, 90], lambda r: 5 + 11 * r, paged=paged, lead=2, trail=3)
        ref = want(b, q, end * 0, end, 0.09)
        for host in ("all", "none"):
            assert_close(shared(b, q, groups, [200, 90], end * 0, end, 0.09, host=host), ref)


@pytest.mark.parametrize("dtype", ["f32", "q8"])
def test_windows_that_cut_the_prefix(backend, dtype):
    """Rows whose window begins inside the prefix, behind it or nowhere, or ends inside it; empty rows; groups of none."""
    rng = np.random.default_rng(6)
    sizes, prefix = [9, 0, 4], [330, 50, 64]
    b, q, groups, end = make(backend, rng, dtype, 8, 2, 64, sizes, prefix, lambda r: 40 + r)
    start = np.array([0, 5, 100, 320, 329, 330, 350, 0, 377, 0, 0, 70, 20])
    end = end.copy()
    end[7], end[8], end[9], end[10] = 200, 377, 60, 0
    ref = want(b, q, start, end, 0.125, 20.0)
    for host in ("all", "windows", "none"):
        got = shared(b, q, groups, prefix, start, end - start, 0.125, 20.0, host=host)
        assert_close(got, ref)
        assert np.all(got[8] == 0) and np.all(got[10] == 0)


@pytest.mark.parametrize("dtype", ["f32", "q8"])
def test_one_page_and_one_position(backend, dtype):
    rng = np.random.default_rng(9)
    b, q, groups, end = make(backend, rng, dtype, 4, 4, 64, [6], [16], lambda r: 0)
    assert_close(shared(b, q, groups, [16], end * 0, end, 0.125), want(b, q, end * 0, end, 0.125))
    one = np.ones_like(end)
    assert_close(shared(b, q, groups, [16], end * 0, one, 0.125), want(b, q, end * 0, one, 0.125))


@pytest.mark.parametrize("dtype", ["f32", "q8"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_magnitudes(backend, dtype, d):
    """Keys, values and queries of unlike magnitudes in the prefix: what counts is the largest that a row meets."""
    rng = np.random.default_rng(10)

    def fill(b):
        at = b.at(0, np.arange(400))
        b.k[at] *= (2.0 ** rng.integers(-6, 3, (400, 1))).astype(np.float32)
        b.v[at] *= (2.0 ** rng.integers(-20, 6, (400, 1))).astype(np.float32)
        if dtype == "f32":
            b.v[at[100:200], ::7] *= np.float32(1e-12)
            b.k[at[7], :] = 0
            b.k[at[40:60], 3] = 1e-30

    b, q, groups, end = make(backend, rng, dtype, 8, 2, d, [7], [400], lambda r: 30 + r, fill=fill)
    q *= (2.0 ** rng.integers(-8, 3, (len(q), 8, 1))).astype(np.float32)
    scale = d ** -0.5
    ref = want(b, q, end * 0, end, scale)
    # a score's error: 2^-21 of the sum of |q k| (pieces of 22 bits) and d roundings of partial sums; it moves a weight by
    # as much, relative, and the output by twice that of the largest value
    worst = 0.0
    for r in range(len(q)):
        rows = b.at(r, np.arange(end[r]))
        worst = max(worst, float((np.abs(b.k[rows]).reshape(-1, 2, d)[:, np.arange(8) // 4] * np.abs(q[r])).sum(-1).max()) * scale)
    tol = 2 * (2.0 ** -21 + d * 2.0 ** -24) * worst * np.abs(b.v[b.at(0, np.arange(400))]).max() + 1e-5
    assert np.abs(shared(b, q, groups, [400], end * 0, end, scale) - ref).max() <= tol


@pytest.mark.parametrize("d", [64, 128, 256])
def test_small_blocks_of_values(backend, d):
    """Q8_0 values whose magnitudes differ from block to block of a head, by up to 2^18: each block's outputs are as near as
    its own largest value asks. One position of the prefix has nearly all the weight, so that what is lost of the small
    weights is not averaged away."""
    rng, n, H, n_kv = np.random.default_rng(11), 32, 8, 2  # (two pages: one wave's step)
    mul = np.exp2(np.resize([8.0, -10.0, -6.0, 0.0], d // 32)).repeat(32)
    u = rng.choice([-1.0, 1.0], (n_kv, d))
    scale = d ** -0.5

    def fill(b):
        b.k *= np.float32(0.03)
        b.k[b.at(0, 17)] = (9 * scale * u).reshape(-1)
        b.v *= np.tile(mul, n_kv).astype(np.float32)

    b, q, groups, end = make(backend, rng, "q8", H, n_kv, d, [5], [n], lambda r: 1 + r, fill=fill)
    q = (u.repeat(H // n_kv, 0) * rng.uniform(0.97, 1.03, q.shape)).astype(np.float32)
    ref = want(b, q, end * 0, end, scale)
    got = shared(b, q, groups, [n], end * 0, end, scale)
    # Scores: 9 * (1 +- 0.04) at the one position, |s| < 0.5 elsewhere, so that the others' weights are together below
    # `rest`. A score is off by e as in test_magnitudes (sum |q k| scale < 9.4); a weight by as much, relative, and 2^-20 for
    # the exponential; that moves an output by 2 e rest twice the block's largest value. Sums of up to n terms: n 2^-24.
    # A probability times a scale is held in steps of 2^-24 of 2^-13 of the largest scale (two f16 pieces, the largest in
    # 2^13 .. 2^14, rounded), 127 of them a value, for n positions.
    e = 2 * (2.0 ** -21 + d * 2.0 ** -24) * 9.4 + 2.0 ** -20
    rest = (n + 5) * np.exp(0.5 - 8.6)
    top = np.stack([np.abs(b.v[b.at(r, np.arange(end[r]))]).max(0) for r in range(len(q))]).max(0)
    top = top.reshape(n_kv, d // 32, 32).max(-1)[np.arange(H) * n_kv // H]  # [H][blocks]
    tol = (4 * e * rest + n * 2.0 ** -24) * top + n * 2.0 ** -25 * 2.0 ** -13 * top.max(-1, keepdims=True)
    err = np.abs(got - ref).reshape(len(q), H, d // 32, 32).max(-1)
    assert np.all(err <= tol), (err / tol).max((0, 1))


@pytest.mark.parametrize("dtype", ["f32", "q8"])
@pytest.mark.parametrize("n", [64, 65, 128, 300])
def test_many_groups(backend, dtype, n):
    """More groups than a wave has lanes, of unlike sizes and prefixes, some of no rows and some that share nothing; rows of no
    group before and behind them."""
    rng = np.random.default_rng(n)
    sizes = rng.integers(0, 4, n)
    sizes[[0, n // 2, n - 1]] = 2, 9, 3
    prefix = rng.integers(1, 80, n) * (rng.random(n) < 0.8)
    prefix[[0, n // 2, n - 1]] = 70, 200, 33
    b, q, groups, end = make(backend, rng, dtype, 6, 2, 64, sizes, prefix, lambda r: 1 + r % 40, lead=3, trail=2)
    ref = want(b, q, end * 0, end, 0.125)
    for host, slack in (("all", 0), ("all", 50), ("windows", 0), ("none", 21)):
        assert_close(shared(b, q, groups, prefix, end * 0, end, 0.125, host=host, slack=slack), ref)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_prefix_pages_that_no_row_sees(backend, d):
    """Windows that leave the prefix's first pages out: those are not read, so that values as large as they come there
    take nothing of the range of those that are seen."""
    rng, n = np.random.default_rng(13), 400

    def fill(b):
        b.v *= np.float32(2.0 ** -13)
        b.v[b.at(0, np.arange(176))] = 1e6 * rng.standard_normal((176, 2 * d))  # (11 pages: waves take two at least)

    b, q, groups, end = make(backend, rng, "q8", 8, 2, d, [5], [n], lambda r: 20 + r, fill=fill)
    start = np.array([176, 177, 191, 240, 300])
    ref = want(b, q, start, end, d ** -0.5)
    top = np.abs(b.v[b.at(0, np.arange(176, n))]).max()
    for host in ("all", "windows", "none"):
        got = shared(b, q, groups, [n], start, end - start, d ** -0.5, host=host)
        # (N(0, 1) data: outputs are averages of some ten values; 1e-4 of the largest, as for values near 1)
        assert np.abs(got - ref).max() <= 1e-4 * top


@pytest.mark.parametrize("dtype", ["f32", "q8"])
def test_non_finite_data(backend, dtype):
    """A NaN key makes the heads of its group NaN for the rows that see it, an infinite value its dimension; positions that
    no row sees do not count."""
    rng = np.random.default_rng(12)
    H, n_kv, d = 8, 2, 64

    def fill(b):
        b.v[b.at(0, 70), 5] = np.inf           # group 0, KV head 0
        b.k[b.at(4, 30), d + 3] = np.inf if dtype == "q8" else np.nan  # group 1, KV head 1
        gone = np.setdiff1d(np.arange(len(b.k)), np.concatenate([b.at(r, np.arange(e)) for r, e in enumerate(b.lens)]))
        b.k[gone], b.v[gone] = np.nan, np.inf

    b, q, groups, end = make(backend, rng, dtype, H, n_kv, d, [4, 3], [100, 41], lambda r: 10 + r, fill=fill)
    start = end * 0
    start[1], start[5] = 71, 31
    with np.errstate(invalid="ignore", over="ignore"):
        ref = want(b, q, start, end, 0.125)
    got = shared(b, q, groups, [100, 41], start, end - start, 0.125)
    assert np.array_equal(np.isnan(got), np.isnan(ref)) and np.array_equal(np.isposinf(got), np.isposinf(ref))
    ok = np.isfinite(ref)
    assert ok[1].all() and ok[5].all() and not ok[0].all() and not ok[4].all()
    assert np.all(np.abs(got - np.where(ok, ref, 0))[ok] <= 1e-4)


@pytest.mark.parametrize("dtype", ["f32", "q8"])
def test_captured_as_rows_grow(backend, dtype):
    """A captured call with the bounds of every replay, as the rows grow and the groups change; two streams."""
    be, rng = backend, np.random.default_rng(14)
    b, q, groups, end = make(be, rng, dtype, 8, 2, 128, [5, 12], [500, 160], lambda r: 200)
    n = len(q)
    dq, outs = be.buffer(q), [be.empty(q.nbytes) for _ in range(3)]
    start, length, gs, pl = be.buffer(end * 0), be.empty(4 * n), be.empty(12), be.empty(8)

    def call(out):
        be.decode_shared(b.kv, dq, out, start, length, n, b.limit, 8, 0.09, gs, pl, 2, n, 512, b.limit, **b.where)

    length.upload(end.astype(np.int32))
    gs.upload(groups.astype(np.int32))
    pl.upload(np.array([500, 160], np.int32))
    call(outs[0])
    graph = be.capture(lambda: call(outs[1]))
    other = HipStream()
    for step, (at, pre) in enumerate((([0, 5, 17], [500, 160]), ([0, 5, 9], [400, 160]), ([5, 5, 17], [16, 100]), ([0, 5, 17], [0, 0]))):
        now = end - 199 + 50 * step
        length.upload(now.astype(np.int32))
        gs.upload(np.array(at, np.int32))
        pl.upload(np.array(pre, np.int32))
        graph.replay()
        be.sync()
        be.set_stream(other)
        call(outs[2])
        be.set_stream(None)
        call(outs[0])
        be.sync()
        other.synchronize()
        got = [o.download(q.shape) for o in outs]
        assert np.array_equal(got[0].view(np.uint32), got[1].view(np.uint32))
        assert np.array_equal(got[0].view(np.uint32), got[2].view(np.uint32))
        assert_close(got[0], want(b, q, end * 0, now, 0.09))
    graph.destroy()
    other.destroy()


def test_malformed_device_values_stay_inside(backend):
    """Group starts that fall or leave the batch, prefixes and lengths past the storage: no fault, and the call after works."""
    rng = np.random.default_rng(15)
    for dtype in ("f32", "q8"):
        b, q, groups, end = make(backend, rng, dtype, 8, 2, 64, [4], [90], lambda r: 30)
        for at, pre in (([0, 9000], [90]), ([-5, 4], [90]), ([3, 1], [90]), ([0, 4], [2 ** 31 - 1]), ([0, 4], [-7])):
            shared(b, q, at, pre, end * 0, end, 0.125, host="none", bounds=(4, b.limit, b.limit))
        length = np.array([2 ** 31 - 1, -1, 40, 5])
        shared(b, q, [0, 4], [90], np.array([0, 0, 2 ** 31 - 1, -3]), length, 0.125, host="none", bounds=(4, b.limit, b.limit))
        assert_close(shared(b, q, groups, [90], end * 0, end, 0.125), want(b, q, end * 0, end, 0.125))


def test_refusals(backend):
    rng = np.random.default_rng(16)
    b, q, groups, end = make(backend, rng, "f32", 8, 2, 64, [2, 2], [90, 40], lambda r: 30)
    ok = dict(groups=groups, prefix=[90, 40], start=end * 0, length=end)
    shared(b, q, scale=0.1, **ok)
    for bad in (dict(groups=[0, 3, 2]), dict(groups=[-1, 2, 4]), dict(groups=[0, 2, 5]), dict(prefix=[-1, 40], bounds=(2, 90, 200)),
                dict(bounds=(1, 90, 30)), dict(bounds=(2, 89, 30)), dict(bounds=(2, 90, 29)), dict(bounds=(-1, 90, 30)),
                dict(bounds=(2, -1, 30)), dict(bounds=(2, 90, -1)), dict(n_groups=-1, host="windows"), dict(n_groups=5, host="windows"),
                dict(start=end * 0 - 1), dict(length=end + 10000)):
        with pytest.raises(_lib.GlaError) as e:
            shared(b, q, scale=0.1, **{**ok, **bad})
        assert e.value.code == _lib.GLA_ERR_INVALID, bad
    with pytest.raises(ValueError):
        backend.decode_shared(b.kv, None, None, None, None, 4, 1, 8, 0.1, None, None, 2, 1, 1, 1, group_start_host=groups)
    assert_close(shared(b, q, scale=0.1, **ok), want(b, q, end * 0, end, 0.1))
    assert_close(shared(b, q, [0], [], end * 0, end, 0.1), want(b, q, end * 0, end, 0.1))
