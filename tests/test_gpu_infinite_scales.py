"""Q8_0 values of which one block's scale is infinite: what a row sees of it is infinite or NaN there, as the values are, and
every other output is as near as without it, whether the others are large (a power of two for the infinity's sake would
overflow them) or small (it would lose their last bits)."""
import numpy as np
import pytest

from seen_ref import Batch, seen

pytestmark = pytest.mark.gpu

H, N_KV, AT, END = 8, 2, 20, 100  # the position of the infinite scale, and the rows' positions


def call(be, b, q, start, end, kind, scale):
    """Decode of all rows, of windows with sinks (the position is none), or with the first 96 positions read apart."""
    out, n = be.buffer(np.full(q.shape, -7.0, np.float32)), len(q)
    ints = lambda a: be.buffer(np.asarray(a, np.int32))
    args = (b.kv, be.buffer(q), out, ints(start), ints(end - start), n, b.limit, H, scale)
    if kind == "shared":
        be.decode_shared(*args, ints([0, n]), ints([96]), 1, n, 96, b.limit, **b.where)
    else:
        be.decode(*args, n_sinks=3 if kind == "sinks" else 0, **b.where)
    be.sync()
    return out.download(q.shape)


@pytest.mark.parametrize("kind", ["decode", "sinks", "shared"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("mul", [1e6, 2.0 ** -13])
@pytest.mark.parametrize("planted", [np.inf, 1e8])  # quants of 0, quants of the values' own
def test_other_values_beside_an_infinite_scale(backend, monkeypatch, kind, d, mul, planted):
    monkeypatch.setenv("GLA_DECODE_PREFIX", "1")
    rng, scale = np.random.default_rng(d), d ** -0.5

    def fill(b):
        b.v *= np.float32(mul)
        row = b.v[b.at(0, AT), :32]
        b.v[b.at(0, AT), :32] = planted * np.sign(row) * rng.uniform(0.5, 1.0, 32).astype(np.float32)

    end = np.full(4, END)
    b = Batch(backend, rng, "q8", True, end, N_KV, d, common=[0, 96, 96, 96], common_of=[0] * 4, fill=fill)
    q = rng.standard_normal((4, H, d)).astype(np.float32)
    start = np.array([0, AT + 1, 40, AT])  # two rows that see it, two that do not
    with np.errstate(invalid="ignore", over="ignore"):
        ref = np.stack([b.attend(r, q[r], seen(start[r], END, 3 if kind == "sinks" else 0), scale) for r in range(4)])
        got = call(backend, b, q, start, end, kind, scale)
    for f in (np.isnan, np.isposinf, np.isneginf):
        assert np.array_equal(f(got), f(ref)), f.__name__
    fin = np.isfinite(ref)
    assert fin[1].all() and fin[2].all() and not fin[0, 0, :32].any() and not fin[3, 0, :32].any()
    assert fin[0, :, 32:].all() and fin[0, H // N_KV:].all()
    # a score is off by 2^-21 of the sum of |q k| (pieces of 22 bits) and d roundings of partial sums; it moves a weight by
    # as much, relative, and the output by twice that of the largest value; the exponentials are off by 2^-22, and sums of
    # END terms by END 2^-24. A value is held in steps of 2^-24 of 2^-13 of the largest, for each position.
    worst = max(float((np.abs(b.k[b.at(r, np.arange(END))]).reshape(-1, N_KV, d)[:, np.arange(H) * N_KV // H]
                       * np.abs(q[r])).sum(-1).max()) for r in range(4)) * scale
    rows = b.v[b.at(0, np.arange(END))]
    top = np.abs(np.delete(rows, AT, 0)).max()
    tol = (2 * (2.0 ** -21 + d * 2.0 ** -24) * worst + 2.0 ** -21 + END * 2.0 ** -24 + END * 2.0 ** -38) * top
    assert np.abs(got - np.where(fin, ref, 0))[fin].max() <= tol
