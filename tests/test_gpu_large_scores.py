"""Scores so large that a float near them no longer holds whole numbers, as far as 2^40: the largest takes the weight, equal
ones of one kernel share it, and nothing overflows, whatever power of two the Q8_0 kernels give their probabilities."""
import numpy as np
import pytest

from seen_ref import Batch, seen

pytestmark = pytest.mark.gpu

H, N_KV, END = 8, 2, 500


def call(be, b, q, kind, scale):
    out, n = be.buffer(np.full(q.shape, -7.0, np.float32)), len(q)
    ints = lambda a: be.buffer(np.asarray(a, np.int32))
    args = (b.kv, be.buffer(q), out, ints([0] * n), ints([END] * n), n, b.limit, H, scale)
    if kind == "shared":
        be.decode_shared(*args, ints([0, n]), ints([480]), 1, n, 480, b.limit, **b.where)
    else:
        be.decode(*args, n_sinks=3 if kind == "sinks" else 0, **b.where)
    be.sync()
    return out.download(q.shape)


def batch(be, rng, dtype, d, keys):
    def fill(b):
        at = b.at(0, np.arange(END))
        b.k[at] = keys
        b.k[b.at(1, np.arange(480, END))] = b.k[b.at(0, np.arange(480, END))]
        # magnitudes from page to page, so that waves scale their probabilities by powers of their own
        b.v *= np.exp2(np.arange(len(b.v)) // 16 % 11 - 5.0)[:, None].astype(np.float32)
    return Batch(be, rng, dtype, True, [END] * 2, N_KV, d, common=[0, 480], common_of=[0, 0], fill=fill)


@pytest.mark.parametrize("kind", ["decode", "sinks", "shared"])
@pytest.mark.parametrize("dtype", ["f32", "q8"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_large_scores(backend, monkeypatch, kind, dtype, d):
    monkeypatch.setenv("GLA_DECODE_PREFIX", "1")
    monkeypatch.setenv("GLA_Q8_CHUNK_PAGES", "2")  # (several waves and workgroups a row)
    rng, scale = np.random.default_rng(d), d ** -0.5
    u = rng.choice([-1.0, 1.0], (N_KV, d))
    q1 = u.repeat(H // N_KV, 0)
    for top in list(np.arange(20, 31, 0.75)) + [36.0, 40.0]:
        a = float(np.exp2(top / 2) * d ** -0.25)  # a score of 2^top
        q = np.tile((a * q1).astype(np.float32), (2, 1, 1))
        # one key above the others, at some place of the prefix or behind it; all alike, of either sign
        for at in (37, 250, 495):
            keys = np.tile(-a * u.reshape(1, -1), (END, 1))
            keys[at] = a * u.reshape(-1)
            b = batch(backend, rng, dtype, d, keys)
            ref = np.stack([b.attend(r, q[r], seen(0, END, 0), scale) for r in range(2)])
            got = call(backend, b, q, kind, scale)
            # (its value alone, in two halves of 11 bits or as it is)
            assert np.all(np.abs(got - ref) <= 2.0 ** -20 * np.abs(ref) + 2.0 ** -25 * np.abs(b.v).max()), (top, at)
        for sign in (1, -1):
            keys = np.tile(sign * a * u.reshape(1, -1), (END, 1))
            # (those behind the prefix are another kernel's, which adds d products in another order: d 2^-24 of a score is
            # more than 1 from 2^18 on, so that they cannot be told to be alike; they are lower)
            keys[480:] = -2 * a * u.reshape(-1)
            b = batch(backend, rng, dtype, d, keys)
            ref = np.stack([b.attend(r, q[r], seen(0, END, 0), scale) for r in range(2)])
            got = call(backend, b, q, kind, scale)
            # (the mean of END values: END roundings of sums, pieces of 22 bits)
            assert np.abs(got - ref).max() <= (END * 2.0 ** -24 + 2.0 ** -20) * np.abs(b.v).max(), (top, sign)
