"""Prefill with sinks at head_dim 256 where a call has more row blocks than the device has units: workgroups of eight waves,
whose rows are those of four waves bit for bit."""
import numpy as np
import pytest

from helpers import assert_close
from seen_ref import Batch
from test_gpu_sinks import prefill, want_prefill

pytestmark = pytest.mark.gpu

# (query heads, KV heads, rows of each sequence): groups of 2, 4, 1 and 3, an empty sequence, blocks that end inside a wave's tile
CASES = [(16, 8, [601, 333]), (32, 8, [250, 0, 301, 97]), (8, 8, [900, 130]), (12, 4, [1030])]


@pytest.mark.parametrize("cap", [None, 25.0])
@pytest.mark.parametrize("dtype", ["f32", "q8"])
@pytest.mark.parametrize("H, n_kv, rows", CASES, ids=str)
def test_many_rows(backend, H, n_kv, rows, dtype, cap):
    rng = np.random.default_rng(H + len(rows))
    d, window, sinks = 256, 150, 35
    past = [int(p) for p in rng.integers(0, 300, len(rows))]

    def fill(b):
        at = b.at(0, np.arange(past[0] + rows[0]))
        b.v[at] *= (2.0 ** rng.integers(-3, 3, (len(at), 1))).astype(np.float32)
        b.k[at[::97]] *= np.float32(2.0 ** -9)
        if dtype == "f32":
            b.v[at[past[0] + 40], 5], b.k[at[past[0] + 60], :8] = 1e-38, 1e-20

    b = Batch(backend, rng, dtype, True, [p + n for p, n in zip(past, rows)], n_kv, d, fill=fill)
    q_start = np.concatenate([[0], np.cumsum(rows)])
    q = rng.standard_normal((q_start[-1], H, d)).astype(np.float32)
    got = prefill(b, q, q_start, past, window, sinks, d ** -0.5, cap)
    pick = sorted(set(rng.choice(q_start[-1], 30, replace=False).tolist()) | {0, int(q_start[-1]) - 1})
    assert_close(got[pick], want_prefill(b, q, q_start, past, window, sinks, d ** -0.5, cap, set(pick))[pick])
    # the first sequence's first rows by themselves, its pages those of the batch's first row
    n = min(70, rows[0])
    alone = prefill(b, q[:n], [0, n], past[:1], window, sinks, d ** -0.5, cap)
    assert np.array_equal(alone.view(np.uint32), got[:n].view(np.uint32))


@pytest.mark.parametrize("dtype", ["f32", "q8"])
def test_captured(backend, dtype):
    be, rng = backend, np.random.default_rng(5)
    rows, past, H, n_kv, d = [601, 333], [10, 200], 16, 8, 256
    b = Batch(be, rng, dtype, True, [p + n for p, n in zip(past, rows)], n_kv, d)
    q = rng.standard_normal((sum(rows), H, d)).astype(np.float32)
    want = prefill(b, q, [0, 601, 934], past, 100, 5, 0.06)
    dq, out = be.buffer(q), be.empty(q.nbytes)
    at, first = be.buffer(np.array([0, 601, 934], np.int32)), be.buffer(np.array(past, np.int32))
    graph = be.capture(lambda: be.prefill(b.kv, dq, out, at, first, 2, 601, H, 0.06, None, 100, n_sinks=5, **b.where))
    for _ in range(3):
        out.upload(np.zeros_like(q))
        graph.replay()
        be.sync()
        assert np.array_equal(out.download(q.shape).view(np.uint32), want.view(np.uint32))
    graph.destroy()
