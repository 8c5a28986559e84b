"""Two blocks as a model with alternating layers has them: norms, projection, append, attention in a window with sinks or over
a shared prefix, projection, norms; a prompt, then steps of its forks, every stage against 64 bits from the stage's own
input on the device; and the same step captured into a graph that is replayed as the rows grow."""
import numpy as np
import pytest

import test_gpu_matvec_q4 as q4
from helpers import assert_close, attention_f64
from test_gpu_append import PAGE, View, read
from test_gpu_block_norm import formula
from test_gpu_layer_steps import D, H, HKV, MODEL, SCALE, SPEC, WIDTH, Layer

pytestmark = pytest.mark.gpu

WINDOW, SINKS, PREFIX, CAP, EPS = 24, 5, 70, 128, 1e-5
SHARED = PREFIX // PAGE * PAGE  # positions in pages that the forks have in common


class Block:
    def __init__(self, be, seed):
        rng = np.random.default_rng(seed)
        self.layer = Layer(be, "q4_0", seed)
        self.post, self.gate = (rng.standard_normal(MODEL).astype(np.float32) for _ in range(2))
        self.pre = rng.standard_normal(MODEL).astype(np.float32)
        self.dpost, self.dgate, self.dpre = (be.buffer(t) for t in (self.post, self.gate, self.pre))


class Step:
    """Buffers of n rows: the stream, its norm, and what the stages of each block leave."""

    def __init__(self, be, n):
        self.n = n
        self.x, self.h = ([be.empty(4 * n * MODEL) for _ in range(3)] for _ in "xh")
        self.row, self.q, self.att, self.y = ([be.empty(4 * n * w) for _ in range(2)] for w in (WIDTH, H * D, H * D, MODEL))


class Model:
    def __init__(self, be, dtype, B):
        self.be, self.B = be, B
        rng = np.random.default_rng(B)
        self.blocks, self.plan = [Block(be, 3), Block(be, 4)], be.create_rope_plan(D, **SPEC)
        common, own = SHARED // PAGE, CAP // PAGE - SHARED // PAGE
        perm = rng.permutation(common + B * own).astype(np.int32)
        self.table = np.concatenate([np.tile(perm[:common], (B, 1)), perm[common:].reshape(B, own)], 1)
        self.kv = [be.create_page_pool(len(perm), HKV, D, dtype) for _ in range(2)]
        self.where = dict(page_table=be.buffer(np.ascontiguousarray(self.table)), page_table_stride=self.table.shape[1])
        self.groups, self.prefix = be.buffer(np.array([0, B], np.int32)), be.buffer(np.array([SHARED], np.int32))
        self.starts, self.zeros = be.buffer(np.arange(B + 1, dtype=np.int32)), be.buffer(np.zeros(B, np.int32))
        self.offsets, self.ends, self.first, self.length = (be.empty(4 * B) for _ in range(4))

    def at(self, past):
        past = np.asarray(past, np.int32)
        first = np.maximum(past + 1 - WINDOW, 0)
        for buf, v in ((self.offsets, past), (self.ends, past + 1), (self.first, first), (self.length, past + 1 - first)):
            buf.upload(v)

    def run(self, s, rows, attend):
        """The stages over s.n rows; `rows` says where they are, `attend(block, q, out)` is the attention."""
        be = self.be
        be.block_norm(s.x[0], s.n, MODEL, EPS, pre=self.blocks[0].dpre, norm_out=s.h[0])
        for i, b in enumerate(self.blocks):
            be.matvec_q4(b.layer.qkv, s.h[i], s.n, s.row[i])
            be.append(self.kv[i], View(s.row[i], H * D), View(s.row[i], (H + HKV) * D), *rows, rope=self.plan, q=s.row[i],
                      q_out=s.q[i], n_heads=H, k_stride=WIDTH, v_stride=WIDTH, q_stride=WIDTH, **self.where)
            attend(i, s.q[i], s.att[i])
            be.matvec_q4(b.layer.out, s.att[i], s.n, s.y[i])
            be.block_norm(s.x[i], s.n, MODEL, EPS, y=s.y[i], post=b.dpost, gate=b.dgate, scale=0.5, x_out=s.x[i + 1],
                          pre=self.blocks[1 - i].dpre, norm_out=s.h[i + 1])

    def token(self, s):
        def attend(i, q, out):
            if i == 0:
                self.be.decode(self.kv[0], q, out, self.first, self.length, self.B, WINDOW, H, SCALE, n_sinks=SINKS, **self.where)
            else:
                self.be.decode_shared(self.kv[1], q, out, self.zeros, self.ends, self.B, CAP, H, SCALE, self.groups, self.prefix,
                                      1, self.B, SHARED, CAP - SHARED, **self.where)
        self.run(s, (self.starts, self.offsets, self.B, 1), attend)

    def check(self, s, table, pos):
        """Every stage of the rows at `pos` of the sequences whose pages are the rows of `table`."""
        n, b0 = s.n, self.blocks[0]
        x = [t.download((n, MODEL)) for t in s.x]
        h = [t.download((n, MODEL)) for t in s.h]
        _, _, want, tol = formula(x[0], None, None, None, 1.0, b0.pre, EPS)
        assert np.all(np.abs(h[0] - want) <= tol)
        for i, b in enumerate(self.blocks):
            row, q, att, y = (t[i].download(shape) for t, shape in ((s.row, (n, WIDTH)), (s.q, (n, H, D)), (s.att, (n, H, D)),
                                                                    (s.y, (n, MODEL))))
            q4.check(row, h[i], *b.layer.qkv_parts)
            for r in range(n):
                j = np.arange(pos[r] + 1)
                j = j[(j > pos[r] - WINDOW) | (j < SINKS)] if i == 0 else j
                k, v = (t.reshape(-1, HKV, D) for t in read(self.be, self.kv[i], table[r, j // PAGE].astype(np.int64) * PAGE + j % PAGE))
                for head in range(H):
                    g = head // (H // HKV)
                    assert_close(att[r, head], attention_f64(q[r, head], k[:, g], v[:, g], SCALE), what=f"block {i} row {r}")
            q4.check(y, att.reshape(n, -1), *b.layer.out_parts)
            want_x, dx, want_h, dh = formula(x[i], y, b.post, b.gate, 0.5, self.blocks[1 - i].pre, EPS)
            assert np.all(np.abs(x[i + 1] - want_x) <= dx) and np.all(np.abs(h[i + 1] - want_h) <= dh)


def prompt(m, rng):
    """The common prompt through the first row's pages, its own tail copied to the forks' by the same call for each."""
    be = m.be
    s = Step(be, PREFIX)
    x = rng.standard_normal((PREFIX, MODEL)).astype(np.float32)
    starts, zero = be.buffer(np.array([0, PREFIX], np.int32)), be.buffer(np.zeros(1, np.int32))
    for b in reversed(range(m.B)):
        where, m.where = m.where, dict(page_table=be.buffer(np.ascontiguousarray(m.table[b:b + 1])), page_table_stride=m.table.shape[1])

        def attend(i, q, out):
            be.prefill(m.kv[i], q, out, starts, zero, 1, PREFIX, H, SCALE, sliding_window=WINDOW if i == 0 else None,
                       n_sinks=SINKS if i == 0 else 0, **m.where)
        s.x[0].upload(x)
        m.run(s, (starts, zero, 1, PREFIX), attend)
        be.sync()
        m.where = where
    m.check(s, np.repeat(m.table[:1], PREFIX, 0), np.arange(PREFIX))


@pytest.mark.parametrize("apart", ["0", "1"])
@pytest.mark.parametrize("dtype", ["f32", "q8"])
def test_prompt_and_steps_of_its_forks(backend, dtype, apart, monkeypatch):
    monkeypatch.setenv("GLA_DECODE_PREFIX", apart)
    rng = np.random.default_rng(17)
    m = Model(backend, dtype, 6)
    prompt(m, rng)
    s = Step(backend, m.B)
    for step in range(3):
        past = np.full(m.B, PREFIX + step)
        m.at(past)
        s.x[0].upload(rng.standard_normal((m.B, MODEL)).astype(np.float32))
        m.token(s)
        backend.sync()
        m.check(s, m.table, past)


@pytest.mark.parametrize("apart", ["0", "1"])
@pytest.mark.parametrize("dtype", ["f32", "q8"])
def test_captured_steps_equal_eager_ones(backend, dtype, apart, monkeypatch):
    """A captured step replayed as the rows grow, with eager steps of another batch between: the bits of eager steps."""
    monkeypatch.setenv("GLA_DECODE_PREFIX", apart)
    be, rng = backend, np.random.default_rng(19)
    m, other = Model(be, dtype, 5), Model(be, dtype, 9)
    for t in (m, other):
        prompt(t, rng)
    eager, replayed, aside = Step(be, 5), Step(be, 5), Step(be, 9)
    m.at(np.full(5, PREFIX))
    other.at(np.full(9, PREFIX))
    for t in (eager, replayed):
        t.x[0].upload(rng.standard_normal((5, MODEL)).astype(np.float32))
    aside.x[0].upload(rng.standard_normal((9, MODEL)).astype(np.float32))
    other.token(aside)
    m.token(eager)
    graph = be.capture(lambda: m.token(replayed))
    for step in range(5):
        m.at(PREFIX + step + np.array([0, 3, 1, 0, 7]))
        x = rng.standard_normal((5, MODEL)).astype(np.float32)
        eager.x[0].upload(x)
        replayed.x[0].upload(x)
        m.token(eager)
        other.token(aside)
        graph.replay()
        be.sync()
        for name in ("x", "h", "row", "q", "att", "y"):
            for a, b in zip(getattr(eager, name), getattr(replayed, name)):
                assert np.array_equal(a.download((a.nbytes // 4,)).view(np.uint32), b.download((b.nbytes // 4,)).view(np.uint32)), name
    graph.destroy()
