"""A batch's K and V in a device pool or cache, and attention over the positions that a rule lets a row see, in 64 bits."""
from __future__ import annotations

import numpy as np

import oracle as orc

PAGE = 16


def held(x, dtype):
    """The values that the storage holds of f32 rows [n][kv_dim]."""
    if dtype == "f32":
        return np.asarray(x, np.float64)
    raw = orc.q8_quantize_rows(np.ascontiguousarray(x, np.float32)).reshape(len(x), -1, 34)
    d = raw[..., :2].copy().view(np.float16).astype(np.float64)
    return (raw[..., 2:].view(np.int8).astype(np.float64) * d).reshape(len(x), -1)


class Batch:
    """K and V [position][kv_dim] of each sequence in a pool of shuffled pages, or in a cache whose sequences are taken in
    another order than the batch's. `common[b]`: leading positions (whole pages) that row b reads from row common_of[b]'s
    pages."""

    def __init__(self, be, rng, dtype, paged, lens, n_kv, d, common=None, common_of=None, spare=2, k_mul=1.0, fill=None):
        self.be, self.dtype, self.paged, self.lens = be, dtype, paged, list(lens)
        self.n_kv, self.d = n_kv, d
        kv_dim, n = n_kv * d, len(self.lens)
        pages = [(e + PAGE - 1) // PAGE for e in self.lens]
        width = max(pages + [1]) + 1
        if paged:
            common = common or [0] * n
            total = sum(pages) - sum(c // PAGE for c in common) + spare
            perm = rng.permutation(total)
            self.table = np.full((n, width), -1, np.int32)
            at = 0
            for b in range(n):
                c = common[b] // PAGE
                if c:
                    self.table[b, :c] = self.table[common_of[b], :c]
                self.table[b, c:pages[b]] = perm[at:at + pages[b] - c]
                at += pages[b] - c
            rows = np.arange(total * PAGE, dtype=np.int64)
            self.kv = be.create_page_pool(total, n_kv, d, dtype)
            self.where = {"page_table": be.buffer(self.table), "page_table_stride": width}
            self.limit = width * PAGE
        else:
            max_seq = max(self.lens + [1]) + 3
            ppl = (max_seq + PAGE - 1) // PAGE
            self.slot = rng.permutation(n + 1)[:n].astype(np.int32)
            self.kv = be.create_kv_cache(2, max_seq, n_kv, d, dtype, n_seqs=n + 1)
            self.table = (self.slot[:, None] * 2 + 1) * ppl + np.arange(ppl)[None]
            rows = np.arange((n + 1) * 2 * ppl * PAGE, dtype=np.int64)
            self.where = {"layer": 1, "seq_slot": be.buffer(self.slot)}
            self.limit = max_seq
        self.k = (k_mul * rng.standard_normal((len(rows), kv_dim))).astype(np.float32)
        self.v = rng.standard_normal((len(rows), kv_dim)).astype(np.float32)
        if fill is not None:
            fill(self)
        self.kv.write_rows(rows, self.k, self.v)

    def at(self, b, pos):
        """Storage rows of positions of sequence b."""
        pos = np.asarray(pos)
        return self.table[b, pos // PAGE].astype(np.int64) * PAGE + pos % PAGE

    def attend(self, b, q, pos, scale, cap=None):
        """q [H][d] over the positions `pos` of sequence b, in 64 bits: [H][d]."""
        H, out = len(q), np.zeros(q.shape)
        if len(pos) == 0:
            return out
        rows = self.at(b, pos)
        k = held(self.k[rows], self.dtype).reshape(-1, self.n_kv, self.d)
        v = held(self.v[rows], self.dtype).reshape(-1, self.n_kv, self.d)
        for h in range(H):
            s = k[:, h * self.n_kv // H] @ q[h].astype(np.float64) * scale
            if cap:
                s = cap * np.tanh(s / cap)
            w = np.exp(s - s.max())
            out[h] = w @ v[:, h * self.n_kv // H] / w.sum()
        return out


def seen(start, end, sinks, low=0):
    """Positions that a row sees: before `end`, in the window from `start` on or among the first `sinks`."""
    if end <= start:
        return np.zeros(0, np.int64)
    j = np.arange(end)
    return j[(j >= start) | (j < sinks)]
