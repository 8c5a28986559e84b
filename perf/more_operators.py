"""What is timed of attention that keeps or shares a context's beginning, and of the norms between two blocks.

Four kinds of case, in the head shapes and widths of the benchmark and the tests:

* ``window``: one token of each sequence over a sliding window and a few first tokens that stay visible (sinks);
* ``chunk``: the same for the rows of prompts and prompt chunks;
* ``shared``: one token of each sequence of a batch whose groups begin with the same long prefix;
* ``norm``: a block's output normed, gated, scaled and added to the residual stream, and the sum normed for the next block.

K, V, queries and activations are N(0, 1). Lengths, groups and page tables follow from the case, values from the seed.
Where a case has layers, each has inputs of its own. Device buffers are torch tensors whose addresses the entry points
take.
"""
import ctypes
import math
import random

import numpy as np
import torch

own = False

PAGE = 16
SOFTCAP = 50.0
EPS = 1e-6

# (query heads, KV heads, head_dim, model width): SmolLM-135M, Llama-3-8B and Gemma-2-9B
SHAPES = {"smol": (9, 3, 64, 576), "llama": (32, 8, 128, 4096), "gemma": (16, 8, 256, 3584)}

_backend = None


def backend():
    """One backend for the process, as an engine keeps one."""
    global _backend
    if _backend is None:
        from glint_amd.attn import GpuBackend
        _backend = GpuBackend(0)
    return _backend


class Dev:
    """A torch tensor as the device buffer that the entry points take."""

    def __init__(self, t):
        self.t = t
        self.ptr = ctypes.c_void_p(t.data_ptr())


# ------------------------------------------------------------------ the cases

def window_case(shape, dtype="f32", paged=False, batch=1, lo=512, hi=512, window=256, sinks=4, layers=1, graph=False):
    return {"kind": "window", "shape": shape, "dtype": dtype, "paged": paged, "batch": batch, "lo": lo, "hi": hi,
            "window": window, "sinks": sinks, "layers": layers, "graph": graph}


def chunk_case(shape, dtype="f32", paged=False, batch=1, lo=512, hi=512, past=0, window=256, sinks=4):
    return {"kind": "chunk", "shape": shape, "dtype": dtype, "paged": paged, "batch": batch, "lo": lo, "hi": hi,
            "past": past, "window": window, "sinks": sinks, "layers": 1, "graph": False}


def shared_case(shape, dtype="q8", groups=1, batch=8, prefix=1024, lo=64, hi=512, layers=1, graph=False):
    return {"kind": "shared", "shape": shape, "dtype": dtype, "paged": True, "groups": groups, "batch": batch,
            "prefix": prefix, "lo": lo, "hi": hi, "layers": layers, "graph": graph}


def norm_case(width, rows, post=False, gate="none", scale=1.0, layers=1, graph=False):
    return {"kind": "norm", "width": width, "rows": rows, "post": post, "gate": gate, "scale": scale, "layers": layers,
            "graph": graph}


def listed():
    return [
        # one user's token of an endless chat on a small model: the default f32 cache, 16 layers captured
        dict(window_case("smol", lo=1531, hi=1531, window=512, sinks=4, layers=16, graph=True), name="window_one"),
        # a server's decode step: 64 conversations over a Q8_0 page pool
        dict(window_case("llama", "q8", True, batch=64, lo=128, hi=8192, window=2048, sinks=16), name="window_q8_b64"),
        # wide heads, soft-capped, the long window of an alternating model's local layers, f32 pages
        dict(window_case("gemma", "f32", True, batch=8, lo=4097, hi=9001, window=4096, sinks=64), name="window_f32_b8"),
        # a small model's next 40 tokens of a running chat
        dict(chunk_case("smol", batch=1, lo=40, hi=40, past=700, window=256, sinks=4), name="chunk_small"),
        # ragged prompts of a batch from their first tokens
        dict(chunk_case("llama", "q8", True, batch=4, lo=301, hi=2048, window=512, sinks=4), name="chunk_q8_prompts"),
        # chunks of two long documents behind a window's worth of cached positions, soft-capped wide heads
        dict(chunk_case("gemma", "f32", True, batch=2, lo=777, hi=1000, past=5000, window=4096, sinks=33), name="chunk_f32_long"),
        # four short samples of one prompt on a small model, 8 layers captured
        dict(shared_case("smol", "f32", batch=4, prefix=704, lo=1, hi=33, layers=8, graph=True), name="shared_small"),
        # a server whose 64 conversations begin with the same long instructions, Q8_0 pages
        dict(shared_case("llama", "q8", batch=64, prefix=8192, lo=64, hi=1000), name="shared_q8_b64"),
        # three documents asked about by 24 users, soft-capped wide heads, f32 pages
        dict(shared_case("gemma", "f32", groups=3, batch=24, prefix=4096, lo=17, hi=300), name="shared_f32_3"),
        # one token's residual stream between two blocks of a small model, 16 layers captured
        dict(norm_case(576, 1, layers=16, graph=True), name="norm_one"),
        # a decode batch between two blocks of a model that norms a block's output too, gated and scaled, 8 layers captured
        dict(norm_case(3584, 64, post=True, gate="vector", scale=0.5, layers=8, graph=True), name="norm_b64"),
        # a long prompt's rows, each with a gate of its own
        dict(norm_case(4096, 7993, post=True, gate="rows"), name="norm_prompt"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    limits = {"window": 5.5e8, "chunk": 2.41e9, "shared": 2.2e8, "norm": 6.6e8}  # of the largest listed case
    while True:
        kind = rng.choice(("window", "window", "chunk", "chunk", "shared", "shared", "norm"))
        if kind == "norm":
            width, rows = rng.choice((576, 3584, 4096, _log_int(rng, 33, 8192))), _log_int(rng, 1, 8192)
            c = norm_case(width, rows, rng.random() < 0.5, rng.choice(("none", "vector", "rows")), rng.choice((1.0, 0.5)),
                          4 if rows <= 64 else 1, rows <= 64 and rng.random() < 0.5)
        else:
            shape, dtype = rng.choice(tuple(SHAPES)), rng.choice(("f32", "q8"))
            paged = rng.random() < 0.7
            if kind == "window":
                hi = _log_int(rng, 20, 8192)
                c = window_case(shape, dtype, paged, _log_int(rng, 1, 64), rng.randint(1, hi), hi, _log_int(rng, 16, 4096),
                                _log_int(rng, 1, 128), 2, rng.random() < 0.5)
            elif kind == "chunk":
                hi = _log_int(rng, 2, 2048)
                c = chunk_case(shape, dtype, paged, _log_int(rng, 1, 4), rng.randint(max(1, hi // 8), hi), hi,
                               rng.choice((0, _log_int(rng, 10, 6000))), _log_int(rng, 16, 4096), _log_int(rng, 1, 128))
            else:
                hi, groups = _log_int(rng, 2, 1000), rng.choice((1, 1, 2, 4))
                c = shared_case(shape, dtype, groups, _log_int(rng, 2 * groups, 64), _log_int(rng, 64, 8192),
                                rng.randint(1, hi), hi, 2, rng.random() < 0.5)
        w = work(c)
        if max(w["bytes"], w["flops"] / 50) <= limits[kind]:
            return c


# ------------------------------------------------------------------ what follows from a case alone

def _rng(case, what):
    return random.Random(what + "/" + "/".join("%s=%s" % (k, case[k]) for k in sorted(case) if k != "name"))


def _ragged(case, what):
    """Lengths of the sequences. Ragged ones reach both ends."""
    r = _rng(case, what)
    n = [r.randint(case["lo"], case["hi"]) for _ in range(case["batch"])]
    n[0] = case["hi"]
    if case["batch"] > 1:
        n[-1] = case["lo"]
    return n


def group_starts(case):
    """The first row of each group of a shared case, and the number of rows."""
    cut = sorted(_rng(case, "groups").sample(range(1, case["batch"]), case["groups"] - 1))
    return [0] + cut + [case["batch"]]


def prefixes(case):
    """Positions that the rows of each group share."""
    r = _rng(case, "prefix")
    return [case["prefix"]] + [r.randint(case["prefix"] // 4, case["prefix"]) for _ in range(case["groups"] - 1)]


def group_of(case):
    starts = group_starts(case)
    return [g for g in range(case["groups"]) for _ in range(starts[g], starts[g + 1])]


def rows_of(case):
    """New rows of each sequence of a chunk case."""
    return _ragged(case, "lengths")


def pasts(case):
    """Positions that each sequence of a chunk case has in the cache already."""
    r = _rng(case, "past")
    return [case["past"]] + [r.randint(case["past"] // 2, case["past"]) for _ in range(case["batch"] - 1)]


def contexts(case):
    """Positions of each sequence, the last one's included."""
    if case["kind"] == "chunk":
        return [p + n for p, n in zip(pasts(case), rows_of(case))]
    n = _ragged(case, "lengths")
    if case["kind"] == "shared":
        n = [prefixes(case)[g] + m for g, m in zip(group_of(case), n)]
    return n


def page_table(case):
    """[B][pages] physical pages, a permutation of the pool, and the pool's size. The rows of a group have the whole pages
    of their prefix in common."""
    need = [(n + PAGE - 1) // PAGE for n in contexts(case)]
    common = [0] * len(need)
    if case["kind"] == "shared":
        group, starts = group_of(case), group_starts(case)
        common = [prefixes(case)[g] // PAGE if b > starts[g] else 0 for b, g in enumerate(group)]
    perm = list(range(sum(need) - sum(common)))
    _rng(case, "pages").shuffle(perm)
    table = np.zeros((len(need), max(need)), np.int32)
    at = 0
    for b, (n, c) in enumerate(zip(need, common)):
        if c:
            table[b, :c] = table[group_starts(case)[group_of(case)[b]], :c]
        table[b, c:n] = perm[at:at + n - c]
        at += n - c
    return table, len(perm)


def slots(case):
    """Rows of one layer's storage: positions of the contiguous caches (whole pages), slots of the pool."""
    if case["paged"]:
        return page_table(case)[1] * PAGE
    return case["batch"] * ((max(contexts(case)) + PAGE - 1) // PAGE * PAGE)


def storage_rows(case):
    """[B][positions] the storage row, in one layer's storage of a case of one layer, of each position."""
    pos = np.arange(max(contexts(case)))
    if case["paged"]:
        return page_table(case)[0][:, pos // PAGE].astype(np.int64) * PAGE + pos % PAGE
    return np.arange(case["batch"])[:, None] * (slots(case) // case["batch"]) + pos


def kv_row_bytes(case):
    """K and V of one position."""
    _, n_kv, d, _ = SHAPES[case["shape"]]
    return 2 * n_kv * d * 4 if case["dtype"] == "f32" else 2 * n_kv * (d // 32) * 34


def seen(case):
    """(positions of the storage that are read, pairs of a query row and a position that it sees)."""
    if case["kind"] == "shared":
        tails = [n - prefixes(case)[g] for n, g in zip(contexts(case), group_of(case))]
        return sum(prefixes(case)) + sum(tails), sum(contexts(case))
    w, s = case["window"], case["sinks"]
    if case["kind"] == "window":
        n = sum(min(e, w + min(s, max(e - w, 0))) for e in contexts(case))
        return n, n
    read = pairs = 0
    for past, n in zip(pasts(case), rows_of(case)):
        low = max(past - w + 1, 0)
        read += past + n - low + min(s, low)
        first = np.maximum(np.arange(past, past + n) - w + 1, 0)
        pairs += int((np.arange(past, past + n) + 1 - first + np.minimum(first, s)).sum())
    return read, pairs


def work(case):
    if case["kind"] == "norm":
        n, w = case["rows"], case["width"]
        vectors = 1 + case["post"] + (case["gate"] == "vector")
        rows = 4 + (case["gate"] == "rows")  # the block's output and the stream in, the stream and its norm out, a gate
        return {"bytes": case["layers"] * 4 * w * (rows * n + vectors), "flops": case["layers"] * 10 * n * w}
    n_heads, _, d, _ = SHAPES[case["shape"]]
    read, pairs = seen(case)
    rows = sum(rows_of(case)) if case["kind"] == "chunk" else case["batch"]
    return {"bytes": case["layers"] * (read * kv_row_bytes(case) + 8 * rows * n_heads * d),
            "flops": case["layers"] * 4 * n_heads * d * pairs}


# ------------------------------------------------------------------ inputs

def _gen(seed, what):
    g = torch.Generator(device="cuda")
    g.manual_seed((seed * 1000003 + what) & 0x7FFFFFFF)
    return g


def _normal(seed, what, shape, mul=1.0):
    t = torch.randn(shape, generator=_gen(seed, what), device="cuda", dtype=torch.float32)
    return t.mul_(mul) if mul != 1.0 else t


def queries(case, seed):
    n_heads, _, d, _ = SHAPES[case["shape"]]
    rows = sum(rows_of(case)) if case["kind"] == "chunk" else case["batch"]
    return _normal(seed, 2, (case["layers"], rows, n_heads, d))


def stored(case, seed, layer):
    """K and V [slots, kv_dim] of one layer as they were written. Pages that hold the end of a group's prefix beside a
    row's own positions have the same there."""
    _, n_kv, d, _ = SHAPES[case["shape"]]
    kv = [_normal(seed, 51 + 2 * layer + i, (slots(case), n_kv * d)) for i in (0, 1)]
    if case["kind"] == "shared":
        at, starts = storage_rows(case), group_starts(case)
        for g, n in enumerate(prefixes(case)):
            tail, rows = n // PAGE * PAGE, slice(starts[g] + 1, starts[g + 1])
            if tail < n and starts[g] + 1 < starts[g + 1]:
                src, dst = (torch.from_numpy(at[r, tail:n].copy()).cuda() for r in (starts[g], rows))
                for t in kv:
                    t[dst] = t[src]
    return kv


def norm_inputs(case, seed):
    """y, x, the post and pre weights, the gate: each with layers first, None where the case has none."""
    layers, n, w = case["layers"], case["rows"], case["width"]
    gate = {"none": None, "vector": (layers, 1, w), "rows": (layers, n, w)}[case["gate"]]
    return (_normal(seed, 1, (layers, n, w)), _normal(seed, 2, (layers, n, w)),
            _normal(seed, 3, (layers, w)) if case["post"] else None, _normal(seed, 4, (layers, w)),
            None if gate is None else _normal(seed, 5, gate))


def _rounded(x):
    """(quants, f16 scales) of f32 rows [..., kv_dim] by the Q8_0 cache's rules: the scale is max|x| / 127 (1 for an empty
    block), the quant x times its inverse, rounded half away from zero."""
    b = x.unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True)
    one = torch.ones_like(top)
    d = torch.where(top > 0, top / (127.0 * one), one)  # a tensor divisor: a plain number would become a product
    r = b * (one / d)
    q = torch.trunc(r)
    q = (q + torch.where((r - q).abs() >= 0.5, torch.sign(r), torch.zeros_like(r))).clamp_(-127.0, 127.0)
    return q.to(torch.int8), d.squeeze(-1).half()


def prepare(case, seed):
    s = {"case": case}
    if case["kind"] == "norm":
        s["y"], s["x"], s["post"], s["pre"], s["gate"] = norm_inputs(case, seed)
    else:
        s["q"] = queries(case, seed)
        s["end"] = np.array(contexts(case), np.int32)
        s["start"] = np.maximum(s["end"] - case["window"], 0) if case["kind"] == "window" else np.zeros_like(s["end"])
        if not own:
            kv = [stored(case, seed, layer) for layer in range(case["layers"])]
            s["k"], s["v"] = ([_rounded(t[i]) if case["dtype"] == "q8" else t[i] for t in kv] for i in (0, 1))
            s["at"] = torch.from_numpy(storage_rows(case)).cuda()
    if own:
        _prepare_own(s, seed)
    torch.cuda.synchronize()
    return s


# ------------------------------------------------------------------ the framework's calls

def _ints(a):
    return Dev(torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda())


def _prepare_own(s, seed):
    be, case = backend(), s["case"]
    layers = case["layers"]
    if case["kind"] == "norm":
        s["h"], s["sum"] = torch.zeros_like(s["x"]), torch.zeros_like(s["x"])
        s["devs"] = [{k: None if s[k] is None else Dev(s[k][layer]) for k in ("y", "x", "post", "pre", "gate", "h", "sum")}
                     for layer in range(layers)]
    else:
        _, n_kv, d, _ = SHAPES[case["shape"]]
        if case["paged"]:
            table, pages = page_table(case)
            s["kv"] = be.create_page_pool(layers * pages, n_kv, d, case["dtype"])
            s["table"], s["stride"] = [_ints(table + layer * pages) for layer in range(layers)], table.shape[1]
        else:
            s["kv"] = be.create_kv_cache(layers, slots(case) // case["batch"], n_kv, d, case["dtype"], n_seqs=case["batch"])
        for layer in range(layers):
            k, v = stored(case, seed, layer)
            row = torch.arange(slots(case), device="cuda")
            if case["paged"]:
                row += layer * slots(case)
            else:  # a cache holds the layers of a sequence one after the other
                each = slots(case) // case["batch"]
                row = (row // each * layers + layer) * each + row % each
            torch.cuda.synchronize()
            s["kv"].write_rows_device(Dev(row), Dev(k), Dev(v), len(row))
            be.sync()
        s["out"] = torch.zeros_like(s["q"])
        s["qd"], s["outd"] = [Dev(t) for t in s["q"]], [Dev(t) for t in s["out"]]
        s["len"] = s["end"] - s["start"]
        s["startd"], s["lend"] = _ints(s["start"]), _ints(s["len"])
        if case["kind"] == "chunk":
            s["rowsd"], s["pastd"] = _ints([0] + list(np.cumsum(rows_of(case)))), _ints(pasts(case))
        if case["kind"] == "shared":
            s["groups"], s["prefix"] = (np.array(f(case), np.int32) for f in (group_starts, prefixes))
            s["groupsd"], s["prefixd"] = _ints(s["groups"]), _ints(s["prefix"])
    torch.cuda.synchronize()
    if case["graph"]:
        _step(s)  # sizes the scratch
        be.sync()
        s["graph"] = be.capture(lambda: _step(s))


def _step(s):
    be, case = backend(), s["case"]
    if case["kind"] == "norm":
        stride = case["width"] if case["gate"] == "rows" else 0
        for d in s["devs"]:
            be.block_norm(d["x"], case["rows"], case["width"], EPS, y=d["y"], post=d["post"], gate=d["gate"],
                          gate_stride=stride, scale=case["scale"], x_out=d["sum"], pre=d["pre"], norm_out=d["h"])
        return
    n_heads, _, d, _ = SHAPES[case["shape"]]
    cap = SOFTCAP if case["shape"] == "gemma" else None
    for layer in range(case["layers"]):
        where = ({"page_table": s["table"][layer], "page_table_stride": s["stride"]} if case["paged"] else {"layer": layer})
        if case["kind"] == "chunk":
            be.prefill(s["kv"], s["qd"][layer], s["outd"][layer], s["rowsd"], s["pastd"], case["batch"], case["hi"], n_heads,
                       1.0 / math.sqrt(d), softcap=cap, sliding_window=case["window"], n_sinks=case["sinks"], **where)
            continue
        if not case["graph"]:
            where.update(kv_start_host=s["start"], kv_len_host=s["len"])
        if case["kind"] == "window":
            be.decode(s["kv"], s["qd"][layer], s["outd"][layer], s["startd"], s["lend"], case["batch"], int(s["len"].max()),
                      n_heads, 1.0 / math.sqrt(d), softcap=cap, n_sinks=case["sinks"], **where)
        else:
            if not case["graph"]:
                where.update(group_start_host=s["groups"], prefix_len_host=s["prefix"])
            be.decode_shared(s["kv"], s["qd"][layer], s["outd"][layer], s["startd"], s["lend"], case["batch"],
                             int(s["len"].max()), n_heads, 1.0 / math.sqrt(d), s["groupsd"], s["prefixd"], case["groups"],
                             int(np.diff(s["groups"]).max()), int(s["prefix"].max()), case["hi"], softcap=cap, **where)


# ------------------------------------------------------------------ the plain forms

def _held(store, at):
    """The values of storage rows [..., kv_dim]."""
    if isinstance(store, tuple):
        return (store[0][at].float() * store[1][at].float().unsqueeze(-1)).flatten(-2)
    return store[at]


def _scores(q, k, cap):
    """q [..., kv heads, rows, d] and k [..., kv heads, positions, d]."""
    t = torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(q.shape[-1])
    return t if cap is None else cap * torch.tanh(t / cap)


def _heads(store, at, n_kv):
    """K or V of storage rows [..., positions] as [..., kv heads, positions, d]."""
    return _held(store, at).unflatten(-1, (n_kv, -1)).transpose(-2, -3)


def _window_plain(s, layer, cap, n_kv):
    case = s["case"]
    end, start = (torch.from_numpy(s[k]).cuda().long() for k in ("end", "start"))
    first = torch.minimum(start, torch.tensor(case["sinks"], device="cuda"))  # sinks in front of the window
    most = int((first + end - start).max())
    i = torch.arange(most, device="cuda")
    pos = torch.where(i < first.unsqueeze(1), i, i - first.unsqueeze(1) + start.unsqueeze(1))
    hidden = pos >= end.unsqueeze(1)
    at = s["at"].gather(1, pos.clamp(max=s["at"].shape[1] - 1))
    k, v = _heads(s["k"][layer], at, n_kv), _heads(s["v"][layer], at, n_kv)
    q = s["q"][layer].unflatten(1, (n_kv, -1))
    t = _scores(q, k, cap).masked_fill(hidden[:, None, None], -math.inf)
    p = torch.exp(t - t.amax(-1, keepdim=True))
    return (torch.matmul(p, v) / p.sum(-1, keepdim=True)).flatten(1, 2)


def _chunk_plain(s, layer, cap, n_kv):
    case, outs, at_row = s["case"], [], 0
    for b, (past, n) in enumerate(zip(pasts(case), rows_of(case))):
        low = max(past - case["window"] + 1, 0)
        pos = torch.cat((torch.arange(min(case["sinks"], low), device="cuda"), torch.arange(low, past + n, device="cuda")))
        mine = torch.arange(past, past + n, device="cuda").unsqueeze(1)
        sees = (pos <= mine) & ((pos > mine - case["window"]) | (pos < case["sinks"]))
        k, v = _heads(s["k"][layer], s["at"][b, pos], n_kv), _heads(s["v"][layer], s["at"][b, pos], n_kv)
        q = s["q"][layer][at_row:at_row + n].unflatten(1, (n_kv, -1)).permute(1, 2, 0, 3)
        t = _scores(q, k.unsqueeze(1), cap).masked_fill(~sees, -math.inf)
        p = torch.exp(t - t.amax(-1, keepdim=True))
        outs.append((torch.matmul(p, v.unsqueeze(1)) / p.sum(-1, keepdim=True)).permute(2, 0, 1, 3).flatten(1, 2))
        at_row += n
    return torch.cat(outs)


def _shared_plain(s, layer, cap, n_kv):
    case, outs = s["case"], []
    starts, end = group_starts(case), s["end"]
    for g, n in enumerate(prefixes(case)):
        a, b = starts[g], starts[g + 1]
        q = s["q"][layer][a:b].unflatten(1, (n_kv, -1))  # [rows, kv heads, heads, d]
        # the prefix once: the rows and heads that share a KV head are the rows of one product
        at = s["at"][a, :n]
        k, v = _heads(s["k"][layer], at, n_kv), _heads(s["v"][layer], at, n_kv)
        t = _scores(q.transpose(0, 1).flatten(1, 2), k, cap)
        m0 = t.amax(-1, keepdim=True)
        p = torch.exp(t - m0)
        l0, o0 = (x.unflatten(1, (b - a, -1)).transpose(0, 1) for x in (p.sum(-1, keepdim=True), torch.matmul(p, v)))
        m0 = m0.unflatten(1, (b - a, -1)).transpose(0, 1)
        # what each row has of its own
        most = int(end[a:b].max()) - n
        pos = n + torch.arange(most, device="cuda")
        hidden = pos >= torch.from_numpy(end[a:b]).cuda().unsqueeze(1)
        at = s["at"][a:b, n:n + most]
        k, v = _heads(s["k"][layer], at, n_kv), _heads(s["v"][layer], at, n_kv)
        t = _scores(q, k, cap).masked_fill(hidden[:, None, None], -math.inf)
        m = torch.maximum(m0, t.amax(-1, keepdim=True))
        p, f = torch.exp(t - m), torch.exp(m0 - m)
        o = (o0 * f + torch.matmul(p, v)) / (l0 * f + p.sum(-1, keepdim=True))
        outs.append(o.flatten(1, 2))
    return torch.cat(outs)


def _normed(x, weight):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.unsqueeze(-2)


def _run_plain(s):
    case = s["case"]
    if case["kind"] == "norm":
        z = s["y"] if s["post"] is None else _normed(s["y"], s["post"])
        z = z if s["gate"] is None else z * s["gate"]
        x = s["x"] + case["scale"] * z
        return {"x": x, "h": _normed(x, s["pre"])}
    form = {"window": _window_plain, "chunk": _chunk_plain, "shared": _shared_plain}[case["kind"]]
    cap = SOFTCAP if case["shape"] == "gemma" else None
    return {"out": torch.stack([form(s, layer, cap, SHAPES[case["shape"]][1]) for layer in range(case["layers"])])}


def run(state):
    if not own:
        return _run_plain(state)
    if "graph" in state:
        state["graph"].replay()
    else:
        _step(state)
    return {"x": state["sum"], "h": state["h"]} if state["case"]["kind"] == "norm" else {"out": state["out"]}


# ------------------------------------------------------------------ the same in 64 bits

def _values64(x, dtype):
    """f64 values that the storage holds of f32 rows; Q8_0's scale and quants are defined in f32."""
    if dtype == "f32":
        return x.double()
    b = x.double().reshape(x.shape[0], -1, 32)
    top = b.abs().max(-1, keepdim=True).values
    d = torch.where(top > 0, (top / 127).float().double(), torch.ones_like(top))
    r = (b * (1 / d).float().double()).float().double()
    q = (torch.sign(r) * torch.floor(r.abs() + 0.5)).clamp(-127, 127)
    return (q * d.half().double()).reshape(x.shape)


def exact(case, seed):
    if case["kind"] == "norm":
        y, x, post, pre, gate = (None if t is None else t.double() for t in norm_inputs(case, seed))

        def normed(t, w):
            return w[:, None] * t / torch.sqrt(t.square().sum(-1, keepdim=True) / t.shape[-1] + EPS)

        z = normed(y, post) if case["post"] else y
        x = x + case["scale"] * (z if gate is None else gate * z)
        return {"x": x, "h": normed(x, pre)}
    n_heads, n_kv, d, _ = SHAPES[case["shape"]]
    at, ends = storage_rows(case), contexts(case)
    counts = rows_of(case) if case["kind"] == "chunk" else [1] * case["batch"]
    outs = []
    for layer, q in enumerate(queries(case, seed).double()):
        k_all, v_all = stored(case, seed, layer)
        out, row = torch.empty_like(q), 0
        for b, (e, n) in enumerate(zip(ends, counts)):
            # every position up to the last one that any row of the sequence sees, and a bound on each side of each row
            low = 0 if case["kind"] == "shared" else max(e - n - case["window"] + 1, 0)
            keep = np.array([j for j in range(e) if j >= low or j < case.get("sinks", 0)])
            rows = torch.from_numpy(at[b, keep]).cuda()
            k, v = (_values64(t[rows], case["dtype"]).reshape(-1, n_kv, d) for t in (k_all, v_all))
            j, p = torch.from_numpy(keep).cuda(), torch.arange(e - n, e, device="cuda")[:, None]
            ok = j <= p
            if case["kind"] != "shared":
                ok &= (p - j < case["window"]) | (j < case["sinks"])
            for h in range(n_heads):
                kh, vh = k[:, h * n_kv // n_heads], v[:, h * n_kv // n_heads]
                t = q[row:row + n, h] @ kh.T.contiguous() / math.sqrt(d)
                if case["shape"] == "gemma":
                    t = SOFTCAP * torch.tanh(t / SOFTCAP)
                t[~ok] = -math.inf
                out[row:row + n, h] = torch.softmax(t, -1) @ vh
            row += n
        outs.append(out)
    return {"out": torch.stack(outs)}
