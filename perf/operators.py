"""What is timed of the operators around a cache step: rotary positions, the cache append and 4-bit projections.

Four kinds of case, in the head shapes of the benchmark and the tests:

* ``rope``: rotary positions of query rows, in both layouts, part of a head, scaled for long contexts;
* ``append``: the K and V of fused projection rows rotated, quantised and written into a cache or a page pool, their
  queries rotated beside them, and the written rows read back as the values that the storage holds;
* ``proj``: a projection with 4-bit weights (Q4_0 or Q4_K) of one token, a decode batch or a prompt chunk;
* ``layer``: a whole attention layer of a decode step through them: 4-bit Q/K/V projection, append, attention, 4-bit
  output projection.

Activations are N(0, 1), weights N(0, 1/cols) quantised. Lengths, positions and page tables follow from the case, values
from the seed. Where a case has layers, each has inputs of its own. Device buffers are torch tensors whose addresses the
entry points take.
"""
import ctypes
import math
import random

import numpy as np
import torch

own = False

PAGE = 16

# (query heads, KV heads, head_dim, model width): SmolLM-135M, Llama-3-8B and Gemma-2-9B
SHAPES = {"smol": (9, 3, 64, 576), "llama": (32, 8, 128, 4096), "gemma": (16, 8, 256, 3584)}

# how the frequencies are stretched for long contexts: the rule and its parameters
ROPES = {
    "plain": {"freq_base": 10000.0, "scaling": "none"},
    "linear": {"freq_base": 10000.0, "scaling": "linear", "factor": 4.0},
    "bands": {"freq_base": 500000.0, "scaling": "bands", "factor": 8.0, "original_ctx": 8192, "low": 1.0, "high": 4.0},
    "yarn": {"freq_base": 10000.0, "scaling": "yarn", "factor": 16.0, "original_ctx": 4096, "low": 1.0, "high": 32.0},
}

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

def rope_case(shape, rope, half, rows, rot=0, far=8192, layers=1, graph=False):
    return {"kind": "rope", "shape": shape, "rope": rope, "half": half, "rows": rows, "rot": rot, "far": far,
            "layers": layers, "graph": graph}


def append_case(shape, rope, half, dtype="f32", paged=False, batch=1, lo=1, hi=1, past=512, rot=0, layers=1, graph=False):
    return {"kind": "append", "shape": shape, "rope": rope, "half": half, "dtype": dtype, "paged": paged, "batch": batch,
            "lo": lo, "hi": hi, "past": past, "rot": rot, "layers": layers, "graph": graph}


def proj_case(fmt, rows, cols, n_vec, layers=1, graph=False):
    return {"kind": "proj", "fmt": fmt, "rows": rows, "cols": cols, "n_vec": n_vec, "layers": layers, "graph": graph}


def layer_case(shape, rope, half, qkv, out, batch, past, layers=1, graph=False):
    return {"kind": "layer", "shape": shape, "rope": rope, "half": half, "qkv": qkv, "out": out, "batch": batch,
            "lo": 1, "hi": 1, "past": past, "rot": 0, "dtype": "f32", "paged": True, "layers": layers, "graph": graph}


def listed():
    return [
        # one user's token: the query heads of 16 layers, a launch each, captured as a decode step is
        dict(rope_case("llama", "bands", True, 1, layers=16, graph=True), name="rope_one"),
        # the query rows of a long prompt chunk, a context stretched sixteen times
        dict(rope_case("llama", "yarn", False, 7993, far=65536), name="rope_prompt"),
        # one user's token into the default f32 cache, 16 layers captured
        dict(append_case("llama", "plain", False, past=4095, layers=16, graph=True), name="append_f32_one"),
        # a server's decode step: a token of each of 64 sequences into a Q8_0 page pool, 4 layers captured
        dict(append_case("llama", "bands", True, "q8", True, batch=64, past=8000, layers=4, graph=True), name="append_q8_b64"),
        # ragged prompts of a batch, the rest of cached conversations, into a Q8_0 page pool
        dict(append_case("llama", "bands", True, "q8", True, batch=6, lo=31, hi=2049, past=300), name="append_q8_prompts"),
        # wide heads rotated in part, prompt chunks into f32 caches
        dict(append_case("gemma", "linear", True, "f32", False, batch=3, lo=301, hi=1500, past=77, rot=96),
             name="append_f32_prompts"),
        # a small model's projection of a few tokens: launches and latency, 8 layers captured
        dict(proj_case("q4_0", 960, 576, 7, layers=8, graph=True), name="proj_q4_0_small_7"),
        # one user's token through the output projection, eight layers' weights in turn
        dict(proj_case("q4_0", 4096, 4096, 1, layers=8), name="proj_q4_0_1"),
        # one user's token through the fused Q/K/V projection
        dict(proj_case("q4_k", 6144, 4096, 1, layers=8), name="proj_q4_k_1"),
        # the same of a 64-sequence decode batch
        dict(proj_case("q4_k", 6144, 4096, 64, layers=4), name="proj_q4_k_64"),
        # and of the tokens of a long prompt
        dict(proj_case("q4_0", 6144, 4096, 1999), name="proj_q4_0_1999"),
        # a decode step's attention layer for 16 sequences, four layers captured
        dict(layer_case("llama", "bands", True, "q4_k", "q4_0", 16, 1500, layers=4, graph=True), name="layer_b16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    limit = 2.01e9  # of the largest listed case
    while True:
        kind = rng.choice(("rope", "append", "append", "proj", "proj", "layer"))
        shape = rng.choice(tuple(SHAPES))
        rope, half = rng.choice(tuple(ROPES)), rng.random() < 0.5
        d = SHAPES[shape][2]
        rot = rng.choice((0, 0, 2 * rng.randint(1, d // 2 - 1)))
        if kind == "rope":
            rows = _log_int(rng, 1, 8192)
            c = rope_case(shape, rope, half, rows, rot, _log_int(rng, 8192, 131072), 8 if rows <= 64 else 1,
                          rows <= 64 and rng.random() < 0.5)
        elif kind == "append":
            hi = rng.choice((1, 1, _log_int(rng, 2, 2048)))
            batch = _log_int(rng, 1, 128 if hi == 1 else 8)
            paged = rng.random() < 0.7
            c = append_case(shape, rope, half, rng.choice(("f32", "q8")), paged, batch, rng.randint(max(1, hi // 16), hi), hi,
                            _log_int(rng, 1, 8000 if paged else 1000), rot, 8 if hi == 1 else 1, hi == 1 and rng.random() < 0.5)
        elif kind == "proj":
            fmt = rng.choice(("q4_0", "q4_k"))
            rows, cols = rng.choice(((6144, 4096), (4096, 4096), (1024, 4096), (8192, 3584), (3584, 4096), (4096, 16384))
                                    + (((960, 576), (576, 576)) if fmt == "q4_0" else ((511, 512), (130, 256))))
            n_vec = _log_int(rng, 1, 2048)
            c = proj_case(fmt, rows, cols, n_vec, 4 if n_vec <= 64 else 1, n_vec <= 64 and rng.random() < 0.5)
        else:
            fmt = ("q4_0",) if SHAPES[shape][3] % 256 else ("q4_0", "q4_k")
            c = layer_case(shape, rope, half, rng.choice(fmt), rng.choice(fmt), _log_int(rng, 1, 32), _log_int(rng, 20, 2000),
                           2, rng.random() < 0.6)
        w = work(c)
        if max(w["bytes"], w["flops"] / 50) <= limit:
            return c


# ------------------------------------------------------------------ what follows from a case alone

def _rng(case, what):
    return random.Random(what + "/" + "/".join("%s=%s" % (k, case[k]) for k in sorted(case) if k != "name"))


def lengths(case):
    """New rows of each sequence of an append. Ragged ones reach both ends."""
    r = _rng(case, "lengths")
    n = [r.randint(case["lo"], case["hi"]) for _ in range(case["batch"])]
    if case["batch"] > 1:
        n[0], n[-1] = case["hi"], case["lo"]
    return n


def pasts(case):
    """Positions that each sequence has in the cache already."""
    r = _rng(case, "past")
    return [case["past"]] + [r.randint(case["past"] // 8, case["past"]) for _ in range(case["batch"] - 1)]


def page_table(case):
    """[B][pages] physical pages, a permutation of the pool, and the pool's size."""
    need = [(p + n + PAGE - 1) // PAGE for p, n in zip(pasts(case), lengths(case))]
    perm = list(range(sum(need)))
    _rng(case, "pages").shuffle(perm)
    table = np.zeros((len(need), max(need)), np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    return table, len(perm)


def slots(case):
    """Rows of one layer's storage: positions of the contiguous caches (whole pages), slots of the pool."""
    if case["paged"]:
        return page_table(case)[1] * PAGE
    return case["batch"] * ((max(p + n for p, n in zip(pasts(case), lengths(case))) + PAGE - 1) // PAGE * PAGE)


def kv_row_bytes(case):
    """K and V of one position."""
    _, n_kv, d, _ = SHAPES[case["shape"]]
    return 2 * n_kv * d * 4 if case["dtype"] == "f32" else 2 * n_kv * (d // 32) * 34


def weight_bytes(fmt, rows, cols):
    return rows * (cols // 32) * 18 if fmt == "q4_0" else rows * (cols // 256) * 144


def work(case):
    layers = case["layers"]
    if case["kind"] == "proj":
        r, c, n = case["rows"], case["cols"], case["n_vec"]
        return {"bytes": layers * (weight_bytes(case["fmt"], r, c) + 4 * n * (r + c)), "flops": layers * 2 * n * r * c}
    n_heads, n_kv, d, width = SHAPES[case["shape"]]
    rot = case["rot"] or d
    if case["kind"] == "rope":
        n = case["rows"]
        return {"bytes": layers * (8 * n * n_heads * d + 4 * n), "flops": layers * 3 * n * n_heads * rot}
    n = sum(lengths(case))
    step = 4 * n * (2 * n_heads + 2 * n_kv) * d + n * kv_row_bytes(case)  # the append: rows in, queries and storage out
    flops = 3 * n * (n_heads + n_kv) * rot
    if case["kind"] == "append":  # and the rows read back
        return {"bytes": layers * (step + n * kv_row_bytes(case) + 8 * n * n_kv * d), "flops": layers * flops}
    qkv, out = ((n_heads + 2 * n_kv) * d, width), (width, n_heads * d)
    seen = sum(pasts(case)) + n
    return {"bytes": layers * (weight_bytes(case["qkv"], *qkv) + weight_bytes(case["out"], *out) + n * kv_row_bytes(case)
                               + seen * kv_row_bytes(case) + 8 * n * width + 8 * n * n_heads * d),
            "flops": layers * (2 * n * (qkv[0] * qkv[1] + out[0] * out[1]) + 4 * n_heads * d * seen + flops)}


# ------------------------------------------------------------------ inputs

def _gen(seed, what):
    g = torch.Generator(device="cuda")
    g.manual_seed((seed * 1000003 + what) & 0x7FFFFFFF)
    return g


def _normal(seed, what, shape, mul=1.0):
    t = torch.randn(shape, generator=_gen(seed, what), device="cuda", dtype=torch.float32)
    return t.mul_(mul) if mul != 1.0 else t


def weights(seed, what, fmt, layers, rows, cols):
    """GGML bytes [layers, rows, blocks, 18 or 144] of N(0, 1/cols) matrices, on the GPU."""
    x = _normal(seed, what, (layers, rows, cols), 1.0 / math.sqrt(cols))
    if fmt == "q4_0":
        b = x.reshape(layers, rows, cols // 32, 32)
        top = b.gather(-1, b.abs().argmax(-1, keepdim=True))  # the value of the largest magnitude, with its sign
        d = top / -8.0
        q = torch.floor(b / torch.where(d == 0, torch.ones_like(d), d) + 8.5).clamp_(0, 15).to(torch.uint8)
        return torch.cat((d.half().view(torch.uint8), q[..., :16] | (q[..., 16:] << 4)), -1).contiguous()
    b = x.reshape(layers, rows, cols // 256, 8, 32)
    low = b.amin(-1).clamp_(max=0.0).neg_()
    step = (b.amax(-1) + low).clamp_(min=0.0) / 15.0
    d, dmin = (step.amax(-1, keepdim=True) / 63.0).half(), (low.amax(-1, keepdim=True) / 63.0).half()
    one = torch.ones_like(d, dtype=torch.float32)
    sc = torch.round(step / torch.where(d > 0, d.float(), one)).clamp_(0, 63)
    mn = torch.round(low / torch.where(dmin > 0, dmin.float(), one)).clamp_(0, 63)
    s, m = (d.float() * sc).unsqueeze(-1), (dmin.float() * mn).unsqueeze(-1)
    q = torch.round((b + m) / torch.where(s > 0, s, torch.ones_like(s))).clamp_(0, 15).to(torch.uint8)
    sc, mn = sc.to(torch.uint8), mn.to(torch.uint8)
    packed = torch.cat((sc[..., :4] | (sc[..., 4:] >> 4 << 6), mn[..., :4] | (mn[..., 4:] >> 4 << 6),
                        (sc[..., 4:] & 15) | (mn[..., 4:] & 15) << 4), -1)
    quants = (q[..., 0::2, :] | q[..., 1::2, :] << 4).reshape(layers, rows, cols // 256, 128)
    return torch.cat((d.view(torch.uint8), dmin.view(torch.uint8), packed, quants), -1).contiguous()


def frequencies(case):
    """Radians a position turns each pair by, in 64 bits, and what cos and sin are multiplied by."""
    r, rot = ROPES[case["rope"]], case["rot"] or SHAPES[case["shape"]][2]
    pair = torch.arange(rot // 2, dtype=torch.float64)
    f = r["freq_base"] ** (-2.0 * pair / rot)
    if r["scaling"] == "none":
        return f, 1.0
    if r["scaling"] == "linear":
        return f / r["factor"], 1.0
    if r["scaling"] == "bands":  # by the turns that a pair makes in the context the model was trained on
        keep = ((r["original_ctx"] * f / (2 * math.pi) - r["low"]) / (r["high"] - r["low"])).clamp(0.0, 1.0)
        return f * keep + f / r["factor"] * (1 - keep), 1.0
    edge = [rot * math.log(r["original_ctx"] / (b * 2 * math.pi)) / (2 * math.log(r["freq_base"])) for b in (r["high"], r["low"])]
    first, last = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), rot - 1)
    ramp = ((pair - first) / max(last - first, 0.001)).clamp(0.0, 1.0)
    return f * (1 - ramp) + f / r["factor"] * ramp, 0.1 * math.log(r["factor"]) + 1.0


def rope_positions(case):
    """Rows of a rope case: the end of a context, as a chunk of it comes."""
    return np.arange(case["far"] - case["rows"], case["far"], dtype=np.int32)


def _where(case):
    """The storage row of each new row in one layer's storage."""
    n, past = lengths(case), pasts(case)
    owner = np.repeat(np.arange(len(n)), n)
    pos = np.concatenate([np.arange(p, p + m) for p, m in zip(past, n)])
    if case["paged"]:
        return page_table(case)[0][owner, pos // PAGE].astype(np.int64) * PAGE + pos % PAGE
    return owner.astype(np.int64) * case["layers"] * (slots(case) // case["batch"]) + pos


def layer_rows(case):
    """From a row of one layer's storage to the same row of the next layer's."""
    return slots(case) if case["paged"] else slots(case) // case["batch"]


def stored(case, seed):
    """K and V [layers, slots, kv_dim] that the storage of a layer case holds before the step."""
    _, n_kv, d, _ = SHAPES[case["shape"]]
    return [_normal(seed, what, (case["layers"], slots(case), n_kv * d)) for what in (51, 52)]


def prepare(case, seed):
    s = {"case": case}
    layers = case["layers"]
    dev = {"device": "cuda"}
    if case["kind"] == "proj":
        s["raw"] = weights(seed, 1, case["fmt"], layers, case["rows"], case["cols"])
        s["x"] = _normal(seed, 2, (layers, case["n_vec"], case["cols"]))
    else:
        n_heads, n_kv, d, width = SHAPES[case["shape"]]
        freq, s["amp"] = frequencies(case)
        s["freq"] = freq.cuda()
        if case["kind"] == "rope":
            s["pos"] = torch.from_numpy(rope_positions(case)).cuda()
            s["x"] = _normal(seed, 2, (layers, case["rows"], n_heads, d))
        else:
            n = sum(lengths(case))
            s["n"] = n
            s["q_start"] = torch.tensor([0] + list(np.cumsum(lengths(case))), dtype=torch.int32, **dev)
            s["offset"] = torch.tensor(pasts(case), dtype=torch.int32, **dev)
            if case["paged"]:
                table, pages = page_table(case)
                s["table"] = torch.from_numpy(np.stack([table + layer * pages for layer in range(layers)])).cuda()
            if case["kind"] == "append":
                s["qkv"] = _normal(seed, 2, (layers, n, (n_heads + 2 * n_kv) * d))
            else:
                s["x"] = _normal(seed, 2, (layers, n, width))
                s["raw_qkv"] = weights(seed, 3, case["qkv"], layers, (n_heads + 2 * n_kv) * d, width)
                s["raw_out"] = weights(seed, 4, case["out"], layers, width, n_heads * d)
            if not own:
                full = (layers * slots(case), n_kv * d)
                if case["kind"] == "layer":
                    s["k"], s["v"] = (t.reshape(full) for t in stored(case, seed))
                elif case["dtype"] == "f32":
                    s["k"], s["v"] = torch.zeros(full, **dev), torch.zeros(full, **dev)
                else:
                    s["k"], s["v"] = ((torch.zeros((full[0], full[1] // 32, 32), dtype=torch.int8, **dev),
                                       torch.zeros((full[0], full[1] // 32), dtype=torch.float16, **dev)) for _ in "kv")
    if own:
        _prepare_own(s, seed)
    torch.cuda.synchronize()
    return s


# ------------------------------------------------------------------ the framework's calls

def _devs(t):
    return [Dev(x) for x in t]


def _handles(raw, fmt, rows, cols):
    return [backend().create_q4_weights(w.cpu().numpy(), rows, cols, fmt) for w in raw]


def _prepare_own(s, seed):
    be, case = backend(), s["case"]
    layers = case["layers"]
    if case["kind"] == "proj":
        s["w"] = _handles(s["raw"], case["fmt"], case["rows"], case["cols"])
        s["y"] = torch.zeros((layers, case["n_vec"], case["rows"]), device="cuda")
        s["xd"], s["yd"] = _devs(s["x"]), _devs(s["y"])
    else:
        n_heads, n_kv, d, width = SHAPES[case["shape"]]
        s["plan"] = be.create_rope_plan(d, rot_dim=case["rot"] or d, layout="half" if case["half"] else "interleaved",
                                        **ROPES[case["rope"]])
        if case["kind"] == "rope":
            s["out"] = torch.zeros_like(s["x"])
            s["xd"], s["outd"], s["posd"] = _devs(s["x"]), _devs(s["out"]), Dev(s["pos"])
        else:
            n, kv_dim = s["n"], n_kv * d
            if case["paged"]:
                s["kv"] = be.create_page_pool(layers * slots(case) // PAGE, n_kv, d, case["dtype"])
                s["tabled"], s["stride"] = _devs(s["table"]), s["table"].shape[2]
            else:
                s["kv"] = be.create_kv_cache(layers, slots(case) // case["batch"], n_kv, d, case["dtype"], n_seqs=case["batch"])
            s["qs"], s["off"] = Dev(s["q_start"]), Dev(s["offset"])
            s["q"] = torch.zeros((layers, n, n_heads, d), device="cuda")
            s["qd"] = _devs(s["q"])
            if case["kind"] == "layer":
                s["qkv"] = torch.zeros((layers, n, (n_heads + 2 * n_kv) * d), device="cuda")
            s["parts"] = [(Dev(t), Dev(t[:, n_heads * d:]), Dev(t[:, n_heads * d + kv_dim:])) for t in s["qkv"]]
            if case["kind"] == "append":
                where = torch.from_numpy(np.stack([_where(case) + layer * layer_rows(case) for layer in range(layers)])).cuda()
                s["k"], s["v"] = (torch.zeros((layers, n, kv_dim), device="cuda") for _ in "kv")
                s["at"], s["kd"], s["vd"] = _devs(where), _devs(s["k"]), _devs(s["v"])
            else:
                k, v = stored(case, seed)
                rows = torch.arange(layers * slots(case), device="cuda")
                torch.cuda.synchronize()
                s["kv"].write_rows_device(Dev(rows), Dev(k), Dev(v), len(rows))
                be.sync()
                s["w_qkv"] = _handles(s["raw_qkv"], case["qkv"], (n_heads + 2 * n_kv) * d, width)
                s["w_out"] = _handles(s["raw_out"], case["out"], width, n_heads * d)
                s["out"] = torch.zeros((layers, n, n_heads, d), device="cuda")
                s["y"] = torch.zeros((layers, n, width), device="cuda")
                s["xd"], s["qkvd"], s["outd"], s["yd"] = (_devs(s[k]) for k in ("x", "qkv", "out", "y"))
                s["len"] = np.array(pasts(case), np.int32) + 1
                s["start"] = np.zeros_like(s["len"])
                s["lend"], s["startd"] = (Dev(torch.from_numpy(s[k]).cuda()) for k in ("len", "start"))
    torch.cuda.synchronize()
    if case["graph"]:
        _step(s)  # sizes the scratch
        be.sync()
        s["graph"] = be.capture(lambda: _step(s))


def _append(s, layer):
    case = s["case"]
    n_heads, n_kv, d, _ = SHAPES[case["shape"]]
    q, k, v = s["parts"][layer]
    width = (n_heads + 2 * n_kv) * d
    pages = {"page_table": s["tabled"][layer], "page_table_stride": s["stride"]} if case["paged"] else {"layer": layer}
    backend().append(s["kv"], k, v, s["qs"], s["off"], case["batch"], case["hi"], rope=s["plan"], k_stride=width,
                     v_stride=width, q=q, q_stride=width, q_out=s["qd"][layer], n_heads=n_heads, **pages)


def _step(s):
    be, case = backend(), s["case"]
    for layer in range(case["layers"]):
        if case["kind"] == "proj":
            be.matvec_q4(s["w"][layer], s["xd"][layer], case["n_vec"], s["yd"][layer])
        elif case["kind"] == "rope":
            be.rope_rows(s["plan"], s["xd"][layer], case["rows"], SHAPES[case["shape"]][0], s["posd"], out=s["outd"][layer])
        elif case["kind"] == "append":
            _append(s, layer)
            s["kv"].read_rows_device(s["at"][layer], s["kd"][layer], s["vd"][layer], s["n"])
        else:
            n_heads, _, d, _ = SHAPES[case["shape"]]
            be.matvec_q4(s["w_qkv"][layer], s["xd"][layer], s["n"], s["qkvd"][layer])
            _append(s, layer)
            host = {} if case["graph"] else {"kv_start_host": s["start"], "kv_len_host": s["len"]}
            be.decode(s["kv"], s["qd"][layer], s["outd"][layer], s["startd"], s["lend"], case["batch"], int(s["len"].max()),
                      n_heads, 1.0 / math.sqrt(d), page_table=s["tabled"][layer], page_table_stride=s["stride"], **host)
            be.matvec_q4(s["w_out"][layer], s["outd"][layer], s["n"], s["yd"][layer])


# ------------------------------------------------------------------ the plain forms

def _dequantize(raw, fmt):
    """f32 weights [layers, rows, cols] of GGML bytes."""
    halves = raw[..., :2 if fmt == "q4_0" else 4].contiguous().view(torch.float16).float()
    if fmt == "q4_0":
        q = torch.cat((raw[..., 2:] & 15, raw[..., 2:] >> 4), -1)
        return ((q.float() - 8.0) * halves).flatten(2)
    a, b, c = raw[..., 4:8], raw[..., 8:12], raw[..., 12:16]
    sc = torch.cat((a & 63, (c & 15) | (a >> 6 << 4)), -1).float() * halves[..., :1]
    mn = torch.cat((b & 63, (c >> 4) | (b >> 6 << 4)), -1).float() * halves[..., 1:]
    q = raw[..., 16:].unflatten(-1, (4, 1, 32))
    q = torch.cat((q & 15, q >> 4), -2).flatten(-3, -2).float()
    return (q * sc.unsqueeze(-1) - mn.unsqueeze(-1)).flatten(2)


def _project(x, raw, fmt):
    return torch.matmul(x, _dequantize(raw, fmt).transpose(1, 2))


def _turns(s, pos):
    """cos and sin [rows, 1, pairs] of the positions' angles, in 64 bits."""
    angle = pos.double().unsqueeze(-1) * s["freq"]
    return (torch.cos(angle) * s["amp"]).unsqueeze(-2), (torch.sin(angle) * s["amp"]).unsqueeze(-2)


def _rotate(x, cos, sin, half):
    """x [..., rows, heads, d] with its first 2 * pairs dimensions rotated."""
    n = cos.shape[-1]
    a, b = (x[..., :n], x[..., n:2 * n]) if half else (x[..., 0:2 * n:2], x[..., 1:2 * n:2])
    turned = (a * cos - b * sin, a * sin + b * cos)
    return torch.cat((torch.cat(turned, -1) if half else torch.stack(turned, -1).flatten(-2), x[..., 2 * n:]), -1)


def _rounded(x):
    """(quants, f16 scales) of f32 rows [..., kv_dim] by the quantiser's rules: the scale is max|x| / 127 (1 for an empty
    block), the quant x times its inverse, rounded half away from zero."""
    b = x.unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True)
    one = torch.ones_like(top)
    d = torch.where(top > 0, top / (127.0 * one), one)  # a tensor divisor: a plain number would become a product
    r = b * (one / d)
    q = torch.trunc(r)
    q = (q + torch.where((r - q).abs() >= 0.5, torch.sign(r), torch.zeros_like(r))).clamp_(-127.0, 127.0)
    return q.to(torch.int8), d.squeeze(-1).half()


def _append_plain(s, qkv):
    """Rotates and stores the rows; the rotated queries, and the storage row of each new row."""
    case = s["case"]
    n_heads, n_kv, d, _ = SHAPES[case["shape"]]
    layers, n = case["layers"], s["n"]
    row = torch.arange(n, device="cuda")
    owner = torch.searchsorted(s["q_start"], row.int(), right=True) - 1
    pos = s["offset"][owner].long() + row - s["q_start"][owner]
    if case["paged"]:
        at = s["table"][:, owner, pos // PAGE].long() * PAGE + pos % PAGE
    else:
        seq = slots(case) // case["batch"]
        at = (owner * layers + torch.arange(layers, device="cuda").unsqueeze(1)) * seq + pos
    cos, sin = _turns(s, pos)
    heads = qkv.reshape(layers, n, n_heads + 2 * n_kv, d)
    q = _rotate(heads[:, :, :n_heads], cos.float(), sin.float(), case["half"])
    k = heads[:, :, n_heads:n_heads + n_kv]
    if case["dtype"] == "q8":  # in 64 bits and rounded once: values next to a quant's border
        k = _rotate(k.double(), cos, sin, case["half"]).float().flatten(2)
    else:
        k = _rotate(k, cos.float(), sin.float(), case["half"]).flatten(2)
    v = heads[:, :, n_heads + n_kv:].flatten(2)
    if case["dtype"] == "q8":
        kq, ks = _rounded(k)
        vq, vs = _rounded(v)
        s["k"][0][at], s["k"][1][at], s["v"][0][at], s["v"][1][at] = kq, ks, vq, vs
    else:
        s["k"][at], s["v"][at] = k, v
    return q, at


def _held(store, at):
    """The values of storage rows."""
    if isinstance(store, tuple):
        return (store[0][at].float() * store[1][at].float().unsqueeze(-1)).flatten(-2)
    return store[at]


def _attend(s, q):
    """One token of each sequence over its pages: [layers, batch, heads, d]."""
    case = s["case"]
    n_heads, n_kv, d, _ = SHAPES[case["shape"]]
    table = s["table"].long()
    at = (table.unsqueeze(-1) * PAGE + torch.arange(PAGE, device="cuda")).flatten(2)
    k = s["k"][at].unflatten(-1, (n_kv, d)).permute(0, 1, 3, 2, 4)
    v = s["v"][at].unflatten(-1, (n_kv, d)).permute(0, 1, 3, 2, 4)
    t = torch.matmul(q.unflatten(2, (n_kv, -1)), k.transpose(-1, -2)) / math.sqrt(d)
    hidden = torch.arange(at.shape[2], device="cuda") > s["offset"].reshape(-1, 1, 1, 1)
    t = t.masked_fill(hidden, -math.inf)
    p = torch.exp(t - t.amax(-1, keepdim=True))
    return torch.matmul(p / p.sum(-1, keepdim=True), v).flatten(2, 3)


def _run_plain(s):
    case = s["case"]
    if case["kind"] == "proj":
        return {"y": _project(s["x"], s["raw"], case["fmt"])}
    if case["kind"] == "rope":
        cos, sin = _turns(s, s["pos"])
        return {"out": _rotate(s["x"], cos.float(), sin.float(), case["half"])}
    if case["kind"] == "append":
        q, at = _append_plain(s, s["qkv"])
        return {"q": q, "k": _held(s["k"], at), "v": _held(s["v"], at)}
    qkv = _project(s["x"], s["raw_qkv"], case["qkv"])
    q, _ = _append_plain(s, qkv)
    out = _attend(s, q)
    return {"qkv": qkv, "q": q, "out": out, "y": _project(out.flatten(2), s["raw_out"], case["out"])}


def run(state):
    if not own:
        return _run_plain(state)
    if "graph" in state:
        state["graph"].replay()
    else:
        _step(state)
    names = {"proj": ("y",), "rope": ("out",), "append": ("q", "k", "v"), "layer": ("qkv", "q", "out", "y")}
    return {k: state[k] for k in names[state["case"]["kind"]]}


# ------------------------------------------------------------------ the same in 64 bits

def _weights64(raw, fmt):
    """One matrix's f64 values, block by block of the format."""
    raw = raw.cpu().numpy()
    rows, blocks, size = raw.shape
    if fmt == "q4_0":
        d = raw[..., :2].copy().view(np.float16).astype(np.float64)
        out = np.empty((rows, blocks, 32))
        out[..., :16] = (raw[..., 2:] % 16).astype(np.float64) - 8
        out[..., 16:] = (raw[..., 2:] // 16).astype(np.float64) - 8
        out *= d
    else:
        d, dmin = (raw[..., i:i + 2].copy().view(np.float16).astype(np.float64)[..., 0] for i in (0, 2))
        bits = raw[..., 4:16].astype(np.int64)
        out = np.empty((rows, blocks, 8, 32))
        for j in range(8):
            if j < 4:
                sc, mn = bits[..., j] % 64, bits[..., j + 4] % 64
            else:
                sc = bits[..., j + 4] % 16 + 16 * (bits[..., j - 4] // 64)
                mn = bits[..., j + 4] // 16 + 16 * (bits[..., j] // 64)
            q = raw[..., 16 + 32 * (j // 2):48 + 32 * (j // 2)]
            q = q // 16 if j % 2 else q % 16
            out[..., j, :] = (d * sc)[..., None] * q - (dmin * mn)[..., None]
    return torch.from_numpy(out.reshape(rows, -1)).cuda()


def _frequencies64(case):
    """(frequency of each pair, the amplitude), pair by pair."""
    r, rot = ROPES[case["rope"]], case["rot"] or SHAPES[case["shape"]][2]
    rule, got = r["scaling"], []
    for p in range(rot // 2):
        f = math.exp(-math.log(r["freq_base"]) * 2 * p / rot)
        slow = f / r.get("factor", 1.0)
        if rule == "linear":
            f = slow
        elif rule == "bands":
            turns = r["original_ctx"] * f / (2 * math.pi)
            if turns < r["low"]:
                f = slow
            elif turns <= r["high"]:
                t = (turns - r["low"]) / (r["high"] - r["low"])
                f = (1 - t) * slow + t * f
        elif rule == "yarn":
            def pair_of(turns):
                return rot / 2 * math.log(r["original_ctx"] / (2 * math.pi * turns), r["freq_base"])
            a, b = max(0, math.floor(pair_of(r["high"]))), min(rot - 1, math.ceil(pair_of(r["low"])))
            t = min(1.0, max(0.0, (p - a) / max(b - a, 0.001)))
            f = (1 - t) * f + t * slow
        got.append(f)
    return np.array(got), 1.0 + 0.1 * math.log(r["factor"]) if rule == "yarn" else 1.0


def _rotate64(x, pos, case):
    """x [rows, heads, d] f64 at the positions [rows], as complex numbers."""
    f, amp = _frequencies64(case)
    n = len(f)
    angle = torch.from_numpy(np.asarray(pos, np.float64)[:, None] * f).cuda()
    turn = torch.polar(torch.full_like(angle, amp), angle).unsqueeze(1)
    first, second = (slice(0, n), slice(n, 2 * n)) if case["half"] else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turn
    out = x.clone()
    out[..., first], out[..., second] = z.real, z.imag
    return out


def _held64(x, case):
    """f64 values that the storage holds of rows, which reach it in f32; Q8_0's scale and quants are defined in f32."""
    if case["dtype"] == "f32":
        return x
    b = x.float().double().reshape(x.shape[0], -1, 32)
    top = b.abs().max(-1, keepdim=True).values
    d = torch.where(top > 0, (top / 127).float().double(), torch.ones_like(top))
    r = (b * (1 / d).float().double()).float().double()
    q = (torch.sign(r) * torch.floor(r.abs() + 0.5)).clamp(-127, 127)
    return (q * d.half().double()).reshape(x.shape)


def exact(case, seed):
    layers = case["layers"]
    if case["kind"] == "proj":
        raw = weights(seed, 1, case["fmt"], layers, case["rows"], case["cols"])
        x = _normal(seed, 2, (layers, case["n_vec"], case["cols"])).double()
        return {"y": torch.stack([x[i] @ _weights64(raw[i], case["fmt"]).T.contiguous() for i in range(layers)])}
    n_heads, n_kv, d, width = SHAPES[case["shape"]]
    if case["kind"] == "rope":
        x = _normal(seed, 2, (layers, case["rows"], n_heads, d)).double()
        return {"out": torch.stack([_rotate64(t, rope_positions(case), case) for t in x])}
    n = sum(lengths(case))
    pos = np.concatenate([p + np.arange(m) for p, m in zip(pasts(case), lengths(case))])
    got = {}

    def put(**outs):
        for name, t in outs.items():
            got.setdefault(name, []).append(t)

    def split(rows):
        heads = rows.reshape(n, -1, d)
        return (_rotate64(heads[:, :n_heads], pos, case), _rotate64(heads[:, n_heads:n_heads + n_kv], pos, case).reshape(n, -1),
                heads[:, n_heads + n_kv:].reshape(n, -1))

    if case["kind"] == "append":
        for rows in _normal(seed, 2, (layers, n, (n_heads + 2 * n_kv) * d)).double():
            q, k, v = split(rows)
            put(q=q, k=_held64(k, case), v=_held64(v, case))
        return {name: torch.stack(t) for name, t in got.items()}
    x = _normal(seed, 2, (layers, n, width)).double()
    raw_qkv = weights(seed, 3, case["qkv"], layers, (n_heads + 2 * n_kv) * d, width)
    raw_out = weights(seed, 4, case["out"], layers, width, n_heads * d)
    k_all, v_all = stored(case, seed)
    table, _ = page_table(case)
    for i in range(layers):
        rows = x[i] @ _weights64(raw_qkv[i], case["qkv"]).T.contiguous()
        q, k, v = split(rows)
        out = torch.empty_like(q)
        for b, past in enumerate(pasts(case)):
            at = torch.from_numpy(table[b, np.arange(past) // PAGE].astype(np.int64) * PAGE + np.arange(past) % PAGE).cuda()
            keys = torch.cat((k_all[i][at].double(), k[b:b + 1])).reshape(-1, n_kv, d)
            vals = torch.cat((v_all[i][at].double(), v[b:b + 1])).reshape(-1, n_kv, d)
            for h in range(n_heads):
                p = torch.softmax(keys[:, h * n_kv // n_heads] @ q[b, h] / math.sqrt(d), 0)
                out[b, h] = p @ vals[:, h * n_kv // n_heads]
        put(qkv=rows, q=q, out=out, y=out.reshape(n, -1) @ _weights64(raw_out[i], case["out"]).T.contiguous())
    return {name: torch.stack(t) for name, t in got.items()}
