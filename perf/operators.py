"""Operators of a prompt that is taken in chunks, over a paged key/value cache, as measurable cases.

  write    rope_kv_paged: head norm and rotation of a chunk's queries and keys, keys and values into the pages of their
           sequences, as bf16 or as int8 with a scale for each token and head
  read     kv_read_paged: ranges of tokens of the cache as dense bf16 rows
  attend   attn_paged: the chunk's queries against the pages, causal, with a sliding window and first tokens that stay visible
  product  gemv_w8: the rows of a chunk against int8 weights with a scale for each output channel

A chunk is a ragged batch: rows `row_start[s]` to `row_start[s + 1]` are the new tokens of sequence s, which follow `context[s]`
tokens of it; rows behind the last sequence are padding. Page i of a sequence is page `page_table[s, i]` of the cache.

`run` computes the operators in torch (fp32, rounded once), or, where `own` is true, through the framework's public entry points.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

# ---- cases ------------------------------------------------------------------------------------------------------

_GEMMA = {"n_q": 4, "n_kv": 1, "d": 256}     # the decoder workload's heads
_GROUPED = {"n_q": 32, "n_kv": 8, "d": 128}  # eight groups of four, as decoders of a few billion weights have


def listed():
    return [
        # one user's next token: one row of q/k/v into the cache, where a launch is all there is
        {"name": "write one token", "kind": "write", **_GEMMA, "seqs": 1, "rows": 1, "ctx": 1000, "page": 16, "cache": "bf16", "norm": True, "pad": 0, "even": True},
        # prompts of several users in one chunk, into an int8 cache, and read back as a transfer to another cache does
        {"name": "write and read 5 prompts", "kind": "write", **_GROUPED, "seqs": 5, "rows": 4001, "ctx": 3000, "page": 32, "cache": "i8", "norm": True, "pad": 31, "even": False},
        # the largest chunk: one long prompt of the decoder workload, heads without norms
        {"name": "write 16384 rows", "kind": "write", **_GEMMA, "seqs": 1, "rows": 16384, "ctx": 0, "page": 64, "cache": "bf16", "norm": False, "pad": 0, "even": True},
        # three sequences leave an int8 cache
        {"name": "read 3 sequences", "kind": "read", **_GEMMA, "seqs": 3, "rows": 20011, "ctx": 0, "page": 16, "cache": "i8", "pad": 0, "even": False},
        # decode: one user behind a 1024-token prompt; the smallest call
        {"name": "attend one token", "kind": "attend", **_GEMMA, "seqs": 1, "rows": 1, "ctx": 1024, "page": 16, "cache": "bf16", "window": 0, "sinks": 0, "pad": 0, "even": True},
        # decode of 32 users with contexts of all lengths, int8 cache
        {"name": "attend 32 users int8", "kind": "attend", **_GROUPED, "seqs": 32, "rows": 32, "ctx": 8000, "page": 32, "cache": "i8", "window": 0, "sinks": 0, "pad": 0, "even": False},
        # decode of 48 users through a local layer: a window of 512 and four first tokens
        {"name": "attend 48 windows", "kind": "attend", **_GEMMA, "seqs": 48, "rows": 48, "ctx": 9000, "page": 16, "cache": "bf16", "window": 512, "sinks": 4, "pad": 0, "even": False},
        # a prompt of the decoder workload in one chunk, a global layer
        {"name": "attend prompt 4096", "kind": "attend", **_GEMMA, "seqs": 1, "rows": 4096, "ctx": 0, "page": 64, "cache": "bf16", "window": 0, "sinks": 0, "pad": 0, "even": True},
        # five users' chunks behind contexts of different lengths, int8 cache
        {"name": "attend 5 chunks int8", "kind": "attend", **_GROUPED, "seqs": 5, "rows": 1999, "ctx": 7000, "page": 32, "cache": "i8", "window": 0, "sinks": 0, "pad": 49, "even": False},
        # a long prompt through a local layer of heads of 64: window and first tokens
        {"name": "attend window 8192", "kind": "attend", "n_q": 16, "n_kv": 2, "d": 64, "seqs": 1, "rows": 8192, "ctx": 0, "page": 16, "cache": "bf16", "window": 512, "sinks": 4, "pad": 0, "even": True},
        # a short prompt's attention product (the decoder workload's q/k/v weights)
        {"name": "product 77 x 1536 x 1152", "kind": "product", "rows": 77, "n": 1536, "k": 1152, "f32": False},
        # a chunk of a long prompt through the gate and up weights
        {"name": "product 4000 x 13824 x 1152", "kind": "product", "rows": 4000, "n": 13824, "k": 1152, "f32": False},
    ]


def _log(rng, lo, hi, multiple=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999)))
    return int(min(hi, max(lo, multiple * max(1, round(v / multiple)) if multiple > 1 else int(v))))


def draw(rng):
    kind = rng.choice(["write", "read", "attend", "attend", "attend", "product"])
    if kind == "product":
        c = {"kind": kind, "rows": _log(rng, 33, 4000), "n": _log(rng, 200, 13824), "k": _log(rng, 64, 6912, 16), "f32": rng.random() < 0.25}
        while work(c)["flops"] > 1.2e11:
            c["rows"] = (c["rows"] + 1) // 2
        return c
    n_kv = rng.choice([1, 1, 2, 4, 8])
    c = {"kind": kind, "n_q": n_kv * rng.choice([1, 2, 4, 4, 8, 3]), "n_kv": n_kv, "d": rng.choice([64, 128, 128, 256, 256, 80, 96, 192]),
         "seqs": _log(rng, 1, 48), "page": rng.choice([8, 16, 16, 32, 64, 128, 24]), "cache": rng.choice(["bf16", "i8"]), "pad": rng.choice([0, 0, 5, 40]),
         "even": rng.random() < 0.3}
    if kind == "write":
        c |= {"rows": _log(rng, c["seqs"], 6000), "ctx": _log(rng, 1, 20000), "norm": rng.random() < 0.5}
    elif kind == "read":
        c |= {"rows": _log(rng, c["seqs"], 20000), "ctx": rng.choice([0, 0, 1000])}
    else:
        c |= {"window": rng.choice([0, 0, _log(rng, 16, 4096)]), "ctx": _log(rng, 1, 16000)}
        c["sinks"] = rng.choice([0, 1, 4, 70]) if c["window"] else 0
        c["rows"] = c["seqs"] if rng.random() < 0.4 else _log(rng, c["seqs"], 4000)
        while c["n_q"] * c["seqs"] * _most(c) * (c["ctx"] + _most(c)) > 1.1e9:  # what the plain form holds at once
            c["rows"], c["ctx"] = max(c["seqs"], c["rows"] * 2 // 3), max(1, c["ctx"] * 2 // 3)
            if c["rows"] == c["seqs"] and c["ctx"] < 500:
                c["n_q"] = c["n_kv"]
    while c["seqs"] * (c["ctx"] + _most(c)) * c["n_kv"] * c["d"] > 6.5e7 or work(c)["flops"] > 1.2e11:
        c["ctx"], c["rows"] = c["ctx"] * 2 // 3, max(c["seqs"], c["rows"] * 4 // 5)
    return c


def _lengths(c):
    """New tokens and context of each sequence: even, or spread over a factor of about eight."""
    rng = random.Random(c["rows"] * 31 + c["seqs"])
    if c["even"] or c["seqs"] == 1:
        share = [1.0] * c["seqs"]
    else:
        share = [math.exp(rng.uniform(-1.05, 1.05)) for _ in range(c["seqs"])]
    free, total = c["rows"] - c["seqs"], sum(share)
    new = [1 + int(free * s / total) for s in share]
    new[0] += c["rows"] - sum(new)
    if c["kind"] == "read":
        return new, [c["ctx"]] * c["seqs"]
    ctx = [c["ctx"] if c["even"] or c["seqs"] == 1 else int(c["ctx"] * math.exp(rng.uniform(-2.1, 0.0))) for _ in range(c["seqs"])]
    return new, ctx


def _most(c):
    return max(_lengths(c)[0])


# ---- inputs -----------------------------------------------------------------------------------------------------

def _theta(c):
    return 1.0e6 if c["d"] != 256 else 1.0e4


class _State(dict):
    """What a program holds: tensors, and with the framework the loaded executable and the bindings of its buffers."""

    def close(self):
        for b in self.pop("bound", []):
            b.free()
        ex = self.pop("ex", None)
        if ex is not None:
            ex.destroy()

    __del__ = close


def prepare(case, seed):
    c = case
    gen = torch.Generator("cuda").manual_seed(seed)

    def normal(*shape, std=1.0):
        return (torch.randn(shape, device="cuda", generator=gen) * std).to(torch.bfloat16)

    s = _State(c=c)
    if c["kind"] == "product":
        # activations behind a norm; weights uniform over int8, scales that keep the result's spread near one
        s["x"] = normal(c["rows"], c["k"])
        s["w"] = torch.randint(-127, 128, (c["n"], c["k"]), dtype=torch.int8, device="cuda", generator=gen)
        s["scale"] = ((0.8 + 0.45 * torch.rand(c["n"], device="cuda", generator=gen)) / (73.0 * math.sqrt(c["k"]))).to(torch.bfloat16)
        s["out"] = torch.zeros((c["rows"], c["n"]), dtype=torch.float32 if c["f32"] else torch.bfloat16, device="cuda")
        if own:
            _load(s)
        return s
    new, ctx = _lengths(c)
    rows, n_q, n_kv, d, page = c["rows"] + c["pad"], c["n_q"], c["n_kv"], c["d"], c["page"]
    per_seq = [-(-(a + b) // page) for a, b in zip(new, ctx)]
    table = torch.full((c["seqs"], max(per_seq)), -1, dtype=torch.int32)
    pages = sum(per_seq) + 3
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    at = 0
    for i, n in enumerate(per_seq):
        table[i, :n] = order[at:at + n]
        at += n
    s["row_start"] = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32).cuda()
    s["context"] = torch.tensor(ctx, dtype=torch.int32).cuda()
    s["table"], s["pages"] = table.cuda(), pages
    s["n"], s["nmax"], s["kmax"] = sum(new), max(new), max(a + b for a, b in zip(new, ctx))
    shape = (1, pages, page, n_kv * d)
    if c["cache"] == "bf16":
        s["k"], s["v"] = normal(*shape), normal(*shape)
    else:
        s["k"], s["v"] = (torch.randint(-127, 128, shape, dtype=torch.int8, device="cuda", generator=gen) for _ in range(2))
        s["scales"] = (0.5 + torch.rand((1, pages, page, 2 * n_kv), device="cuda", generator=gen)) / 73.0
    if c["kind"] == "write":
        s["qkv"] = normal(rows, (n_q + 2 * n_kv) * d)
        if c["norm"]:
            s["qw"], s["kw"] = normal(d, std=0.1), normal(d, std=0.1)
        s["q"] = torch.zeros((rows, n_q * d), dtype=torch.bfloat16, device="cuda")
    if c["kind"] == "attend":
        s["q"] = normal(rows, n_q * d, std=2.5)  # scores of unequal keys, as trained heads give
        s["out"] = torch.zeros_like(s["q"])
    if c["kind"] == "read" or (c["kind"] == "write" and c["cache"] == "i8"):
        s["k_out"], s["v_out"] = (torch.zeros((rows, n_kv * d), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    if own:
        _load(s)
    return s


# ---- the framework's operators ------------------------------------------------------------------------------------

_device = None


def _load(s):
    global _device
    for p in (os.getcwd(), os.path.join(os.getcwd(), "torq-compiler_b200")):
        if p not in sys.path:
            sys.path.insert(0, p)
    from torq_b200.oplist import Graph
    from torq_b200.runtime import Device, Executable
    if _device is None:
        _device = Device(0)
    c, g = s["c"], Graph()
    dtypes = {torch.bfloat16: "bf16", torch.int8: "i8", torch.int32: "i32", torch.float32: "f32"}
    ins = []

    def bind(*names):
        ins.extend(names)
        return [g.input(tuple(s[n].shape), dtypes[s[n].dtype]) for n in names]

    def bits(t):
        return t.view(torch.int16).cpu().numpy().view(np.uint16)

    if c["kind"] == "product":
        (x,) = bind("x")
        g.output(g.gemv_w8(x, s["w"].cpu().numpy(), bits(s["scale"]), out_dtype="f32" if c["f32"] else "bf16"))
        outs = ["out"]
    else:
        heads = {"n_kv": c["n_kv"], "head_dim": c["d"]}
        row_start, context, table, k, v = bind("row_start", "context", "table", "k", "v")
        if "scales" in s:
            (heads["scales"],) = bind("scales")
        if c["kind"] == "write":
            (qkv,) = bind("qkv")
            norms = (bits(s["qw"]), bits(s["kw"])) if c["norm"] else ()
            g.output(g.rope_kv_paged(qkv, row_start, context, table, k, v, *norms, n_q=c["n_q"], theta=_theta(c), eps=1e-6, **heads))
            outs = ["q"]
        elif c["kind"] == "attend":
            (q,) = bind("q")
            g.output(g.attn_paged(q, row_start, context, table, k, v, n_q=c["n_q"], scale=c["d"] ** -0.5, window=c["window"], sinks=c["sinks"],
                                  max_new=1 if c["rows"] == c["seqs"] else 0, **heads))
            outs = ["out"]
        else:
            outs = []
        if "k_out" in s:
            for t in g.kv_read_paged(row_start, context, table, k, v, rows=s["k_out"].shape[0], **heads):
                g.output(t)
            outs += ["k_out", "v_out"]
    s["ex"] = Executable(_device, g.serialize())
    s["ins"], s["outs"] = ([_device.import_pointer(s[n].data_ptr(), s[n].numel() * s[n].element_size()) for n in names] for names in (ins, outs))
    s["bound"] = s["ins"] + s["outs"]


# ---- the plain form ---------------------------------------------------------------------------------------------

def _row_places(s, dtype=torch.float32):
    """Of every new token: its sequence, its row within the sequence, its position."""
    row = torch.arange(s["n"], device="cuda")
    seq = torch.searchsorted(s["row_start"].long(), row, right=True) - 1
    within = row - s["row_start"].long()[seq]
    return seq, within, within + s["context"].long()[seq]


def _slots(s, seq, pos):
    page = s["c"]["page"]
    return s["table"].long()[seq, pos // page] * page + pos % page


def _plain_product(s):
    y = (s["x"].float() @ s["w"].float().T) * s["scale"].float()
    s["out"].copy_(y)
    return {"y": s["out"]}


def _plain_write(s):
    c = s["c"]
    n, n_q, n_kv, d = s["n"], c["n_q"], c["n_kv"], c["d"]
    seq, _, pos = _row_places(s)
    heads = s["qkv"][:n].float().view(n, n_q + 2 * n_kv, d)
    q, k, v = heads[:, :n_q], heads[:, n_q:n_q + n_kv], heads[:, n_q + n_kv:]
    if c["norm"]:
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + 1e-6) * (1.0 + s["qw"].float())
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + 1e-6) * (1.0 + s["kw"].float())
    half = d // 2
    freq = _theta(c) ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    angle = pos.double()[:, None] * freq  # far positions: 64 bits
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    q, k = (torch.cat([x[..., :half] * cos - x[..., half:] * sin, x[..., half:] * cos + x[..., :half] * sin], -1) for x in (q, k))
    s["q"][:n] = q.reshape(n, -1).to(torch.bfloat16)
    slot = _slots(s, seq, pos)
    pages_k, pages_v = s["k"].view(-1, n_kv, d), s["v"].view(-1, n_kv, d)
    if c["cache"] == "bf16":
        pages_k[slot], pages_v[slot] = k.to(torch.bfloat16), v.to(torch.bfloat16)
        return {"q": s["q"], "k": s["k"], "v": s["v"]}
    scales = torch.cat([k.abs().amax(-1), v.abs().amax(-1)], -1) / 127.0
    inverse = torch.where(scales > 0, 1.0 / scales, torch.zeros_like(scales))[..., None]
    pages_k[slot] = (k * inverse[:, :n_kv]).round().clamp(-127, 127).to(torch.int8)
    pages_v[slot] = (v * inverse[:, n_kv:]).round().clamp(-127, 127).to(torch.int8)
    s["scales"].view(-1, 2 * n_kv)[slot] = scales
    return {"q": s["q"], "scales": s["scales"], **_plain_read(s)}


def _plain_read(s):
    c = s["c"]
    n, n_kv, d = s["n"], c["n_kv"], c["d"]
    seq, _, pos = _row_places(s)
    slot = _slots(s, seq, pos)
    k, v = (s[x].view(-1, n_kv, d)[slot].float() for x in "kv")
    if c["cache"] == "i8":
        scale = s["scales"].view(-1, 2 * n_kv)[slot][..., None]
        k, v = k * scale[:, :n_kv], v * scale[:, n_kv:]
    s["k_out"][:n], s["v_out"][:n] = k.reshape(n, -1).to(torch.bfloat16), v.reshape(n, -1).to(torch.bfloat16)
    return {"k_read": s["k_out"], "v_read": s["v_out"]}


def _plain_attend(s):
    c = s["c"]
    n, nmax, kmax, n_kv, d = s["n"], s["nmax"], s["kmax"], c["n_kv"], c["d"]
    group, seqs = c["n_q"] // n_kv, c["seqs"]
    seq, within, _ = _row_places(s)
    start, ctx = s["row_start"].long(), s["context"].long()
    # every sequence's queries and keys, padded to the longest
    j = torch.arange(nmax, device="cuda")
    rows = (start[:-1, None] + j).clamp(max=n - 1)
    q = s["q"].float().view(-1, n_kv, group, d)[rows].permute(0, 2, 1, 3, 4).reshape(seqs, n_kv, nmax * group, d)
    key = torch.arange(kmax, device="cuda")
    slot = (s["table"].long().clamp(min=0)[:, key // c["page"]] * c["page"] + key % c["page"])
    k, v = (s[x].view(-1, n_kv, d)[slot].float() for x in "kv")
    if c["cache"] == "i8":
        scale = s["scales"].view(-1, 2 * n_kv)[slot][..., None]
        k, v = k * scale[:, :, :n_kv], v * scale[:, :, n_kv:]
    pos = (ctx[:, None] + j)[:, :, None]
    seen = key <= pos
    if c["window"]:
        seen = seen & ((key > pos - c["window"]) | (key < c["sinks"]))
    # keys behind a shorter sequence's end are other tokens' or nobody's: no query sees them
    score = (q @ k.permute(0, 2, 3, 1) * d ** -0.5).view(seqs, n_kv, nmax, group, kmax)
    score = score.masked_fill(~seen[:, None, :, None], -math.inf)
    p = (score - score.amax(-1, keepdim=True)).exp()
    del score
    out = (p.view(seqs, n_kv, nmax * group, kmax) @ v.permute(0, 2, 1, 3)) / p.sum(-1).view(seqs, n_kv, nmax * group, 1)
    out = out.view(seqs, n_kv, nmax, group, d).permute(0, 2, 1, 3, 4).reshape(seqs * nmax, -1)
    s["out"][:n] = out[seq * nmax + within].to(torch.bfloat16)
    return {"out": s["out"]}


def run(state):
    s = state
    kind = s["c"]["kind"]
    if not own:
        return {"product": _plain_product, "write": _plain_write, "read": _plain_read, "attend": _plain_attend}[kind](s)
    s["ex"].dispatch(s["ins"], s["outs"])
    if kind == "product":
        return {"y": s["out"]}
    if kind == "attend":
        return {"out": s["out"]}
    if kind == "read":
        return {"k_read": s["k_out"], "v_read": s["v_out"]}
    if s["c"]["cache"] == "bf16":
        return {"q": s["q"], "k": s["k"], "v": s["v"]}
    return {"q": s["q"], "scales": s["scales"], "k_read": s["k_out"], "v_read": s["v_out"]}


# ---- 64 bits ----------------------------------------------------------------------------------------------------

def exact(case, seed):
    """The definition in 64 bits, sequence by sequence."""
    c, s = case, prepare(case, seed)
    if c["kind"] == "product":
        return {"y": s["x"].double() @ s["w"].double().T * s["scale"].double()}
    n_q, n_kv, d, page = c["n_q"], c["n_kv"], c["d"], c["page"]
    starts, ctxs, table = s["row_start"].tolist(), s["context"].tolist(), s["table"].tolist()
    slots = []  # per sequence: where each of its tokens lies
    for i, ctx in enumerate(ctxs):
        end = ctx + starts[i + 1] - starts[i]
        slots.append(torch.tensor([table[i][t // page] * page + t % page for t in range(end)], device="cuda"))

    def tokens(name, i, cols):
        x = s[name].view(-1, n_kv, d)[slots[i]].double()
        return x if c["cache"] == "bf16" else x * s["scales"].view(-1, 2 * n_kv)[slots[i]][:, cols].double()[..., None]

    k_cols, v_cols = slice(0, n_kv), slice(n_kv, 2 * n_kv)
    if c["kind"] == "read":
        k, v = (torch.zeros_like(s["k_out"], dtype=torch.float64) for _ in range(2))
        for i, ctx in enumerate(ctxs):
            k[starts[i]:starts[i + 1]] = tokens("k", i, k_cols)[ctx:].flatten(1)
            v[starts[i]:starts[i + 1]] = tokens("v", i, v_cols)[ctx:].flatten(1)
        return {"k_read": k, "v_read": v}
    if c["kind"] == "attend":
        if sum((b - a) * (b - a + ctx) for a, b, ctx in zip(starts, starts[1:], ctxs)) * n_q * d > 4e12:
            return None
        out = torch.zeros_like(s["out"], dtype=torch.float64)
        for i, ctx in enumerate(ctxs):
            a, b = starts[i], starts[i + 1]
            k, v = tokens("k", i, k_cols), tokens("v", i, v_cols)
            p, t = torch.arange(ctx, ctx + b - a, device="cuda")[:, None], torch.arange(ctx + b - a, device="cuda")
            hidden = t > p
            if c["window"]:
                hidden |= (t <= p - c["window"]) & (t >= c["sinks"])
            for h in range(n_q):
                kv = h // (n_q // n_kv)
                w = s["q"][a:b, h * d:(h + 1) * d].double() @ k[:, kv].T / math.sqrt(d)
                out[a:b, h * d:(h + 1) * d] = torch.softmax(w.masked_fill(hidden, -math.inf), -1) @ v[:, kv]
        return {"out": out}
    q_out = torch.zeros_like(s["q"], dtype=torch.float64)
    cached = {x: s[x].view(-1, n_kv, d).double() for x in "kv"} if c["cache"] == "bf16" else {}
    read = {x: torch.zeros(s["q"].shape[0], n_kv * d, dtype=torch.float64, device="cuda") for x in "kv"}
    scales = s["scales"].view(-1, 2 * n_kv).double() if c["cache"] == "i8" else None
    turn = torch.tensor([_theta(c) ** (-2.0 * j / d) for j in range(d // 2)], dtype=torch.float64, device="cuda")
    for i, ctx in enumerate(ctxs):
        a, b = starts[i], starts[i + 1]
        x = s["qkv"][a:b].double().view(b - a, -1, d)
        if c["norm"]:
            w = torch.cat([s["qw"].double().expand(n_q, d), s["kw"].double().expand(n_kv, d)])
            y = x[:, :n_q + n_kv]
            y = y / (y.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * (1 + w)
        else:
            y = x[:, :n_q + n_kv]
        z = torch.complex(y[..., :d // 2], y[..., d // 2:])
        t = torch.arange(ctx, ctx + b - a, device="cuda", dtype=torch.float64)[:, None] * turn
        z = z * torch.polar(torch.ones_like(t), t)[:, None]
        y = torch.cat([z.real, z.imag], -1)
        q_out[a:b] = y[:, :n_q].flatten(1)
        for name, val, cols in (("k", y[:, n_q:], k_cols), ("v", x[:, n_q + n_kv:], v_cols)):
            here = slots[i][ctx:]
            if c["cache"] == "bf16":
                cached[name][here] = val
            else:
                step = val.abs().amax(-1) / 127
                scales[here, cols] = step
                read[name][a:b] = (torch.round(val / step.clamp(min=1e-300)[..., None]) * step[..., None]).flatten(1)
    if c["cache"] == "bf16":
        return {"q": q_out, "k": cached["k"].view(s["k"].shape), "v": cached["v"].view(s["v"].shape)}
    return {"q": q_out, "scales": scales.view(s["scales"].shape), "k_read": read["k"], "v_read": read["v"]}


# ---- what a pass cannot do without ------------------------------------------------------------------------------

def _visible(c, first, count, upto):
    """Keys that the tokens at positions first .. first + count - 1 see, in all; and how many different ones."""
    if not c["window"]:
        return sum(range(first + 1, first + count + 1)), upto
    seen = 0
    for p in range(first, first + count):
        w = min(p + 1, c["window"])
        seen += w + min(c["sinks"], p + 1 - w)
    near = min(upto, c["window"] + count - 1)
    return seen, near + min(c["sinks"], upto - near)


def work(case):
    c = case
    if c["kind"] == "product":
        return {"bytes": c["rows"] * c["k"] * 2 + c["n"] * (c["k"] + 2) + c["rows"] * c["n"] * (4 if c["f32"] else 2),
                "flops": 2 * c["rows"] * c["n"] * c["k"]}
    n_q, n_kv, d = c["n_q"], c["n_kv"], c["d"]
    row = n_kv * (2 * d * 2 if c["cache"] == "bf16" else 2 * d + 8)  # keys and values of a token in the cache
    if c["kind"] == "write":
        read_back = n_kv * d * 2 * 2 if c["cache"] == "i8" else 0
        return {"bytes": c["rows"] * ((n_q + 2 * n_kv) * d * 2 + n_q * d * 2 + row + read_back), "flops": c["rows"] * (n_q + n_kv) * d * 7}
    if c["kind"] == "read":
        return {"bytes": c["rows"] * (row + n_kv * d * 4), "flops": c["rows"] * n_kv * d * 2}
    pairs = keys = 0
    for new, ctx in zip(*_lengths(c)):
        a, b = _visible(c, ctx, new, ctx + new)
        pairs, keys = pairs + a, keys + b
    return {"bytes": keys * row + c["rows"] * n_q * d * 4, "flops": pairs * n_q * d * 4}
