"""A paged cache and a ragged batch with its operators in 64 bits, token by token (the definition, not an implementation to be fast)."""
from dataclasses import dataclass

import numpy as np

from torq_b200.bf16 import from_bf16, to_bf16


def bf16(rng, *shape, std=1.0):
    return to_bf16(rng.normal(0, std, shape).astype(np.float32))


@dataclass
class Batch:
    """`new` and `ctx` tokens of each sequence; `lead` and `pad` rows in front of the first and behind the last one."""
    new: list
    ctx: list
    n_q: int = 4
    n_kv: int = 1
    d: int = 256
    page: int = 16
    i8: bool = False
    layers: int = 1
    layer: int = 0
    pad: int = 0
    lead: int = 0
    spare_pages: int = 2
    seed: int = 1

    def __post_init__(self):
        rng = self.rng = np.random.default_rng(self.seed)
        self.seqs = len(self.new)
        self.row_start = (self.lead + np.concatenate([[0], np.cumsum(self.new)])).astype(np.int32)
        self.rows = int(self.row_start[-1]) + self.pad
        self.context = np.array(self.ctx, np.int32)
        need = [-(-(a + b) // self.page) for a, b in zip(self.new, self.ctx)]
        self.pages = sum(need) + self.spare_pages
        order = rng.permutation(self.pages).astype(np.int32)
        self.table = np.full((self.seqs, max(max(need), 1)), -1, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        shape = (self.layers, self.pages, self.page, self.n_kv * self.d)
        if self.i8:
            self.k, self.v = (rng.integers(-127, 128, shape).astype(np.int8) for _ in range(2))
            self.scales = rng.uniform(0.5, 1.5, shape[:3] + (2 * self.n_kv,)).astype(np.float32) / 73
        else:
            self.k, self.v = bf16(rng, *shape), bf16(rng, *shape)
            self.scales = None

    def slot(self, s, p):
        """(page, offset) of position p of sequence s, or None where it holds nothing."""
        i = p // self.page
        if p < 0 or i >= self.table.shape[1] or not 0 <= self.table[s, i] < self.pages:
            return None
        return int(self.table[s, i]), p % self.page

    def cached(self, which, s, count):
        """Values [count, n_kv, d] of a sequence's first tokens in 64 bits, and which of them the cache holds."""
        out, ok = np.zeros((count, self.n_kv, self.d)), np.zeros(count, bool)
        pages = self.k if which == "k" else self.v
        col = 0 if which == "k" else self.n_kv
        for p in range(count):
            at = self.slot(s, p)
            if at is None:
                continue
            ok[p] = True
            raw = pages[self.layer][at].reshape(self.n_kv, self.d)
            out[p] = raw.astype(np.float64) * self.scales[self.layer][at][col:col + self.n_kv, None].astype(np.float64) if self.i8 else from_bf16(raw)
        return out, ok

    def inputs(self, g):
        """The graph's inputs of the cache and the batch, their arrays, and the keywords every paged op takes."""
        dt = "i8" if self.i8 else "bf16"
        arrays = [self.row_start, self.context, self.table, self.k, self.v]
        refs = [g.input(self.row_start.shape, "i32"), g.input(self.context.shape, "i32"), g.input(self.table.shape, "i32"),
                g.input(self.k.shape, dt), g.input(self.v.shape, dt)]
        kw = dict(n_kv=self.n_kv, head_dim=self.d, layer=self.layer)
        if self.i8:
            kw["scales"] = g.input(self.scales.shape, "f32")
            arrays.append(self.scales)
        return refs, arrays, kw


def attention(b, q_bits, scale, window=0, sinks=0, max_new=0):
    """(o, sum of p |v| / sum of p, rows that are written) of attn_paged in 64 bits."""
    q = from_bf16(q_bits).astype(np.float64).reshape(b.rows, b.n_q, b.d)
    out, spread, written = np.zeros_like(q), np.zeros_like(q), np.zeros(b.rows, bool)
    group = b.n_q // b.n_kv
    for s in range(b.seqs):
        count = b.new[s] if not max_new else min(b.new[s], max_new)
        if not count:
            continue
        total = b.ctx[s] + count
        (k, ok), (v, _) = b.cached("k", s, total), b.cached("v", s, total)
        pos, j = np.arange(b.ctx[s], total)[:, None], np.arange(total)[None]
        seen = (j <= pos) & ok[None]
        if window:
            seen &= (j > pos - window) | (j < sinks)
        r0 = int(b.row_start[s])
        written[r0:r0 + count] = True
        for h in range(b.n_q):
            with np.errstate(invalid="ignore"):
                w = np.where(seen, (q[r0:r0 + count, h] @ k[:, h // group].T) * scale, -np.inf)
                top = w.max(-1, keepdims=True)
                p = np.where(seen, np.exp(w - np.where(np.isfinite(top), top, 0)), 0.0)
            total_p = p.sum(-1, keepdims=True)
            p = np.divide(p, total_p, out=np.zeros_like(p), where=total_p != 0)
            vh = v[:, h // group]
            fine = np.where(np.isfinite(vh), vh, 0.0)  # a hidden key counts for nothing, whatever it holds
            o = p @ fine
            for jj in np.nonzero(~np.isfinite(vh).all(-1))[0]:
                hit = p[:, jj] > 0
                o[hit] += np.where(np.isfinite(vh[jj]), 0.0, vh[jj])
            out[r0:r0 + count, h], spread[r0:r0 + count, h] = o, p @ np.abs(fine)
    return out.reshape(b.rows, -1), spread.reshape(b.rows, -1), written


def check_attention(got_bits, before_bits, want, spread, written):
    """Result and probabilities are each rounded to bf16 once (half a step, 2^-8 of the result and of the sum of p |v|); fp32 scores and sums
    stay within 2^-12 of that sum. Rows nobody owns are as they were."""
    got = from_bf16(got_bits).astype(np.float64)
    assert np.array_equal(got_bits[~written], before_bits[~written])
    assert np.array_equal(np.isfinite(got[written]), np.isfinite(want[written]))
    fine = np.isfinite(want) & written[:, None]
    tol = 2.0 ** -8 * np.abs(want) + (2.0 ** -8 + 2.0 ** -12) * spread + 1e-37
    err = np.where(fine, np.abs(np.where(fine, got, 0) - np.where(fine, want, 0)), 0)
    bad = err > tol
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist(), got[bad][:4], want[bad][:4], float((err / tol).max()))


def rope_write(b, qkv_bits, norms, theta, eps):
    """(queries, keys, values) [rows, heads, d] in 64 bits of every row that belongs to a sequence, and [(row, s, position)]."""
    x = from_bf16(qkv_bits).astype(np.float64).reshape(b.rows, b.n_q + 2 * b.n_kv, b.d)
    n_rot = b.n_q + b.n_kv
    y = x[:, :n_rot].copy()
    if norms is not None:
        w = np.concatenate([np.repeat(from_bf16(norms[0])[None], b.n_q, 0), np.repeat(from_bf16(norms[1])[None], b.n_kv, 0)]).astype(np.float64)
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * (1.0 + w)
    places = [(int(b.row_start[s]) + i, s, b.ctx[s] + i) for s in range(b.seqs) for i in range(b.new[s])]
    half = b.d // 2
    freq = float(np.float32(theta)) ** (-np.arange(half) / half)
    rot = np.zeros_like(y)
    for r, _, p in places:
        c, s = np.cos(p * freq), np.sin(p * freq)
        rot[r, :, :half] = y[r, :, :half] * c - y[r, :, half:] * s
        rot[r, :, half:] = y[r, :, half:] * c + y[r, :, :half] * s
    mag = np.abs(y)
    mag = np.concatenate([mag[..., :half] + mag[..., half:]] * 2, -1)  # what cancels in a rotation
    return rot[:, :b.n_q], rot[:, b.n_q:], x[:, n_rot:], mag, places
