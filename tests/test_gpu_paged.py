"""The operators of a chunk over a paged cache against their definition in 64 bits (paged_ref.py), at the sizes, masks and pages where they
can go wrong, each through the C ABI."""
import numpy as np
import pytest

from paged_ref import Batch, attention, bf16, check_attention, rope_write
from torq_b200.bf16 import from_bf16, to_bf16
from torq_b200.oplist import Graph
from torq_b200.runtime import Executable, TorqB200Error

pytestmark = pytest.mark.gpu


def run_in_place(device, graph, arrays, outs_before, times=1):
    """Dispatches `times` times on bound buffers; the outputs' and the inputs' bytes afterwards."""
    ex = Executable(device, graph.serialize())
    bufs = []
    try:
        for a in list(arrays) + list(outs_before):
            b = device.alloc(max(a.nbytes, 16))
            b.upload(np.ascontiguousarray(a))
            bufs.append(b)
        for _ in range(times):
            ex.dispatch(bufs[:len(arrays)], bufs[len(arrays):])
        device.wait()
        res = [b.download(a.shape, a.dtype) for a, b in zip(list(arrays) + list(outs_before), bufs)]
    finally:
        for b in bufs:
            b.free()
        ex.destroy()
    return res[len(arrays):], res[:len(arrays)]


def attend(device, b, q, scale=None, window=0, sinks=0, max_new=0, times=1):
    scale = b.d ** -0.5 if scale is None else scale
    g = Graph()
    refs, arrays, kw = b.inputs(g)
    g.output(g.attn_paged(g.input(q.shape, "bf16"), *refs, n_q=b.n_q, scale=scale, window=window, sinks=sinks, max_new=max_new, **kw))
    before = bf16(np.random.default_rng(99), *q.shape)
    (out,), _ = run_in_place(device, g, arrays + [q], [before], times)
    return out, before


def check(device, b, q=None, std=2.0, **kw):
    q = bf16(b.rng, b.rows, b.n_q * b.d, std=std) if q is None else q
    out, before = attend(device, b, q, **kw)
    kw.pop("times", None)
    want, spread, written = attention(b, q, kw.pop("scale", None) or b.d ** -0.5, **kw)
    check_attention(out, before, want, spread, written)
    return out


HEADS = [(4, 1, 256), (32, 8, 128), (16, 2, 64), (3, 3, 80), (6, 2, 96), (5, 1, 192), (2, 2, 16), (40, 2, 32), (64, 1, 128), (8, 8, 256)]


@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("heads", HEADS)
def test_attention_of_single_tokens(device, heads, i8):
    """A decode step of sequences of all lengths, the empty context and one without a new token among them."""
    n_q, n_kv, d = heads
    b = Batch([1, 1, 0, 1, 1], [0, 130, 17, 15, 700], n_q=n_q, n_kv=n_kv, d=d, i8=i8, pad=2)
    check(device, b, max_new=1)


@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("heads", HEADS)
def test_attention_of_chunks(device, heads, i8):
    n_q, n_kv, d = heads
    b = Batch([70, 0, 1, 200, 33], [0, 40, 300, 5, 260], n_q=n_q, n_kv=n_kv, d=d, i8=i8, page=32, pad=3, lead=2)
    check(device, b)


@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("page", [1, 7, 16, 24, 128, 200])
def test_attention_page_sizes(device, page, i8):
    b = Batch([150, 1, 37], [133, 257, 0], n_q=8, n_kv=2, d=64, i8=i8, page=page, layers=3, layer=1)
    check(device, b)


@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (128, 0), (128, 130), (100, 300), (1000, 4), (64, 128), (1 << 30, 0)])
def test_attention_windows_and_first_tokens(device, window, sinks, i8):
    b = Batch([140, 1, 9], [260, 500, 0], n_q=4, n_kv=1, d=256, i8=i8, page=16)
    check(device, b, window=window, sinks=sinks)
    b = Batch([1, 1, 1], [0, 999, 300], n_q=4, n_kv=1, d=256, i8=i8, page=16)
    check(device, b, window=window, sinks=sinks, max_new=1)


@pytest.mark.parametrize("new", [1, 2, 3, 4, 5, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 256])
def test_attention_chunk_lengths(device, new):
    check(device, Batch([new], [127], n_q=4, n_kv=1, d=128, page=16))
    check(device, Batch([new, new], [0, 1], n_q=6, n_kv=1, d=64, page=8))


@pytest.mark.parametrize("ctx", [0, 1, 62, 63, 64, 126, 127, 128, 129, 255, 256, 4000])
def test_attention_context_lengths(device, ctx):
    check(device, Batch([1], [ctx], n_q=4, n_kv=1, d=256, page=16), max_new=1)
    check(device, Batch([3], [ctx], n_q=2, n_kv=2, d=128, page=16))


def test_attention_long_context_and_few_rows(device):
    """The keys of one token, and of a short chunk, are shared out over the machine."""
    check(device, Batch([1], [30000], n_q=4, n_kv=1, d=64, page=64), max_new=1)
    check(device, Batch([40], [20000], n_q=4, n_kv=1, d=64, page=64, i8=True))
    check(device, Batch([1, 1], [25000, 3], n_q=16, n_kv=2, d=32, page=64, i8=True), max_new=1)


def test_attention_many_sequences(device):
    rng = np.random.default_rng(5)
    new = [int(n) for n in rng.integers(0, 3, 300)]
    check(device, Batch(new, [int(c) for c in rng.integers(0, 60, 300)], n_q=2, n_kv=1, d=32, page=8, pad=1))
    check(device, Batch([1] * 1200, [int(c) for c in rng.integers(0, 20, 1200)], n_q=2, n_kv=1, d=16, page=8), max_new=1)


@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("max_new", [0, 1])
def test_attention_pages_that_hold_nothing(device, max_new, i8):
    """Released pages behind a window, a sequence without any page, ids past the end, positions past the table."""
    b = Batch([1, 1, 1] if max_new else [20, 50, 6], [200, 64, 31], n_q=4, n_kv=2, d=64, page=16, i8=i8)
    b.table[0, :5] = [-1, -1, b.pages, 2 ** 31 - 1, -2 ** 31]
    b.table[1, :] = -1
    out = check(device, b, max_new=max_new)
    r = int(b.row_start[1])
    assert not out[r:r + b.new[1]].any()  # sees no key: zeros
    b.table = np.ascontiguousarray(b.table[:, :1])  # only the first 16 positions are in the table at all
    check(device, b, max_new=max_new)


@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("max_new", [0, 1])
@pytest.mark.parametrize("heads", [(4, 1, 256), (4, 2, 64)])
def test_attention_masked_places_count_for_nothing(device, value, max_new, heads):
    """What lies behind a sequence's end, behind its window, or later in the chunk, may be anything; a value that is seen is not swallowed."""
    n_q, n_kv, d = heads
    new = [1, 1] if max_new else [90, 5]
    b = Batch(new, [300, 40], n_q=n_q, n_kv=n_kv, d=d, page=16)
    bad = to_bf16(np.array([value], np.float32))[0]
    for s in range(2):
        end = b.ctx[s] + b.new[s]
        page, off = b.slot(s, end - 1)
        b.k[0, page, off + 1:], b.v[0, page, off + 1:] = bad, bad  # behind the end
    for p in (20, 21, 150):  # behind the window of every query
        page, off = b.slot(0, p)
        b.k[0, page, off], b.v[0, page, off] = bad, bad
    if not max_new:  # seen by the later rows of the chunk only
        page, off = b.slot(0, 300 + 60)
        b.v[0, page, off, :d] = bad
    check(device, b, window=100, sinks=4, max_new=max_new)


def test_attention_scores_of_any_size(device):
    """Scores whose exponentials would overflow, nearly equal ones, and masks made of the type's lowest value."""
    b = Batch([40, 1], [100, 90], n_q=4, n_kv=1, d=64, page=16)
    check(device, b, std=60.0)
    check(device, b, std=1e-3)
    lowest = to_bf16(np.array([-3.0e38], np.float32))[0]
    q = from_bf16(bf16(b.rng, b.rows, 256)).copy()
    q[:, ::64] = 1.0
    page, off = b.slot(0, 7)
    b.k[0, page, off, 0] = lowest  # one key far below all others
    check(device, b, q=to_bf16(q))
    b.k[..., 0] = lowest           # every key: the same score up to rounding, and finite
    b.k[..., 1:] = 0
    check(device, b, q=to_bf16(q))


@pytest.mark.parametrize("max_new", [0, 1])
@pytest.mark.parametrize("heads", [(4, 1, 256), (8, 2, 64), (3, 3, 96)])
def test_attention_scales_that_the_cache_was_given(device, heads, max_new):
    """Scales are the caller's: zeros over integers that are none, negative ones, ones whose products underflow, among keys that are hidden."""
    n_q, n_kv, d = heads
    b = Batch([1, 1] if max_new else [90, 5], [300, 40], n_q=n_q, n_kv=n_kv, d=d, page=16, i8=True)
    kind = b.rng.integers(0, 6, b.scales.shape)
    b.scales = np.where(kind == 0, 0.0, np.where(kind == 1, -b.scales, np.where(kind == 2, 1e-44, b.scales))).astype(np.float32)
    check(device, b, window=100, sinks=4, max_new=max_new)
    b.scales[...] = 0.0  # every key the same, every value zero
    assert not from_bf16(check(device, b, max_new=max_new)[:int(b.row_start[-1])]).any()


@pytest.mark.parametrize("i8", [False, True])
def test_attention_repeats_bit_by_bit(device, i8):
    b = Batch([1] * 7 + [60], [900, 3, 50, 2000, 128, 7, 64, 1500], n_q=8, n_kv=2, d=128, page=16, i8=i8)
    q = bf16(b.rng, b.rows, b.n_q * b.d)
    first = attend(device, b, q)[0]
    for _ in range(3):
        assert np.array_equal(first, attend(device, b, q, times=3)[0])


def test_attention_two_executables_and_changing_batches(device):
    """Two loaded chunks take turns, and the batch of one changes between its calls (more sequences of few rows, then one of many, then none): nothing
    is kept from a call that another would see."""
    first = Batch([100, 1, 3], [300, 2000, 40], n_q=8, n_kv=2, d=64, page=16, pad=40, seed=3)
    other = Batch([1] * 5, [700, 3, 90, 1500, 128], n_q=4, n_kv=1, d=256, page=32, i8=True, seed=4)
    loaded = []
    try:
        for b in (first, other):
            g = Graph()
            refs, arrays, kw = b.inputs(g)
            q = bf16(b.rng, b.rows, b.n_q * b.d)
            g.output(g.attn_paged(g.input(q.shape, "bf16"), *refs, n_q=b.n_q, scale=b.d ** -0.5, **kw))
            bufs = []
            for a in arrays + [q, bf16(b.rng, *q.shape)]:
                bufs.append(device.alloc(a.nbytes))
                bufs[-1].upload(np.ascontiguousarray(a))
            loaded.append((Executable(device, g.serialize()), bufs, b, q))

        def turn(which):
            ex, bufs, b, q = loaded[which]
            bufs[0].upload(b.row_start)
            bufs[1].upload(b.context)
            before = bf16(b.rng, *q.shape)
            bufs[-1].upload(before)
            ex.dispatch(bufs[:-1], bufs[-1:])
            device.wait()
            check_attention(bufs[-1].download(q.shape, np.uint16), before, *attention(b, q, b.d ** -0.5))

        for new in ([100, 1, 3], [2, 140, 2], [1, 1, 1], [0, 0, 0], [144, 0, 0], [0, 2, 90]):
            first.new = new
            first.row_start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
            first.ctx = [300 - min(300, new[0]), 2000 - new[1], 40 if new[2] < 4 else 0]
            first.context = np.array(first.ctx, np.int32)
            turn(0)
            turn(1)
    finally:
        for ex, bufs, _, _ in loaded:
            for x in bufs:
                x.free()
            ex.destroy()


# ---- cache -------------------------------------------------------------------------------------------------------

def write(device, b, qkv, norms=None, theta=10000.0, eps=1e-6):
    g = Graph()
    refs, arrays, kw = b.inputs(g)
    g.output(g.rope_kv_paged(g.input(qkv.shape, "bf16"), *refs, *(norms or ()), n_q=b.n_q, theta=theta, eps=eps, **kw))
    before = bf16(np.random.default_rng(98), b.rows, b.n_q * b.d)
    (q,), after = run_in_place(device, g, arrays + [qkv], [before])
    return q, before, after


@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("heads", HEADS)
def test_write(device, heads, norm, i8):
    n_q, n_kv, d = heads
    b = Batch([7, 0, 1, 30], [0, 9, 100, 13], n_q=n_q, n_kv=n_kv, d=d, page=24, i8=i8, layers=2, layer=1, pad=3, lead=1)
    b.table[3, 1] = -1  # a page that is not there: what belongs in it is dropped
    qkv = bf16(b.rng, b.rows, (n_q + 2 * n_kv) * d)
    if i8:
        qkv[2, -d:] = 0                                       # a head of zeros
        qkv[4, -d:] = to_bf16(np.array([np.inf], np.float32))[0]  # one that is not finite
    norms = (bf16(b.rng, d, std=0.2), bf16(b.rng, d, std=0.2)) if norm else None
    check_write(device, b, qkv, norms)


def check_write(device, b, qkv, norms, theta=10000.0, eps=1e-6):
    q, before, after = write(device, b, qkv, norms, theta, eps)
    wq, wk, wv, mag, places = rope_write(b, qkv, norms, theta, eps)
    owned = np.zeros(b.rows, bool)
    owned[[r for r, _, _ in places]] = True
    assert np.array_equal(q[~owned], before[~owned])
    # fp32 arithmetic: a rounding (2^-24) each of norm, angle, products and sums, against what cancels; then one to bf16 (2^-8)
    got = from_bf16(q).reshape(wq.shape)[owned]
    tol = 2.0 ** -8 * np.abs(wq[owned]) + 2.0 ** -19 * mag[owned][:, :b.n_q]
    assert (np.abs(got - wq[owned]) <= tol).all()
    k, v = after[3], after[4]
    exp_k, exp_v = b.k.copy(), b.v.copy()
    for r, s, p in places:
        at = b.slot(s, p)
        if at is None:
            continue
        for which, (pages, expect, val, slack) in enumerate(((k, exp_k, wk[r], 2.0 ** -19 * mag[r, b.n_q:]), (v, exp_v, wv[r], np.zeros_like(wv[r])))):
            here = pages[b.layer][at].reshape(b.n_kv, b.d)
            expect[b.layer][at] = pages[b.layer][at]  # what is left of it has to be untouched
            if not b.i8:
                assert (np.abs(from_bf16(here) - val) <= 2.0 ** -8 * np.abs(val) + slack).all()
                continue
            scale = after[5][b.layer][at][which * b.n_kv:(which + 1) * b.n_kv].astype(np.float64)
            for h in range(b.n_kv):
                if not np.isfinite(val[h]).all():
                    assert np.isnan(scale[h])
                    continue
                amax = np.abs(val[h]).max()
                assert abs(scale[h] - amax / 127) <= 2.0 ** -19 * amax / 127 + 2.0 ** -19 * slack[h].max()
                # the nearest integer, but for values that fp32 puts on the other side of a half
                assert (np.abs(here[h] * scale[h] - val[h]) <= scale[h] * (0.5 + 2.0 ** -14)).all()
    assert np.array_equal(k, exp_k) and np.array_equal(v, exp_v)
    if b.i8:
        touched = np.zeros(b.scales.shape[:3], bool)
        for r, s, p in places:
            at = b.slot(s, p)
            if at is not None:
                touched[(b.layer,) + at] = True
        assert np.array_equal(after[5][~touched], b.scales[~touched])


@pytest.mark.parametrize("theta", [1.0, 10000.0, 1.0e6])
def test_write_at_far_positions(device, theta):
    """Angles of a million radians, to the last bit that bf16 can show."""
    b = Batch([5, 3], [1_000_000, 2 ** 20 - 2], n_q=2, n_kv=1, d=64, page=256)
    check_write(device, b, bf16(b.rng, b.rows, 4 * 64), None, theta=theta)


def test_write_many_rows(device):
    """Enough rows that a group of lanes takes several heads."""
    b = Batch([2500, 1200], [3, 90], n_q=6, n_kv=2, d=64, page=32, i8=True)
    check_write(device, b, bf16(b.rng, b.rows, 10 * 64), (bf16(b.rng, 64, std=0.2), bf16(b.rng, 64, std=0.2)))


@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("heads", HEADS)
def test_read(device, heads, i8):
    n_q, n_kv, d = heads
    b = Batch([20, 0, 1, 50], [3, 9, 70, 0], n_kv=n_kv, d=d, page=7, i8=i8, layers=2, layer=1, pad=3, lead=1)
    b.table[0, 1] = -1
    g = Graph()
    refs, arrays, kw = b.inputs(g)
    for t in g.kv_read_paged(*refs, rows=b.rows, **kw):
        g.output(t)
    before = [bf16(b.rng, b.rows, n_kv * d) for _ in range(2)]
    outs, _ = run_in_place(device, g, arrays, before)
    for name, got, old in zip("kv", outs, before):
        want = from_bf16(old).astype(np.float64).reshape(b.rows, n_kv, d)
        for s in range(b.seqs):
            r = int(b.row_start[s])
            want[r:r + b.new[s]] = b.cached(name, s, b.ctx[s] + b.new[s])[0][b.ctx[s]:]
        # integer times scale in fp32 (2^-24), rounded to bf16 (2^-8); bf16 caches as they are
        tol = (2.0 ** -8 + 2.0 ** -23) * np.abs(want) if b.i8 else 0.0 * want
        assert (np.abs(from_bf16(got).reshape(want.shape) - want) <= tol).all()


@pytest.mark.parametrize("i8", [False, True])
def test_a_chunk_as_it_is_used(device, i8):
    """Write, attend and read back in one graph, chunk after chunk: what a later chunk sees is what the earlier ones left."""
    n_q, n_kv, d = 8, 2, 64
    b = Batch([9, 30], [0, 0], n_q=n_q, n_kv=n_kv, d=d, page=8, i8=i8)
    b.table = np.arange(24, dtype=np.int32).reshape(2, 12)
    b.pages = 24
    shape = (1, 24, 8, n_kv * d)
    b.k = b.v = np.zeros(shape, np.int8 if i8 else np.uint16)
    b.scales = np.zeros(shape[:3] + (2 * n_kv,), np.float32) if i8 else None
    g = Graph()
    refs, arrays, kw = b.inputs(g)
    x = g.input((39, (n_q + 2 * n_kv) * d), "bf16")
    q = g.rope_kv_paged(x, *refs, n_q=n_q, theta=10000.0, **kw)
    o = g.attn_paged(q, *refs, n_q=n_q, scale=d ** -0.5, window=25, sinks=2, **kw)
    k, v = g.kv_read_paged(*refs, rows=39, **kw)
    for t in (q, o, k, v):
        g.output(t)
    ex = Executable(device, g.serialize())
    bufs = [device.alloc(a.nbytes) for a in arrays] + [device.alloc(39 * (n_q + 2 * n_kv) * d * 2)]
    outs = [device.alloc(i.nbytes) for i in ex.outputs_info]
    for buf, a in zip(bufs, arrays):
        buf.upload(a)
    for chunk in range(3):
        b.ctx = [int(c) for c in b.context]
        bufs[1].upload(b.context)
        qkv = bf16(b.rng, 39, (n_q + 2 * n_kv) * d)
        bufs[-1].upload(qkv)
        before = np.zeros((39, n_q * d), np.uint16)
        ex.dispatch(bufs, outs)
        gq, go, gk, gv = (buf.download(i.shape, i.np_dtype) for buf, i in zip(outs, ex.outputs_info))
        b.k, b.v = (bufs[i].download(shape, b.k.dtype) for i in (3, 4))
        if i8:
            b.scales = bufs[5].download(b.scales.shape, np.float32)
        want, spread, written = attention(b, gq, d ** -0.5, window=25, sinks=2)
        check_attention(go, before, want, spread, written)
        for name, got in (("k", gk), ("v", gv)):
            for s in range(2):
                r = int(b.row_start[s])
                held = b.cached(name, s, b.ctx[s] + b.new[s])[0][b.ctx[s]:].reshape(b.new[s], -1)
                assert (np.abs(from_bf16(got[r:r + b.new[s]]) - held) <= (2.0 ** -8 + 2.0 ** -23) * np.abs(held)).all()
        b.context = (b.context + np.array(b.new)).astype(np.int32)
    for buf in bufs + outs:
        buf.free()
    ex.destroy()


def test_results_bound_over_what_is_read_are_refused(device):
    """One buffer as queries and result, as product's input and result, as keys and values that are written, or as cache and what is read from it."""
    b = Batch([3, 40], [20, 5], n_q=4, n_kv=4, d=64, page=16)
    room = device.alloc(max(b.k.nbytes, b.rows * 16 * 64 * 2) + 4096)
    rest = [device.alloc(1 << 20) for _ in range(8)]

    def run(graph, inputs, outputs):
        ex = Executable(device, graph.serialize())
        try:
            ex.dispatch(inputs, outputs)
            device.wait()
        finally:
            ex.destroy()

    def refused(make):
        g = Graph()
        refs, arrays, kw = b.inputs(g)
        own = [device.alloc(a.nbytes) for a in arrays]
        try:
            for x, a in zip(own, arrays):
                x.upload(a)
            with pytest.raises(TorqB200Error):
                run(*make(g, refs, kw, own))
        finally:
            for x in own:
                x.free()

    def attend_over(which):
        def make(g, refs, kw, own):
            g.output(g.attn_paged(g.input((b.rows, 256), "bf16"), *refs, n_q=4, scale=0.125, **kw))
            return g, own + [room], [room if which == "q" else own[3]]
        return make

    def write_over(which):
        def make(g, refs, kw, own):
            g.output(g.rope_kv_paged(g.input((b.rows, 12 * 64), "bf16"), *refs, n_q=4, theta=1e4, **kw))
            if which == "kv":
                own = own[:4] + [own[3]]
            return g, own + [room], [rest[0] if which == "kv" else room]
        return make

    def read_over(g, refs, kw, own):
        for t in g.kv_read_paged(*refs, rows=b.rows, **kw):
            g.output(t)
        return g, own, [rest[0], rest[0]]

    def product_over(g, refs, kw, own):
        g = Graph()
        g.output(g.gemv_w8(g.input((40, 64), "bf16"), np.ones((64, 64), np.int8), to_bf16(np.ones(64, np.float32))))
        return g, [room], [room]

    try:
        for make in (attend_over("q"), attend_over("k"), write_over("qkv"), write_over("kv"), read_over, product_over):
            refused(make)
        check(device, b)  # and the device goes on
    finally:
        for x in [room] + rest:
            x.free()
