"""Rows of attn_paged whose sums come out non-finite (a hidden value that is an infinity meets a weight of zero) and are computed once more: over long
contexts, in all the places that may have to do it, and in a time that no wait's limit ends."""
import time

import numpy as np
import pytest

from paged_ref import Batch, attention, bf16, check_attention
from torq_b200.bf16 import from_bf16, to_bf16
from torq_b200.oplist import Graph
from torq_b200.runtime import Executable

pytestmark = pytest.mark.gpu
INF = to_bf16(np.array([np.inf], np.float32))[0]


def attend(device, b, q, **kw):
    g = Graph()
    refs, arrays, heads = b.inputs(g)
    g.output(g.attn_paged(g.input(q.shape, "bf16"), *refs, n_q=b.n_q, scale=b.d ** -0.5, **kw, **heads))
    ex = Executable(device, g.serialize())
    before = bf16(np.random.default_rng(97), *q.shape)
    bufs = []
    try:
        for a in arrays + [q, before]:
            bufs.append(device.alloc(a.nbytes))
            bufs[-1].upload(np.ascontiguousarray(a))
        ex.dispatch(bufs[:-1], bufs[-1:])
        device.wait()
        out = bufs[-1].download(q.shape, np.uint16)
        t = time.perf_counter()
        ex.dispatch(bufs[:-1], bufs[-1:])
        device.wait()
        return out, before, time.perf_counter() - t
    finally:
        for x in bufs:
            x.free()
        ex.destroy()


def check(device, b, q=None, **kw):
    q = bf16(b.rng, b.rows, b.n_q * b.d) if q is None else q
    out, before, seconds = attend(device, b, q, **kw)
    check_attention(out, before, *attention(b, q, b.d ** -0.5, **kw))
    return seconds


def spoil_last(b, s, back=0):
    """What only the last tokens of a sequence see: an infinite value, or a value with a scale of NaN."""
    page, off = b.slot(s, b.ctx[s] + b.new[s] - 1 - back)
    if b.i8:
        b.scales[b.layer, page, off, b.n_kv:] = np.nan
    else:
        b.v[b.layer, page, off] = INF


@pytest.mark.parametrize("i8", [False, True])
def test_a_bad_value_in_a_tile_of_one_block_ends_no_wait(device, i8, monkeypatch):
    """160 heads make more tiles than the machine has blocks, so whole tiles come to one block, whose other roles wait for the next tile meanwhile.
    Their limit is 20 ms here; a row's keys one by one take longer than that."""
    monkeypatch.setenv("TB200_WAIT_LIMIT_MS", "20")
    b = Batch([200], [2000], n_q=160, n_kv=160, d=16, page=64, i8=i8)
    spoil_last(b, 0, back=100)
    assert check(device, b) < 0.25


@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("heads", [(2, 1, 256), (3, 3, 80)])
def test_a_bad_value_in_a_tile_that_blocks_share(device, heads, i8):
    n_q, n_kv, d = heads
    b = Batch([70, 40], [6000, 300], n_q=n_q, n_kv=n_kv, d=d, page=24, i8=i8)
    spoil_last(b, 0, back=5)
    spoil_last(b, 1)
    assert check(device, b) < 0.25


@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("heads", [(4, 1, 256), (10, 2, 64), (1, 1, 16)])
def test_a_bad_value_among_few_rows(device, heads, i8):
    n_q, n_kv, d = heads
    b = Batch([3, 2, 3], [5000, 20, 900], n_q=n_q, n_kv=n_kv, d=d, page=16, i8=i8)
    for s in range(3):
        spoil_last(b, s)
    assert check(device, b, max_new=3) < 0.25
    b = Batch([3] * 200, [30] * 200, n_q=n_q, n_kv=n_kv, d=d, page=16, i8=i8)  # more tiles than blocks
    for s in range(0, 200, 3):
        spoil_last(b, s)
    check(device, b, max_new=3)


@pytest.mark.parametrize("window,sinks", [(0, 0), (700, 0), (700, 5), (5000, 300)])
def test_windows(device, window, sinks):
    b = Batch([150, 3], [3000, 2500], n_q=2, n_kv=1, d=64, page=16)
    for p in (40, 2400, 2999, 3140):
        page, off = b.slot(0, p)
        b.v[0, page, off] = INF
    spoil_last(b, 1)
    b.table[0, 30:33] = -1
    check(device, b, window=window, sinks=sinks)


@pytest.mark.parametrize("new", [[130], [3]])
@pytest.mark.parametrize("first", [1, 130, 300])
def test_first_keys_of_no_weight(device, new, first):
    """The first keys' scores are -inf for every row: no weight, while later keys have some. Beside them a hidden value that is infinite."""
    b = Batch(new, [700], n_q=4, n_kv=1, d=64, page=16)
    q = from_bf16(bf16(b.rng, b.rows, 256)).copy()
    q[:, ::64] = 1.0
    for p in range(first):
        page, off = b.slot(0, p)
        b.k[0, page, off, 0] = to_bf16(np.array([-np.inf], np.float32))[0]
    spoil_last(b, 0)
    check(device, b, q=to_bf16(q), max_new=new[0])
