"""Rows of attn_paged without any weight: a row that sees no key is zeros, one whose visible scores are all -inf has no softmax (NaN), one with a
score above -inf anywhere is computed as ever."""
import numpy as np
import pytest

from paged_ref import Batch, attention, bf16, check_attention
from test_gpu_paged_repair import attend
from torq_b200.bf16 import from_bf16, to_bf16

pytestmark = pytest.mark.gpu
LOWEST = to_bf16(np.array([-np.inf], np.float32))[0]


def batch(new, ctx, i8, n_q=4, n_kv=2, d=64, page=16, **kw):
    """Queries and keys whose scores are sums of positive numbers, so that a key of -inf (int8: a scale of -inf) makes a score of -inf."""
    b = Batch(new, ctx, n_q=n_q, n_kv=n_kv, d=d, page=page, i8=i8, **kw)
    if i8:
        b.k = np.abs(b.k.astype(np.int16)).clip(1, 127).astype(np.int8)
    else:
        b.k = to_bf16(np.abs(from_bf16(b.k)))
    return b, to_bf16(np.abs(from_bf16(bf16(b.rng, b.rows, n_q * d))))


def lowest(b, s, positions, head=None):
    for p in positions:
        page, off = b.slot(s, p)
        heads = range(b.n_kv) if head is None else [head]
        for h in heads:
            if b.i8:
                b.scales[b.layer, page, off, h] = -np.inf
            else:
                b.k[b.layer, page, off, h * b.d] = LOWEST


def check(device, b, q, **kw):
    out, before, _ = attend(device, b, q, **kw)
    want, spread, written = attention(b, q, b.d ** -0.5, **kw)  # zeros where there is no weight
    window, sinks, max_new = kw.get("window", 0), kw.get("sinks", 0), kw.get("max_new", 0)
    empty = np.zeros((b.rows, b.n_q), bool)
    want = want.reshape(b.rows, b.n_q, b.d)
    for s in range(b.seqs):
        count = min(b.new[s], max_new) if max_new else b.new[s]
        k, ok = b.cached("k", s, b.ctx[s] + count)
        gone = ~np.isfinite(k).all(-1)  # [keys, heads]: a score of -inf
        for i in range(count):
            p = b.ctx[s] + i
            j = np.arange(p + 1)
            seen = ok[:p + 1] & ((j > p - window) | (j < sinks) if window else True)
            for h in range(b.n_q):
                hk = h // (b.n_q // b.n_kv)
                r = int(b.row_start[s]) + i
                if seen.any() and gone[:p + 1, hk][seen].all():
                    want[r, h] = np.nan
                    empty[r, h] = True
    check_attention(out, before, want.reshape(b.rows, -1), spread, written)
    got = from_bf16(out).reshape(want.shape)
    assert np.isnan(got[empty]).all()
    return empty, got


@pytest.mark.parametrize("i8", [False, True])
def test_the_one_visible_key(device, i8):
    b, q = batch([1, 1, 1], [0, 40, 700], i8)
    for s in range(3):
        lowest(b, s, [b.ctx[s]], head=s % 2 if s < 2 else None)
    empty, _ = check(device, b, q, max_new=1)
    assert empty[0, :2].all() and not empty[0, 2:].any() and not empty[1:].any()
    empty, _ = check(device, b, q, max_new=1, window=1)
    assert empty.any(1).all() and empty[2].all()


@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("heads", [(2, 2, 64), (4, 1, 256), (3, 1, 80)])
def test_many_rows(device, heads, i8):
    n_q, n_kv, d = heads
    b, q = batch([150, 20], [300, 0], i8, n_q, n_kv, d)
    lowest(b, 0, range(0, 380))
    lowest(b, 1, range(0, 7))
    empty, _ = check(device, b, q)
    assert empty[:80].all() and not empty[80:150].any() and empty[150:157].all() and not empty[157:].any()
    check(device, b, q, window=50, sinks=3)


@pytest.mark.parametrize("i8", [False, True])
def test_many_tiles(device, i8):
    """Whole tiles to a block."""
    b, q = batch([140], [130], i8, 150, 150, 16)
    lowest(b, 0, range(0, 200), head=3)
    lowest(b, 0, range(0, 270), head=149)
    empty, _ = check(device, b, q)
    assert empty[:70, 3].all() and empty[:, 149].all() and empty.sum() == 70 + 140


@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("max_new", [0, 2])
def test_beside_rows_that_see_nothing(device, max_new, i8):
    b, q = batch([2] * 60 if max_new else [40, 33], [60] * 60 if max_new else [60, 200], i8)
    b.table[0, :] = -1        # a sequence without pages
    b.table[1, :-1] = -1      # one with its newest page only
    last = b.ctx[1] + b.new[1] - 1
    lowest(b, 1, [last])
    empty, got = check(device, b, q, max_new=max_new)
    assert not got[:b.new[0]].any() and not empty[:b.new[0]].any()
    if last % b.page == 0:    # the newest row sees its own key alone
        assert empty[int(b.row_start[2]) - 1].all()
