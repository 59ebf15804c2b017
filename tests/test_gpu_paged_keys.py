"""attn_paged key by key, and bit by bit: every marked key counts once and no more, and the weights of few rows have the bits they are said to."""
import numpy as np
import pytest

from paged_ref import Batch
from test_gpu_paged_repair import attend
from torq_b200.bf16 import from_bf16, to_bf16

pytestmark = pytest.mark.gpu


def marked(b, s, keys):
    """Values of zero, but for one key in each dim: 64 there."""
    b.v = np.zeros_like(b.v)
    if b.i8:
        b.scales[..., b.n_kv:] = 1.0
    one = np.int8(64) if b.i8 else to_bf16(np.array([64.0], np.float32))[0]
    for d, key in enumerate(keys):
        page, off = b.slot(s, int(key))
        b.v[b.layer, page, off].reshape(b.n_kv, b.d)[:, d] = one


def check_marked(device, b, s, keys, window=0, sinks=0, **kw):
    """Queries of zero give every key that is seen the same weight, exactly: a row's result is 64 over the number of its keys where it sees the marked
    one, and zero where it does not. fp32: one division and a product (2^-22), then half a step of bf16 (2^-8)."""
    marked(b, s, keys)
    out, _, _ = attend(device, b, np.zeros((b.rows, b.n_q * b.d), np.uint16), window=window, sinks=sinks, **kw)
    got = from_bf16(out).astype(np.float64).reshape(b.rows, b.n_q, b.d)[int(b.row_start[s]):int(b.row_start[s]) + b.new[s]]
    keys = np.asarray(keys)
    for i in range(b.new[s]):
        p = b.ctx[s] + i
        j = np.arange(p + 1)
        seen = (j > p - window) | (j < sinks) if window else np.ones(p + 1, bool)
        want = np.where((keys <= p) & seen[np.minimum(keys, p)], 64.0 / seen.sum(), 0.0)
        assert (np.abs(got[i] - want) <= (2.0 ** -8 + 2.0 ** -22) * want).all(), (i, p, np.argwhere(np.abs(got[i] - want) > 2.0 ** -7 * want)[:4].tolist())


def borders(b, s, window=0, sinks=0):
    """Keys at the borders of blocks and pages, at the ends of the window and the first tokens, and some anywhere; all dims' worth of them."""
    end = b.ctx[s] + b.new[s]
    near = [x + o for x in (0, b.ctx[s], end - 1, end - window, b.ctx[s] - window, sinks) for o in (-1, 0, 1)]
    keys = {k for k in near if 0 <= k < end}
    step = [k + o for k in range(0, end, 128) for o in (-1, 0)] + [k + o for k in range(0, end, b.page) for o in (-1, 0)]
    rest = b.rng.permutation([k for k in step if 0 <= k < end and k not in keys])
    keys = sorted(keys) + list(rest) + list(b.rng.integers(0, end, b.d))
    return [int(k) for k in keys[:b.d]]


@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("new,ctx,heads,page", [([1, 1], [30000, 77], (4, 1, 256), 64), ([3, 1], [9000, 300], (4, 2, 128), 24), ([40, 1], [20000, 9], (4, 1, 256), 64),
                                                ([300], [1700], (4, 2, 128), 16), ([129, 5], [4000, 0], (3, 3, 80), 7)])
def test_every_key_counts_once(device, new, ctx, heads, page, i8):
    n_q, n_kv, d = heads
    b = Batch(new, ctx, n_q=n_q, n_kv=n_kv, d=d, page=page, i8=i8)
    for _ in range(2):
        check_marked(device, b, 0, borders(b, 0), max_new=new[0] if new[0] < 4 else 0)


@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("window,sinks", [(1000, 0), (1000, 4), (512, 70), (200, 16)])
@pytest.mark.parametrize("new,heads,page", [([1, 2], (4, 1, 256), 16), ([150, 1], (4, 1, 256), 16), ([150, 1], (4, 2, 128), 12), ([3, 1], (4, 2, 64), 7)])
def test_every_key_of_a_window_counts_once(device, new, heads, page, window, sinks, i8):
    n_q, n_kv, d = heads
    b = Batch(new, [3000, 40], n_q=n_q, n_kv=n_kv, d=d, page=page, i8=i8)
    check_marked(device, b, 0, borders(b, 0, window, sinks), window=window, sinks=sinks)


@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("heads", [(4, 1, 256), (8, 2, 64), (32, 2, 128)])
def test_weights_of_few_rows_have_two_terms(device, heads, i8):
    """Two keys to a sequence, whose scores differ by d and whose values are 1 and -1: (1 - e^-d) / (1 + e^-d). The second weight in two bf16 terms is off
    by 2^-16 of itself, fp32 arithmetic (score, exponential, sums) by less than 2^-20, of a sum of magnitudes of one; the result then by half
    a step (2^-8). In one term, 2^-8 of the weight, most of these would be off by more."""
    n_q, n_kv, d = heads
    seqs = 150
    b = Batch([1] * seqs, [1] * seqs, n_q=n_q, n_kv=n_kv, d=d, page=2, i8=i8)
    delta = from_bf16(to_bf16(np.exp(np.random.default_rng(3).uniform(np.log(2.0 ** -9), np.log(0.4), seqs)).astype(np.float32)))
    b.k, b.v = np.zeros_like(b.k), np.zeros_like(b.v)
    if i8:
        b.scales[...] = 1.0
    q = np.zeros((b.rows, n_q, d), np.float32)
    q[..., 0] = d ** 0.5  # a power of two or not: the scale of the scores is its inverse
    q = to_bf16(q)
    unit = float(from_bf16(q[0, 0, :1])[0]) * d ** -0.5
    for s in range(seqs):
        for p, sign in ((0, 1), (1, -1)):
            page, off = b.slot(s, p)
            k, v = b.k[0, page, off].reshape(n_kv, d), b.v[0, page, off].reshape(n_kv, d)
            v[:] = sign if i8 else to_bf16(np.array([sign], np.float32))[0]
            if p:
                if i8:
                    k[:, 0] = -1
                    b.scales[0, page, off, :n_kv] = delta[s]
                else:
                    k[:, 0] = to_bf16(np.array([-delta[s]], np.float32))[0]
    out, _, _ = attend(device, b, q.reshape(b.rows, -1), max_new=1)
    got = from_bf16(out).astype(np.float64)
    second = np.exp(-delta.astype(np.float64) * unit)
    want = ((1 - second) / (1 + second))[:, None]
    tol = 2.0 ** -8 * np.abs(want) + 2.0 ** -16 + 2.0 ** -20
    assert (np.abs(got - want) <= tol).all(), float((np.abs(got - want) / tol).max())
    rounded = from_bf16(to_bf16(second.astype(np.float32)))
    one_term = ((1 - rounded) / (1 + second))[:, None]
    assert (np.abs(one_term - want) > tol + 2.0 ** -8 * np.abs(want)).mean() > 0.3  # what this test is there to see
