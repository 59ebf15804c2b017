"""A decoder layer over a chunk as a host builds it, from its input to its output: norm, product, write, attend, product, norm, feed-forward part. Each
op's result is held against its definition in 64 bits over what the op in front of it left."""
import math

import numpy as np
import pytest

from paged_ref import Batch, attention, bf16, check_attention, rope_write
from torq_b200.bf16 import from_bf16, to_bf16
from torq_b200.oplist import Graph
from torq_b200.runtime import Executable

pytestmark = pytest.mark.gpu


def weights(rng, n, k):
    return rng.integers(-127, 128, (n, k), dtype=np.int8), to_bf16((rng.uniform(0.8, 1.25, n) / (73.0 * math.sqrt(k))).astype(np.float32))


def close(bits, want, slack):
    """A result of 64 bits, rounded to bf16 once (2^-8), beside `slack` for what fp32 sums lose."""
    err = np.abs(from_bf16(bits).astype(np.float64) - want)
    tol = 2.0 ** -8 * np.abs(want) + slack
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("heads,hidden", [((4, 1, 256), 1152), ((8, 2, 64), 256)])
def test_a_layer(device, heads, hidden, i8):
    n_q, n_kv, d = heads
    b = Batch([50, 1, 0, 30, 1], [0, 700, 3, 90, 0], n_q=n_q, n_kv=n_kv, d=d, page=16, i8=i8, pad=4)
    rng, eps, inner = b.rng, 1e-6, 2 * hidden
    norm_w = [bf16(rng, hidden, std=0.1) for _ in range(4)]
    qk_norm = (bf16(rng, d, std=0.1), bf16(rng, d, std=0.1))
    w_qkv, w_o, w_gu, w_d = weights(rng, (n_q + 2 * n_kv) * d, hidden), weights(rng, hidden, n_q * d), weights(rng, 2 * inner, hidden), weights(rng, hidden, inner)
    x = bf16(rng, b.rows, hidden)

    g = Graph()
    refs, arrays, kw = b.inputs(g)
    x_in = g.input(x.shape, "bf16")
    h = g.rmsnorm(x_in, norm_w[0], eps)
    qkv = g.gemv_w8(h, *w_qkv)
    q = g.rope_kv_paged(qkv, *refs, *qk_norm, n_q=n_q, theta=10000.0, eps=eps, **kw)
    o = g.attn_paged(q, *refs, n_q=n_q, scale=d ** -0.5, window=512, **kw)
    y = g.gemv_w8(o, *w_o)
    x2 = g.rmsnorm(y, norm_w[1], eps, residual=x_in)
    h2 = g.rmsnorm(x2, norm_w[2], eps)
    gu = g.gemv_w8(h2, *w_gu)
    act = g.geglu(gu)
    down = g.gemv_w8(act, *w_d)
    res = g.rmsnorm(down, norm_w[3], eps, residual=x2)
    named = dict(h=h, qkv=qkv, q=q, o=o, y=y, x2=x2, h2=h2, gu=gu, act=act, down=down, res=res)
    for t in named.values():
        g.output(t)

    ex = Executable(device, g.serialize())
    bufs = []
    try:
        for a in arrays + [x]:
            bufs.append(device.alloc(a.nbytes))
            bufs[-1].upload(np.ascontiguousarray(a))
        outs = [device.alloc(i.nbytes) for i in ex.outputs_info]
        bufs += outs
        for buf, i in zip(outs, ex.outputs_info):
            buf.upload(np.zeros(i.shape, np.uint16))  # rows of nobody keep these
        ex.dispatch(bufs[:len(arrays) + 1], outs)
        device.wait()
        got = {n: buf.download(i.shape, i.np_dtype) for n, buf, i in zip(named, outs, ex.outputs_info)}
        cache = [bufs[i].download(a.shape, a.dtype) for i, a in enumerate(arrays)]
    finally:
        for buf in bufs:
            buf.free()
        ex.destroy()

    def f(name):
        return from_bf16(got[name]).astype(np.float64)

    def norm(v, w, res=None):
        n = v / np.sqrt((v * v).mean(-1, keepdims=True) + eps) * (1.0 + from_bf16(w))
        return n if res is None else n + res

    def product(name, src, w):
        w64, s64, v = w[0].astype(np.float64), from_bf16(w[1]).astype(np.float64), f(src)
        close(got[name], v @ w64.T * s64, (w64.shape[1] + 1) * 2.0 ** -23 * (np.abs(v) @ np.abs(w64).T * s64))

    x64 = from_bf16(x).astype(np.float64)
    close(got["h"], norm(x64, norm_w[0]), 2.0 ** -18 * np.abs(norm(x64, norm_w[0])))
    product("qkv", "h", w_qkv)
    wq, wk, wv, mag, places = rope_write(b, got["qkv"], qk_norm, 10000.0, eps)
    owned = [r for r, _, _ in places]
    close(got["q"].reshape(wq.shape)[owned], wq[owned], 2.0 ** -19 * mag[owned][:, :n_q])
    b.k, b.v = cache[3], cache[4]
    if i8:
        b.scales = cache[5]
    for r, s, p in places:  # what the cache holds of the chunk
        page, off = b.slot(s, p)
        for pages, want, col in ((b.k, wk[r], 0), (b.v, wv[r], n_kv)):
            held = pages[0, page, off].reshape(n_kv, d)
            if i8:
                step = b.scales[0, page, off, col:col + n_kv, None].astype(np.float64)
                assert (np.abs(held * step - want) <= step * (0.5 + 2.0 ** -14)).all()
            else:
                assert (np.abs(from_bf16(held) - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -19 * mag[r, n_q:]).all()
    want, spread, written = attention(b, got["q"], d ** -0.5, window=512)
    check_attention(got["o"], np.zeros_like(got["o"]), want, spread, written)
    product("y", "o", w_o)
    # a norm is rounded to bf16 before the residual comes to it: half a step more, of the norm
    n2 = norm(f("y"), norm_w[1])
    close(got["x2"], n2 + x64, (2.0 ** -8 + 2.0 ** -18) * np.abs(n2) * (1 + 2.0 ** -8))
    close(got["h2"], norm(f("x2"), norm_w[2]), 2.0 ** -18 * np.abs(norm(f("x2"), norm_w[2])))
    product("gu", "h2", w_gu)
    gate, up = np.split(f("gu"), 2, -1)
    gelu = 0.5 * gate * (1 + np.tanh(math.sqrt(2 / math.pi) * (gate + 0.044715 * gate ** 3)))
    # the gate's value is rounded to bf16 before the product; its tanh in fp32 is off by 2^-21 of one, or of the gate
    close(got["act"], gelu * up, ((2.0 ** -8 * np.abs(gelu) + 2.0 ** -20 * np.abs(gate)) * np.abs(up)) * (1 + 2.0 ** -8))
    product("down", "act", w_d)
    n3 = norm(f("down"), norm_w[3])
    close(got["res"], n3 + f("x2"), (2.0 ** -8 + 2.0 ** -18) * np.abs(n3) * (1 + 2.0 ** -8))
