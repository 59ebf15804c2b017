"""gemv_w8 with the rows of a chunk (more than 32) against its definition in 64 bits, through the C ABI."""
import numpy as np
import pytest

from gpu_exec import run_graph_gpu
from torq_b200.bf16 import from_bf16, to_bf16
from torq_b200.oplist import Graph
from torq_b200.runtime import Executable

pytestmark = pytest.mark.gpu


def inputs(rows, n, k, seed=0):
    rng = np.random.default_rng(seed + rows * 131 + n * 7 + k)
    x = to_bf16(rng.normal(0, 1, (rows, k)).astype(np.float32))
    w = rng.integers(-128, 128, (n, k), dtype=np.int8)
    s = to_bf16((rng.uniform(0.5, 1.5, n) / (73.0 * np.sqrt(k))).astype(np.float32))
    return x, w, s


def product(device, x, w, s, f32=False, splits=0):
    g = Graph()
    g.output(g.gemv_w8(g.input(x.shape, "bf16"), w, s, out_dtype="f32" if f32 else "bf16", splits=splits))
    got = run_graph_gpu(device, g, [x])[0]
    return got if f32 else from_bf16(got)


def check(got, x, w, s, f32):
    """Products of bf16 and int8 are exact in fp32. Each of K additions may cut off a step of fp32 (2^-23) of a sum that is at most S, the sum
    of the magnitudes; the scale rounds once more, and a bf16 result by half a step."""
    x64, w64, s64 = from_bf16(x).astype(np.float64), w.astype(np.float64), from_bf16(s).astype(np.float64)
    want, size = x64 @ w64.T * s64, np.abs(x64) @ np.abs(w64).T * np.abs(s64)
    tol = (w.shape[1] + 1) * 2.0 ** -23 * size + (0 if f32 else 2.0 ** -8) * np.abs(want)
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist(), got[bad][:4], want[bad][:4])


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("rows,n,k", [(33, 256, 64), (77, 1536, 1152), (64, 200, 16), (65, 1, 48), (128, 127, 1040), (129, 129, 128), (191, 256, 80),
                                      (192, 257, 64), (193, 31, 2000), (385, 513, 1152), (1000, 1152, 1024), (40, 20000, 64), (5000, 33, 64),
                                      (77, 1152, 6912), (600, 4096, 208)])
def test_products(device, rows, n, k, f32):
    x, w, s = inputs(rows, n, k)
    check(product(device, x, w, s, f32), x, w, s, f32)


@pytest.mark.parametrize("rows", list(range(33, 140, 9)) + [255, 256, 257, 320])
def test_row_counts(device, rows):
    x, w, s = inputs(rows, 384, 320)
    check(product(device, x, w, s), x, w, s, False)


def test_slices_asked_for_by_the_caller_change_nothing(device):
    x, w, s = inputs(50, 300, 512)
    assert np.array_equal(product(device, x, w, s, True), product(device, x, w, s, True, splits=3))


@pytest.mark.parametrize("rows,n,k", [(77, 1536, 1152), (400, 300, 1040)])
def test_rows_do_not_touch_each_other(device, rows, n, k):
    """Infinities and NaN stay in their rows; everything else is what it was without them, bit by bit."""
    x, w, s = inputs(rows, n, k)
    first = product(device, x, w, s, True)
    bad = x.copy()
    bad[5, k - 1], bad[rows - 1, 0] = to_bf16(np.array([np.inf, np.nan], np.float32))
    got = product(device, bad, w, s, True)
    keep = np.ones(rows, bool)
    keep[[5, rows - 1]] = False
    assert np.array_equal(got[keep].view(np.int32), first[keep].view(np.int32))
    assert not np.isfinite(got[~keep]).any()


def test_products_behind_one_another(device):
    """A chunk's feed-forward part: two products with a GEGLU between them, the second reading what the first left."""
    rows, h, inner = 150, 256, 384
    x, w1, s1 = inputs(rows, 2 * inner, h)
    _, w2, s2 = inputs(rows, h, inner, 1)
    g = Graph()
    gu = g.gemv_w8(g.input(x.shape, "bf16"), w1, s1)
    act = g.geglu(gu)
    y = g.gemv_w8(act, w2, s2)
    for t in (gu, act, y):
        g.output(t)
    got_gu, got_act, got_y = run_graph_gpu(device, g, [x])
    check(from_bf16(got_gu), x, w1, s1, False)
    check(from_bf16(got_y), got_act, w2, s2, False)


def test_one_executable_on_several_buffers(device):
    """Dispatched by turns on two inputs and two results, and once more on the first: what a call prepares for its addresses is the call's own."""
    x, w, s = inputs(70, 260, 320)
    x2 = inputs(70, 260, 320, 9)[0]
    g = Graph()
    g.output(g.gemv_w8(g.input(x.shape, "bf16"), w, s, out_dtype="f32"))
    ex = Executable(device, g.serialize())
    ins, outs = [device.alloc(x.nbytes) for _ in range(2)], [device.alloc(70 * 260 * 4) for _ in range(2)]
    try:
        for b, a in zip(ins, (x, x2)):
            b.upload(a)
        for i, o in ((0, 0), (1, 1), (1, 0), (0, 1), (0, 0)):
            ex.dispatch([ins[i]], [outs[o]])
        device.wait()
        check(outs[0].download((70, 260), np.float32), x, w, s, True)
        check(outs[1].download((70, 260), np.float32), x, w, s, True)
        ex.dispatch([ins[1]], [outs[1]])
        device.wait()
        check(outs[1].download((70, 260), np.float32), x2, w, s, True)
    finally:
        for b in ins + outs:
            b.free()
        ex.destroy()
