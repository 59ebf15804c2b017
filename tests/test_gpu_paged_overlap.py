"""A chunk's ops are refused at dispatch when a result, or pages and scales that are written, are bound over anything else of the op. Nothing of
the op runs then: the buffers keep their bytes."""
import numpy as np
import pytest

from paged_ref import Batch, bf16
from torq_b200.oplist import Graph
from torq_b200.runtime import Executable, TorqB200Error

pytestmark = pytest.mark.gpu
READ = ["row_start", "context", "table", "k", "v", "scales"]


def graph(b, op):
    """The op's graph, its inputs' names and sizes, its results' sizes."""
    g = Graph()
    refs, arrays, kw = b.inputs(g)
    sizes = dict(zip(READ, (a.nbytes for a in arrays)))
    if op == "attend":
        g.output(g.attn_paged(g.input((b.rows, b.n_q * b.d), "bf16"), *refs, n_q=b.n_q, scale=0.125, **kw))
        sizes["q"] = b.rows * b.n_q * b.d * 2
        return g, sizes, [sizes["q"]], arrays
    if op == "read":
        for t in g.kv_read_paged(*refs, rows=b.rows, **kw):
            g.output(t)
        return g, sizes, [b.rows * b.n_kv * b.d * 2] * 2, arrays
    g.output(g.rope_kv_paged(g.input((b.rows, (b.n_q + 2 * b.n_kv) * b.d), "bf16"), *refs, n_q=b.n_q, theta=1e4, **kw))
    sizes["qkv"] = b.rows * (b.n_q + 2 * b.n_kv) * b.d * 2
    return g, sizes, [b.rows * b.n_q * b.d * 2], arrays


def pairs(op, i8):
    reads = READ if i8 else READ[:-1]
    if op == "attend":
        return [("out0", x) for x in reads + ["q"]]
    if op == "read":
        return [(o, x) for o in ("out0", "out1") for x in reads] + [("out0", "out1")]
    written = ["k", "v"] + (["scales"] if i8 else [])
    res = [("out0", x) for x in reads + ["qkv"]]
    return res + [(w, x) for i, w in enumerate(written) for x in written[i + 1:] + ["row_start", "context", "table", "qkv"]]


@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("op", ["attend", "read", "write"])
def test_overlapping_bindings_are_refused(device, op, i8):
    b = Batch([3, 40], [20, 5], n_q=4, n_kv=4, d=64, page=16, i8=i8)
    g, sizes, outs, arrays = graph(b, op)
    ex = Executable(device, g.serialize())
    names = list(sizes) + [f"out{i}" for i in range(len(outs))]
    size = {**sizes, **{f"out{i}": n for i, n in enumerate(outs)}}
    own = {n: device.alloc(size[n] + 256) for n in names}
    image = {n: bf16(np.random.default_rng(7), (size[n] + 256) // 2) for n in names}
    for n, a in zip(READ, arrays):
        image[n].view(np.uint8)[:a.nbytes] = np.ascontiguousarray(a).view(np.uint8).ravel()
    views = []

    def fill():
        for n in names:
            own[n].upload(image[n])

    def dispatch(bound):
        ex.dispatch([bound[n] for n in sizes], [bound[f"out{i}"] for i in range(len(outs))])
        device.wait()

    try:
        for first, second in pairs(op, i8):
            # at one address, and with one's last 16 bytes under the other's first (a second buffer behind the first one's end)
            for shift in (0, max(0, (size[first] - 1) // 16 * 16)):
                room = device.alloc(shift + max(size[first], size[second]) + 256)
                base = device.import_pointer(room.pointer, room.nbytes)
                over = device.import_pointer(room.pointer + shift, room.nbytes - shift)
                views += [base, over, room]
                mark = bf16(np.random.default_rng(8), room.nbytes // 2)
                room.upload(mark)
                fill()
                with pytest.raises(TorqB200Error):
                    dispatch({**own, first: base, second: over})
                assert np.array_equal(room.download(mark.shape, mark.dtype), mark)
                for n in names:
                    assert np.array_equal(own[n].download(image[n].shape, image[n].dtype), image[n]), n
        fill()
        dispatch(own)  # and apart they run
    finally:
        for x in views + list(own.values()):
            x.free()
        ex.destroy()
