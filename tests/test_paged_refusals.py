"""Calls the builder refuses, and the index arithmetic of pages, without a GPU."""
import os
import subprocess

import numpy as np
import pytest

from torq_b200.oplist import Graph

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "torq-compiler_b200", "csrc")


def parts(g, S=2, pages=5, page=16, n_kv=2, d=64, dtype="bf16", layers=1):
    row_start, context, table = g.input((S + 1,), "i32"), g.input((S,), "i32"), g.input((S, 3), "i32")
    k, v = (g.input((layers, pages, page, n_kv * d), dtype) for _ in range(2))
    return row_start, context, table, k, v


def attend(g, refs, q=None, **kw):
    kw = {"n_q": 4, "n_kv": 2, "head_dim": 64, "scale": 0.125, **kw}
    return g.attn_paged(g.input((7, 4 * 64), "bf16") if q is None else q, *refs, **kw)


def test_what_the_builder_refuses():
    def refused(make):
        g = Graph()
        with pytest.raises(ValueError):
            make(g)

    refused(lambda g: attend(g, parts(g), q=g.input((7, 4 * 64), "f32")))
    refused(lambda g: attend(g, parts(g), q=g.input((7, 4 * 64 + 1), "bf16")))
    refused(lambda g: attend(g, parts(g), q=g.input((7, 3 * 64), "bf16"), n_q=3))           # heads that do not divide
    refused(lambda g: attend(g, parts(g), layer=1))
    refused(lambda g: attend(g, parts(g), n_kv=4, n_q=4))                                   # not the caches' width
    refused(lambda g: attend(g, parts(g, dtype="i8")))                                      # scales missing
    refused(lambda g: attend(g, parts(g), scales=g.input((1, 5, 16, 4), "f32")))            # scales of nothing
    refused(lambda g: attend(g, parts(g, dtype="i8"), scales=g.input((1, 5, 16, 2), "f32")))
    refused(lambda g: attend(g, (lambda p: (p[0], p[1], p[2], p[3], p[3]))(parts(g))))      # one tensor as keys and values
    refused(lambda g: attend(g, (g.input((2,), "i32"),) + parts(g)[1:]))                    # row starts of another count
    refused(lambda g: attend(g, parts(g)[:2] + (g.input((2, 3), "i16"),) + parts(g)[3:]))
    refused(lambda g: g.rope_kv_paged(g.input((7, 8 * 64), "bf16"), *parts(g), np.zeros(64, np.uint16), n_q=4, n_kv=2, head_dim=64, theta=1e4))
    refused(lambda g: g.rope_kv_paged(g.input((7, 7 * 64), "bf16"), *parts(g), n_q=4, n_kv=2, head_dim=64, theta=1e4))

    def intermediate_cache(g):
        p = parts(g)
        attend(g, p[:3] + (g.ew("add", p[3], p[3]), p[4]))
    refused(intermediate_cache)


def test_a_paged_graph_survives_a_round_trip():
    g = Graph()
    p = parts(g, dtype="i8")
    scales = g.input((1, 5, 16, 4), "f32")
    kw = dict(n_kv=2, head_dim=64, scales=scales)
    q = g.rope_kv_paged(g.input((7, 8 * 64), "bf16"), *p, np.zeros(64, np.uint16), np.ones(64, np.uint16), n_q=4, theta=1e4, **kw)
    g.output(g.attn_paged(q, *p, n_q=4, scale=0.125, window=8, sinks=2, max_new=3, **kw))
    for t in g.kv_read_paged(*p, rows=7, **kw):
        g.output(t)
    blob = g.serialize()
    assert Graph.deserialize(blob).serialize() == blob


PROGRAM = r'''
#include <cstdio>
#include "paged.h"
int main() {
  const int ds[] = {1, 2, 3, 5, 7, 8, 16, 24, 64, 100, 127, 128, 129, 200, 1000, 4095, 4096, 65535, 1 << 20, (1 << 30) - 1, 1 << 30};
  for (int d : ds) {
    const tb200::PageDivisor by = tb200::page_divisor(d);
    auto wrong = [&](long long n) { return n >= 0 && n < (1ll << 31) && tb200::page_of((int)n, by) != n / d; };
    for (long long n = 0; n < 300000; n++) if (wrong(n)) { printf("%lld / %d\n", n, d); return 1; }
    for (long long q = 0; q < 20000; q++)
      for (long long n = (0x7fffffffll / d - q) * d - 1; n <= (0x7fffffffll / d - q) * d + 1; n++)
        if (wrong(n)) { printf("%lld / %d\n", n, d); return 1; }
  }
  return 0;
}
'''


def test_the_page_of_a_position(tmp_path):
    src, exe = tmp_path / "page.cc", tmp_path / "page"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
