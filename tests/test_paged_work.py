"""How attention over a paged cache cuts its work (csrc/paged.h, compiled here with g++): pages by multiplication, the key blocks of a tile
against every key its tokens see, and the shares of the blocks of the grid."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "torq-compiler_b200", "csrc")

PROGRAM = r'''
#include <cstdio>
#include <cstdlib>
#include <set>
#include <vector>
#include "paged.h"
using namespace tb200;

static int pages() {
  const int sizes[] = {1, 2, 3, 5, 7, 8, 16, 24, 31, 32, 100, 127, 128, 129, 200, 1000, 4096, 65535, 65537, 1 << 20, (1 << 30) - 1, 1 << 30};
  for (int d : sizes) {
    const PageDivisor by = page_divisor(d);
    for (long long k = 0; k * d <= 0x7fffffffll && k < 3000; k++)
      for (long long n = k * d - 1; n <= k * d + 1; n++)
        if (n >= 0 && n <= 0x7fffffffll && page_of((int)n, by) != n / d) return printf("%lld / %d\n", n, d), 1;
    for (long long n = 0x7fffffffll; n > 0x7fffffffll - 5000; n--)
      if (page_of((int)n, by) != n / d) return printf("%lld / %d\n", n, d), 1;
  }
  return 0;
}

static int spans() {
  for (int i = 0; i < 8000; i++) {
    const int tpt = 1 + rand() % 64, n = 1 + rand() % 200, ctx = rand() % 3 ? rand() % 1500 : 0, tile = rand() % ((n + tpt - 1) / tpt);
    const int window = rand() % 3 ? rand() % 600 : 0, sinks = window && rand() % 2 ? rand() % 400 : 0, capacity = rand() % 4 ? 4000 : 1 + rand() % 1700;
    const TileSpan t = tile_span(ctx, n, tile, tpt, window, sinks, capacity);
    std::set<int> keys;
    if (t.blocks < 1) return printf("no block\n"), 1;
    for (int p = 0; p < t.blocks * kKeyBlock; p++) {
      const int key = tile_key(t.front, t.shift, p);
      if (key < 0 || !keys.insert(key).second) return printf("a key twice: %d\n", key), 1;
      if (p % kSpanAlign && key != tile_key(t.front, t.shift, p - 1) + 1) return printf("keys do not follow one another: %d\n", key), 1;
      if (p % kSpanAlign == 0 && key % kSpanAlign) return printf("key %d begins a run\n", key), 1;
      if (!sinks && p % kKeyBlock == 0 && key % kKeyBlock) return printf("key %d begins a block\n", key), 1;
    }
    std::set<int> needed, blocks;
    for (int k = tile * tpt; k < n && k < (tile + 1) * tpt; k++)
      for (int j = 0; j <= ctx + k && j < capacity; j++) {
        if (window && j <= ctx + k - window && j >= sinks) continue;
        if (!keys.count(j)) return printf("key %d of token %d has no place\n", j, k), 1;
        if (!(j < t.end_key && (j >= t.near_key || j < sinks))) return printf("key %d of token %d counts as unseen\n", j, k), 1;
        needed.insert(j);
        blocks.insert(j / kKeyBlock);
      }
    const int most = sinks ? ((int)needed.size() + 2 * (kSpanAlign - 1) + kKeyBlock - 1) / kKeyBlock : (int)blocks.size();
    if (t.blocks > (most > 1 ? most : 1)) return printf("%d blocks for %d\n", t.blocks, most), 1;
  }
  return 0;
}

static int shares() {
  for (int i = 0; i < 3000; i++) {
    const int parts = 1 + rand() % 500;
    const long long total = parts + (i % 3 ? rand() % 5000 : ((long long)rand() << 6) + rand());
    if (work_begin(total, 0, parts) != 0 || work_begin(total, parts, parts) != total) return printf("ends\n"), 1;
    for (int p = 0; p < parts; p++) {
      const long long b = work_begin(total, p, parts), e = work_begin(total, p + 1, parts);
      if (e <= b || e - b > total / parts + 1) return printf("uneven\n"), 1;
      if (work_owner(b, total, parts) != p || work_owner(e - 1, total, parts) != p) return printf("owner\n"), 1;
    }
  }
  return 0;
}

int main() { return pages() || spans() || shares(); }
'''


def test_pages_blocks_and_shares(tmp_path):
    src, exe = tmp_path / "work.cc", tmp_path / "work"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O2", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
