"""Which buffers may lie over one another in an op that reads while it writes (csrc/paged.h, compiled here with g++)."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "torq-compiler_b200", "csrc")

PROGRAM = r'''
#include <cstdio>
#include <cstdlib>
#include "paged.h"
using namespace tb200;

int main() {
  static char room[64];
  auto at = [&](int from, int bytes) { return ByteRange{room + from, (size_t)bytes}; };
  if (!writes_lie_apart({at(0, 16), at(16, 16), at(32, 8)}, 2)) return printf("neighbours\n"), 1;
  if (writes_lie_apart({at(0, 17), at(16, 16), at(40, 8)}, 2)) return printf("two that are written\n"), 1;
  if (writes_lie_apart({at(0, 16), at(20, 4), at(8, 100)}, 1)) return printf("written over read\n"), 1;
  if (!writes_lie_apart({at(0, 16), at(20, 4), at(20, 4), at(16, 30)}, 1)) return printf("read twice\n"), 1;
  if (!writes_lie_apart({at(0, 16), {nullptr, 0}, at(4, 0)}, 2)) return printf("nowhere\n"), 1;
  if (!writes_lie_apart({at(8, 0), at(0, 16)}, 1)) return printf("nothing written\n"), 1;
  // any three ranges, byte by byte
  for (int i = 0; i < 200000; i++) {
    ByteRange r[3];
    int owner[64] = {}, clash = 0;
    const int written = rand() % 3;
    for (int k = 0; k < 3; k++) {
      const int from = rand() % 40, n = rand() % 20;
      r[k] = at(from, n);
      for (int b = from; b < from + n; b++) {
        for (int o = 0; o < k; o++) clash |= (owner[b] >> o & 1) && o < written;
        owner[b] |= 1 << k;
      }
    }
    if (writes_lie_apart({r[0], r[1], r[2]}, written) == (bool)clash) return printf("case %d\n", i), 1;
  }
  return 0;
}
'''


def test_what_is_written_lies_apart(tmp_path):
    src, exe = tmp_path / "overlap.cc", tmp_path / "overlap"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
