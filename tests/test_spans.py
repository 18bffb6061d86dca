"""No-GPU check of the memory checks in front of a launch: two sets of columns share a byte, or not, against all pairs of columns."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pooled_amd", "csrc")

PROGRAM = r"""
#include "spans.h"
#include <cstdio>
#include <random>
int main() {
  std::mt19937 r(1);
  auto upto = [&](uint32_t n) { return r() % n; };
  int met = 0, between = 0;
  for (int it = 0; it < 400000; it++) {
    const uint32_t n = 1 + upto(6);
    Columns c[2];
    for (Columns& k : c) { k.p = (const void*)(uintptr_t)(1000 + upto(60)); k.bytes = 1 + upto(9); k.step = k.bytes + upto(25); }
    if (upto(2)) { c[1].step = c[0].step; if (c[1].bytes > c[1].step) c[1].bytes = c[1].step; }
    bool any = false;
    for (uint32_t i = 0; i < n; i++)
      for (uint32_t j = 0; j < n; j++)
        any = any || overlap({(const char*)c[0].p + i * c[0].step, c[0].bytes}, {(const char*)c[1].p + j * c[1].step, c[1].bytes});
    if (columns_meet(c[0], c[1], n) != any) {
      printf("n %u: %p %zu %zu, %p %zu %zu: %d\n", n, c[0].p, c[0].step, c[0].bytes, c[1].p, c[1].step, c[1].bytes, any);
      return 1;
    }
    met += any;
    between += !any && overlap({c[0].p, (n - 1) * c[0].step + c[0].bytes}, {c[1].p, (n - 1) * c[1].step + c[1].bytes});
  }
  if (columns_meet({nullptr, 8, 8}, {(const void*)4, 8, 8}, 3)) return 2;
  puts(met > 50000 && between > 20000 ? "ok" : "too few cases");
}
"""


def test_columns_that_share_a_byte(tmp_path):
    src, exe = tmp_path / "t.cc", tmp_path / "t"
    src.write_text(PROGRAM)
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-Wno-unused-function", "-I", CSRC, str(src), "-o", str(exe)])
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr
