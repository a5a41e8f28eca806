"""Records of where parts of results are (csrc/found.cuh), on the CPU: a join forms addresses from them alone, so every unit
has one even where a pass gave up, and no other bits lead out of the workspace."""
from __future__ import annotations

import shutil
import subprocess

import pytest

from asmllm_b200 import build

PROGRAM = r"""
#include <cassert>
#include <climits>
#include <cstdio>
#include <random>
#include <vector>
#include "found.cuh"
using namespace asmllm;

struct Walk {
  int unit, t, nt;
  long long at, end;
};

// Units of random lengths cut over ranges; each range gives up at some tile, and every unit has a record all the same.
void give_up(std::mt19937& rng) {
  const int units = 1 + rng() % 40, ranges = 1 + rng() % 12;
  std::vector<int> nt(units);
  long long total = 0;
  for (int& n : nt) total += n = 1 + rng() % 9;
  std::vector<int> parts(units, -1);
  for (int r = 0; r < ranges; ++r) {
    Walk w;
    w.at = total * r / ranges;
    w.end = total * (r + 1) / ranges;
    if (w.at == w.end) continue;
    long long x = 0;
    for (w.unit = 0; w.at >= x + nt[w.unit]; ++w.unit) x += nt[w.unit];
    w.nt = nt[w.unit];
    w.t = (int)(w.at - x);
    auto advance = [&](int n) {
      w.at += n;
      if (w.at < w.end) {
        w.nt = nt[++w.unit];
        w.t = 0;
      }
    };
    const long long stop = w.at + (long long)(rng() % (unsigned long long)(w.end - w.at));
    while (true) {  // the segments before the one that holds tile `stop` are computed
      const long long n = std::min<long long>(w.nt - w.t, w.end - w.at);
      if (stop < w.at + n) break;
      if (w.t == 0) parts[w.unit] = 2;
      advance((int)n);
    }
    abandon(w, [&]() { parts[w.unit] = 0; }, advance);
    assert(w.at == w.end);
  }
  for (int p : parts) assert(p >= 0);
}

int main() {
  std::mt19937 rng(1);
  for (int i = 0; i < 20000; ++i) give_up(rng);
  auto some = [&](int ranges) {
    switch (rng() % 5) {
      case 0: return (int)(rng() % (2 * ranges + 3)) - 1;
      case 1: return INT_MAX - (int)(rng() % 3);
      case 2: return INT_MIN + (int)(rng() % 3);
      case 3: return (int)(rng() % 3) - 1;
      default: return (int)rng();
    }
  };
  long long held = 0;
  for (int i = 0; i < 2000000; ++i) {
    const int ranges = i & 1 ? 160 : 2400;
    const Found f = {some(ranges), some(ranges), some(ranges), 0};
    const int n = parts_of(f, ranges);
    assert(n >= 0 && n <= ranges && (n == 0 || n == f.parts));
    if (n > 1) {
      ++held;
      assert(f.slot >= 0 && f.slot < 2 * ranges);
      assert(f.first >= 0 && 2ll * ((long long)f.first + n - 1) < 2ll * ranges);
    }
    const int groups = rng() % 9, batch = rng() % 50, s = batch ? rng() % batch : 0;
    const int g = some(8), b = some(50), e = some(50);
    if (in_group(g, b, e, s, groups, batch)) assert(g >= 0 && g < groups && b >= 0 && b <= s && s < e && e <= batch);
  }
  assert(held > 1000);
  // records that passes leave
  assert(parts_of({0, 0, 0, 0}, 160) == 0 && parts_of({1, 159, 319, 0}, 160) == 1 && parts_of({160, 0, 0, 0}, 160) == 160);
  assert(parts_of({2, 158, 317, 0}, 160) == 2 && parts_of({2, 159, 318, 0}, 160) == 0 && parts_of({2, 0, 320, 0}, 160) == 0);
  assert(in_group(0, 0, 3, 2, 1, 3) && !in_group(0, 0, 3, 3, 1, 3) && !in_group(-1, 0, 0, 0, 1, 3));
  puts("ok");
}
"""


def test_records_of_parts(tmp_path):
    compiler = shutil.which("g++")
    if not compiler:
        pytest.skip("no g++")
    source, program = tmp_path / "found.cpp", tmp_path / "found"
    source.write_text("#include <algorithm>\n" + PROGRAM)
    subprocess.run([compiler, "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-x", "c++",
                    f"-I{build.CSRC}", str(source), "-o", str(program)], check=True)
    assert subprocess.run([str(program)], check=True, capture_output=True, text=True).stdout == "ok\n"
