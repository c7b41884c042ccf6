"""Whether strided rows share memory, by the formulas the entry points use,
against every row's bytes."""

from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

HEADER = Path(__file__).resolve().parents[1] / "kiv_amd" / "csrc" / "kiv_rows.h"

PROGRAM = r"""
#include <stdio.h>
#include <random>
#include <set>
#include <vector>
#include "%s"
using namespace kiv;

static std::vector<int64_t> places(const RowSet &a) {
  std::vector<int64_t> v;
  for (int64_t i = 0; i < a.n[0]; ++i)
    for (int64_t j = 0; j < a.n[1]; ++j)
      for (int64_t k = 0; k < a.n[2]; ++k)
        v.push_back((int64_t)(uintptr_t)a.p + i * a.stride[0] + j * a.stride[1] + k * a.stride[2]);
  return v;
}

int main() {
  std::mt19937 g(5);
  auto pick = [&](int lo, int hi) { return lo + (int)(g() %% (unsigned)(hi - lo + 1)); };
  long long bad = 0, met = 0, apart = 0, exact = 0, folded = 0;
  for (int t = 0; t < 200000; ++t) {
    // Slices of one buffer [outer, middle, inner] of rows, its axes in any order.
    const int64_t row = 16, inner = pick(1, 4), middle = pick(1, 4), gap = pick(0, 2);
    int64_t s[3] = {row * inner * (middle + gap), row * inner, row};
    int order[3] = {0, 1, 2};
    std::shuffle(order, order + 3, g);
    const int64_t most[3] = {4, middle, inner};
    const bool nested = pick(0, 4) > 0;
    RowSet a, b;
    a.row = b.row = row;
    for (int i = 0; i < 3; ++i) {
      const int from = order[i], sign = pick(0, 9) ? 1 : -1;
      a.stride[i] = b.stride[i] = sign * (nested ? s[from] : row * pick(0, 6));
      a.n[i] = pick(pick(0, 30) ? 1 : 0, (int)most[from]);
      b.n[i] = pick(pick(0, 30) ? 1 : 0, (int)most[from]);
      if (a.n[i] == 1 && pick(0, 1)) a.stride[i] = row * pick(-9, 9);
      if (!nested && pick(0, 1)) b.stride[i] = row * pick(0, 6);
    }
    a.p = (const void *)(uintptr_t)(100000 + row * pick(0, 40));
    b.p = (const void *)(uintptr_t)(100000 + row * pick(0, 40));
    const auto pa = places(a), pb = places(b);
    bool share = false;
    for (auto x : pa) for (auto y : pb) share |= x < y + row && y < x + row;
    const bool said = rows_overlap(a, b);
    bad += share && !said;
    // Exact between slices of one buffer (each inside it, so that no axis runs over another).
    if (nested) {
      ++exact;
      bad += share != said;
    }
    met += share;
    apart += !said;
    bool fold = false;
    std::set<int64_t> seen;
    for (auto x : pa) fold |= !seen.insert(x).second;
    bad += fold && !rows_fold(a);
    if (nested) bad += fold != rows_fold(a);
    folded += fold;
    if (rows_same(a, b)) bad += pa != pb;
  }
  printf("%%lld bad of %%lld shared, %%lld apart, %%lld exact, %%lld folded\n", bad, met, apart, exact, folded);
  return bad != 0 || met < 1000 || apart < 1000 || folded < 1000;
}
"""


def test_rows_that_share_memory(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    (tmp_path / "rows.cpp").write_text(PROGRAM % HEADER)
    subprocess.run([gxx, "-O1", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                    str(tmp_path / "rows.cpp"), "-o", str(tmp_path / "rows")], check=True)
    res = subprocess.run([str(tmp_path / "rows")], capture_output=True, text=True, timeout=120)
    assert res.returncode == 0, res.stdout + res.stderr
