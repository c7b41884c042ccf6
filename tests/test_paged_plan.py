"""How the paged attention's work is cut and dealt, walked on the host: keys
of a unit against its rows one by one, every tile of every unit in exactly
one share, every partial row that a merge reads written by one block, and
quotients by the page size."""

from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

HEADER = Path(__file__).resolve().parents[1] / "kiv_amd" / "csrc" / "kiv_paged_plan.h"

PROGRAM = r"""
#include <stdio.h>
#include <stdlib.h>
#include <algorithm>
#include <map>
#include <random>
#include <set>
#include <vector>
#include "%s"
using namespace kiv;
static long long bad = 0;
#define EXPECT(x) do { if (!(x)) { if (bad++ < 5) printf("line %%d: %%s\n", __LINE__, #x); } } while (0)

static void divisions() {
  std::mt19937_64 g(1);
  for (int i = 0; i < 3000; ++i) {
    const int d = i < 300 ? i + 1 : (int)(g() %% 2147483647ull) + 1;
    const FastDiv f = FastDiv::of(d);
    const int edge[] = {0, 1, d - 1, d, (int)std::min<long long>(2147483647LL, 2LL * d - 1), 2147483647, 2147483646};
    for (int n : edge) EXPECT(f.div(n) == n / d);
    for (int j = 0; j < 50; ++j) {
      const int n = (int)(g() & 0x7fffffff), m = n / d * d;
      EXPECT(f.div(n) == n / d);
      EXPECT(f.div(m) == m / d);
      if (m > 0) EXPECT(f.div(m - 1) == (m - 1) / d);
    }
  }
}

struct Unit { PagedSeq s; int b, kvh, rt; long long start; int n; };

static void walk(int seed) {
  std::mt19937 g(seed);
  auto pick = [&](int lo, int hi) { return lo + (int)(g() %% (unsigned)(hi - lo + 1)); };
  const int seqs = pick(0, 12), hkv = pick(1, 5), G = pick(1, 3) == 1 ? pick(1, 200) : pick(1, 16);
  const int rows = pick(0, 1) ? 16 : 128, shift = pick(0, 1) ? 7 : 6, page = pick(1, 100), width = pick(0, 40);
  const int cap = page * width, window = pick(0, 2) ? 0 : pick(1, 500);
  const bool whole = pick(0, 4) == 0;
  std::vector<int> cu(1, pick(0, 8) ? 0 : -3), len;
  for (int b = 0; b < seqs; ++b) {
    cu.push_back(cu.back() + (pick(0, 5) ? pick(0, 3) : pick(0, 300)) - (pick(0, 30) ? 0 : 7));
    len.push_back(pick(0, 20) ? pick(0, 4000) : pick(0, 1) ? -5 : 2147483647);
  }
  const int total_q = std::max(0, cu.back() + pick(-2, 3));
  const int fixed = pick(0, 5);
  const PagedShape sh = PagedShape::of(total_q, hkv, G, rows, cap, shift, window, whole, fixed);
  std::vector<Unit> units;
  long long total = 0;
  std::set<std::pair<int, int>> seen_rows;  // (packed row, head)
  for (int b = 0; b < seqs; ++b) {
    const PagedSeq s = sh.seq(cu[b], cu[b + 1], len[b]);
    EXPECT(s.q0 >= 0 && s.qlen >= 0 && s.q0 + s.qlen <= std::max(total_q, s.q0));
    for (int h = 0; h < hkv; ++h)
      for (int rt = 0; rt < sh.row_tiles(s); ++rt) {
        int k0, k1;
        sh.keys(s, rt, k0, k1);
        const int tok0 = sh.token0(rt), nt = sh.tokens(s, tok0), hg = rt %% sh.hpt;
        EXPECT(nt >= 1 && nt * std::min(sh.gw, G - hg * rows) <= rows && G - hg * rows > 0);
        long long lo = 1LL << 40, hi = -1;
        for (int t = tok0; t < tok0 + nt; ++t) {
          const long long last = (long long)s.len - s.qlen + t, from = window ? last - window + 1 : 0;
          const long long a = std::max(0LL, from), z = std::min<long long>(cap - 1, last);
          if (a <= z) { lo = std::min(lo, a); hi = std::max(hi, z); }
          if (h == 0 && s.q0 + t < total_q)
            for (int k = 0; k < std::min(sh.gw, G - hg * rows); ++k)
              seen_rows.insert({s.q0 + t, hg * rows + k});
        }
        if (hi < 0) EXPECT(k0 == k1);
        else EXPECT(k0 <= lo && k1 == hi + 1 && (k0 == lo || lo >= k1));
        EXPECT(k0 >= 0 && k1 <= cap);
        const int n = sh.tiles(k0, k1);
        for (int j : {k0, k1 - 1}) if (k0 < k1) EXPECT((j >> shift) >= sh.first_tile(k0) && (j >> shift) < sh.first_tile(k0) + n);
        units.push_back({s, b, h, rt, total, sh.weight(s, rt)});
        EXPECT(sh.weight(s, rt) == (whole ? 1 : n + fixed));
        total += sh.weight(s, rt);
      }
  }
  if (total == 0) return;
  const int most = pick(1, 560);
  const PagedShares shares = PagedShares::deal((int)total, most, whole);
  EXPECT(shares.n >= 1 && shares.n <= most && shares.n <= total);
  EXPECT(shares.start(0) == 0 && shares.start(shares.n) == total);
  std::map<int, int> written;              // partial slot -> unit
  std::map<int, std::vector<int>> merged;  // unit -> slots its merge reads
  std::vector<long long> taken(units.size(), 0), direct(units.size(), 0);
  for (int i = 0; i < shares.n; ++i) {
    long long w = shares.start(i);
    const long long end = shares.start(i + 1);
    EXPECT(w < end);
    EXPECT(shares.block_of(w) == i && shares.block_of(end - 1) == i);
    size_t u = 0;
    while (units[u].start + units[u].n <= w) ++u;
    auto before = [&](size_t v, long long x) {
      return whole ? (int)(x - units[v].start) : sh.tiles_before((int)(x - units[v].start));
    };
    auto tiles = [&](size_t v) { return whole ? 1 : units[v].n - fixed; };
    if (!whole && before(u, w) > 0 && before(u, shares.start(i - 1)) == 0) {
      const int last = shares.block_of((int)(units[u].start + units[u].n - 1));
      merged[(int)u].push_back(2 * i - 1);
      for (int j = i; j <= last; ++j) merged[(int)u].push_back(2 * j);
    }
    for (; w < end; ++u) {
      const long long ue = units[u].start + units[u].n, e = std::min(end, ue);
      const int t0 = before(u, w), t1 = before(u, e);
      EXPECT(t0 == taken[u]);
      if (t0 == t1) { EXPECT(e == end); break; }
      if (t0 == 0 && t1 == tiles(u)) ++direct[u];
      else EXPECT(written.insert({t0 > 0 ? 2 * i : 2 * i + 1, (int)u}).second);
      taken[u] += t1 - t0;
      w = e;
    }
  }
  for (size_t u = 0; u < units.size(); ++u) {
    EXPECT(taken[u] == (whole ? 1 : units[u].n - fixed));
    EXPECT(direct[u] + (long long)merged.count((int)u) == 1);
  }
  size_t read = 0;
  for (auto &m : merged)
    for (int slot : m.second) {
      ++read;
      EXPECT(written.count(slot) && written[slot] == m.first && slot >= 0 && slot < 2 * shares.n);
    }
  EXPECT(read == written.size());
  bool ordered = true;
  for (int b = 0; b < seqs; ++b) ordered &= cu[b] >= 0 && cu[b + 1] >= cu[b] && cu[b + 1] <= total_q;
  if (ordered && seqs) EXPECT((long long)seen_rows.size() == (long long)(cu[seqs] - cu[0]) * G);
}

int main() {
  divisions();
  for (int i = 0; i < 4000; ++i) walk(i);
  printf("%%lld\n", bad);
  return bad != 0;
}
"""


def test_units_shares_and_quotients(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    (tmp_path / "walk.cpp").write_text(PROGRAM % HEADER)
    subprocess.run([gxx, "-O1", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                    str(tmp_path / "walk.cpp"), "-o", str(tmp_path / "walk")], check=True)
    res = subprocess.run([str(tmp_path / "walk")], capture_output=True, text=True, timeout=120)
    assert res.returncode == 0 and res.stdout.strip() == "0", res.stdout + res.stderr


KEYS = r"""
#include <stdio.h>
#include <algorithm>
#include <random>
#include "%s"
using namespace kiv;

// The key index of packed row r of a sequence is kv_len - cu_q[b + 1] + r,
// also where cu_q leaves the rows that the call has.
int main() {
  std::mt19937 g(3);
  auto pick = [&](int lo, int hi) { return lo + (int)(g() %% (unsigned)(hi - lo + 1)); };
  long long bad = 0, rows = 0;
  for (int i = 0; i < 20000; ++i) {
    const int total_q = pick(0, 60), page = pick(1, 30), cap = page * pick(0, 30), G = pick(1, 20);
    const PagedShape sh = PagedShape::of(total_q, 1, G, pick(0, 1) ? 16 : 128, cap, 6, 0, false, 1);
    const int cu0 = pick(-20, 70), far = pick(0, 4);
    const int cu1 = far == 0 ? 2147483647 : far == 1 ? cu0 + pick(-5, 200) : cu0 + pick(0, 40);
    const int len = pick(0, 9) ? pick(0, 300) : pick(0, 1) ? 2147483647 : -pick(1, 2147483647);
    const PagedSeq s = sh.seq(cu0, cu1, len);
    for (int rt = 0; rt < sh.row_tiles(s); ++rt) {
      int k0, k1;
      sh.keys(s, rt, k0, k1);
      const int tok0 = sh.token0(rt), last = tok0 + sh.tokens(s, tok0) - 1;
      const long long key = (long long)len - cu1 + s.q0 + last;
      const long long want = std::max(0LL, std::min<long long>(cap, key + 1));
      ++rows;
      if (k0 != 0 || k1 != want) {
        if (bad++ < 5) printf("rows %%d cu %%d %%d len %%d: keys to %%d, not %%lld\n", total_q, cu0, cu1, len, k1, want);
      }
    }
  }
  printf("%%lld of %%lld\n", bad, rows);
  return bad != 0 || rows < 10000;
}
"""


def test_keys_where_cu_q_leaves_the_rows(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    (tmp_path / "keys.cpp").write_text(KEYS % HEADER)
    subprocess.run([gxx, "-O1", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                    str(tmp_path / "keys.cpp"), "-o", str(tmp_path / "keys")], check=True)
    res = subprocess.run([str(tmp_path / "keys")], capture_output=True, text=True, timeout=120)
    assert res.returncode == 0, res.stdout + res.stderr
