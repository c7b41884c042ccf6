// How the paged attention's work is cut into units and dealt to blocks.
// Plain C++ beside the kernels that use it, so that the arithmetic is also
// checked on the host.
#pragma once

#include <stdint.h>

#if defined(__HIPCC__)
#define KIV_HD __host__ __device__
#else
#define KIV_HD
#endif

namespace kiv {

// Quotients of 31-bit numbers by a fixed divisor: n / d == (n * mul) >> shift.
// With l = ceil(log2 d), mul = floor(2^(31 + l) / d) + 1 exceeds 2^(31 + l) / d
// by less than 1 <= 2^l / d, so n * mul / 2^(31 + l) exceeds n / d by less
// than n / 2^(31) / d < 1 / d.
struct FastDiv {
  uint32_t mul;
  int shift;
  static FastDiv of(int d) {
    int l = 0;
    while ((int64_t(1) << l) < d) ++l;
    return FastDiv{(uint32_t)((uint64_t(1) << (31 + l)) / (uint64_t)d + 1), 31 + l};
  }
  KIV_HD int div(int n) const { return (int)(((uint64_t)(uint32_t)n * mul) >> shift); }
};

// A sequence as the kernels take it: its packed rows [q0, q0 + qlen), brought
// into range whatever the arrays hold, and its keys up to the last of those
// (the whole length, less the rows behind the call's; then maybe negative).
struct PagedSeq {
  int q0, qlen, len;
};

// A unit is the query rows of one kv head that one block (or several, over
// shares of its keys) attends together: tpu tokens times the G query heads of
// the kv head, at most `rows` rows; with more heads than rows, one token and
// one of hpt groups of heads.  Row r of a unit is its token r / gw, head
// r % gw.  The units of a sequence are numbered kv heads first, then tokens
// (neighbouring shares read the same keys), then head groups.
struct PagedShape {
  int total_q, hkv, G;
  int rows, tpu, hpt, gw;
  int cap;         // keys the block table spans
  int tile_shift;  // keys of a tile: 1 << tile_shift
  int window;      // 0: none
  int whole;       // a unit is never divided (its weight is one)
  int fixed;       // tiles that a unit's first loads and its stores cost

  static PagedShape of(int total_q, int hkv, int G, int rows, int cap, int tile_shift, int window, bool whole,
                       int fixed) {
    PagedShape s;
    s.total_q = total_q;
    s.hkv = hkv;
    s.G = G;
    s.rows = rows;
    s.tpu = G < rows ? rows / G : 1;
    s.hpt = (G + rows - 1) / rows;
    s.gw = G < rows ? G : rows;
    s.cap = cap;
    s.tile_shift = tile_shift;
    s.window = window;
    s.whole = whole;
    s.fixed = fixed;
    return s;
  }
  KIV_HD PagedSeq seq(int cu0, int cu1, int len) const {
    PagedSeq q;
    q.q0 = cu0 < 0 ? 0 : cu0 > total_q ? total_q : cu0;
    const int end = cu1 < 0 ? 0 : cu1 > total_q ? total_q : cu1;
    q.qlen = end > q.q0 ? end - q.q0 : 0;
    // Row r has key kv_len - cu_q[b + 1] + r; a negative length has no keys, as
    // a length of 0.
    q.len = (len < 0 ? 0 : len) - (q.qlen > 0 ? cu1 - end : 0);
    return q;
  }
  // Units of one kv head of a sequence.
  KIV_HD int row_tiles(const PagedSeq &s) const { return (s.qlen + tpu - 1) / tpu * hpt; }
  KIV_HD int token0(int rt) const { return (hpt == 1 ? rt : rt / hpt) * tpu; }
  KIV_HD int tokens(const PagedSeq &s, int tok0) const { return s.qlen - tok0 < tpu ? s.qlen - tok0 : tpu; }
  // Keys [k0, k1) that some row of unit rt sees.
  KIV_HD void keys(const PagedSeq &s, int rt, int &k0, int &k1) const {
    const int tok0 = token0(rt), from = s.len - s.qlen + tok0;  // the first token's key
    const int last = from + tokens(s, tok0);
    k1 = last < 0 ? 0 : last < cap ? last : cap;
    k0 = window > 0 && from >= window ? from - window + 1 : 0;
    if (k0 >= k1) k0 = k1 = 0;
  }
  // First tile and number of tiles of the keys [k0, k1); a unit that sees no
  // key has one, so that a block writes its rows.
  KIV_HD int first_tile(int k0) const { return k0 >> tile_shift; }
  KIV_HD int tiles(int k0, int k1) const { return k0 < k1 ? ((k1 - 1) >> tile_shift) - (k0 >> tile_shift) + 1 : 1; }
  // A unit's weight: its fixed cost, then its tiles.
  KIV_HD int weight(const PagedSeq &s, int rt) const {
    if (whole) return 1;
    int k0, k1;
    keys(s, rt, k0, k1);
    return fixed + tiles(k0, k1);
  }
  // The unit's tiles before its weight w (counted from its first).
  KIV_HD int tiles_before(int w) const { return w > fixed ? w - fixed : 0; }
};

// The weights 0 .. total - 1 in n shares, equal to within one: block i takes
// [start(i), start(i + 1)).
struct PagedShares {
  int total, n, per, rem;
  // Dealt to at most `most` blocks, none without a weight; many blocks are a
  // multiple of the eight dies, unless a block then had a second whole unit.
  KIV_HD static PagedShares deal(int total, int most, bool whole) {
    PagedShares s;
    const int m = total < most ? total : most;
    s.total = total;
    s.n = m >= 64 && !(whole && m == total) ? m & ~7 : m;
    s.per = total / s.n;
    s.rem = total - s.per * s.n;
    return s;
  }
  KIV_HD int start(int i) const { return i * per + (i < rem ? i : rem); }
  KIV_HD int block_of(int w) const {
    const int longer = rem * (per + 1);  // weights of the shares that are one longer
    return w < longer ? w / (per + 1) : rem + (w - longer) / per;
  }
};

}  // namespace kiv
