// Attention of a ragged batch of new tokens over a paged K/V cache.
//
//   o_r = sum_j p_rj v_j,  p_rj = exp(s_rj - m_r) / sum_j exp(s_rj - m_r),
//   s_rj = scaling * q_r . k_j over the keys j that row r sees (the causal
//   rule, a sliding window, pages that are there), m_r their maximum.
//
// One pass over the keys with a running maximum and sum (base 2, fp32); the
// query heads of one kv head are rows of one unit (kiv_paged_plan.h), so each
// K and V row is read once for all of them.  The work of a call, in tiles of
// keys (a unit's first loads and stores count as some more), is dealt to the
// blocks in equal shares: a block finds its share from the sequences' lengths
// itself (no launch, no host copy), takes its units one after the other, and a
// unit that a share's end cuts is merged from partial rows by
// paged_combine_kernel.  Short units go whole, in one launch.
//
// paged_rows_kernel (single tokens, few rows, fp32): units of 16 rows, tiles
// of 128 keys.  Each of a block's four waves takes 32 keys of a tile on its
// own: K rows straight into registers as matrix operands, V rows through
// registers into the wave's own LDS (read back transposed), the next tile's
// rows in flight under this tile's softmax, no barrier until a unit ends.
//   S^T = K Q^T with 16x16 matrix instructions: lane l gives key l % 16 of a
//   16-key sub-tile (A) and query row l % 16 (B), 16-byte chunks l / 16 + 4 st
//   of both, and receives keys 4 (l / 16) + i of the sub-tile for row l % 16.
//   O^T += V^T P^T: B is the lane's own probabilities (with 16-bit types in
//   two operands), A the same keys of dim l % 16 from the LDS.
// Bound: memory (each K and V byte is used by at most 16 rows): 64 sequences
// of up to 8192 keys, 28 heads over 4 of 128, 95 us (5.4 TB/s); one token over
// a million keys 357 us (6.0 TB/s); both without the merge.
#include <algorithm>
#include <climits>
#include <type_traits>

#include "kiv_common.h"
#include "kiv_internal.h"
#include "kiv_paged_plan.h"

namespace kiv {

constexpr int kPgThreads = 256;
constexpr int kPgWaves = kPgThreads / 64;
constexpr float kPgLog2e = 1.4426950408889634f;
// Probabilities are 2^(s - m), m a running maximum of the scores less kPgLift,
// moved when a score exceeds m by more than kPgRoom.  As fp16 operands they
// lose bits below 2^-14 and are 0 below 2^-25, while their fp32 sum keeps them:
// without a lift, keys 17 nats under the maximum counted in the denominator
// and not, or up to twice, in the numerator.  Lifted by 2^11 (and at most 2^15,
// fp16 holds 2^16) they keep every bit down to 2^-25 of the maximum and are
// there down to 2^-36; the factor cancels in o / l.  The headroom this leaves,
// 2^4 where the other types have 2^8, costs nothing: chunks and tokens mixed
// (9 sequences of up to 4099 keys, 32 heads over 8) 104.9 us, 104.5 before; 301
// keys 6.6, 7.1.
template <int DT> constexpr float kPgLift = DT == DT_F16 ? 11.f : 0.f;
template <int DT> constexpr float kPgRoom = DT == DT_F16 ? 15.f : 8.f;
constexpr int kRowsTileShift = 7;  // the rows kernel's tile: 128 keys
constexpr int kRowsOfUnit = 16;

// What the combine needs of a unit that block i continues: written by every
// block (last < 0: nothing to merge here).
struct PagedCut {
  int row0, tokens, head0, heads;  // first packed row, tokens, first query head, heads (rows: tokens x heads)
  int last;                        // the last block that has a part of it
  int pad[3];
};

struct PagedAttnParams {
  const char *q;
  int64_t q_t, q_h;  // byte strides
  const char *k, *v;
  int64_t page_b, head_b, tok_b;  // byte strides of the pool
  const int32_t *cu, *kv_len, *table;
  int64_t table_stride;
  int seqs, num_pages, page_size, hq;
  FastDiv page_div;
  PagedShape sh;
  int blocks;  // most blocks that share the work
  float scale_log2;
  char *out;
  PagedCut *cuts;  // [blocks]
  float *ws_m, *ws_l, *ws_o;  // [2 blocks][rows], [2 blocks][rows][D]
};

// A row of zeros that stands for keys that are not there.
__device__ const uint4 paged_zero_row[64] = {};

__device__ __forceinline__ int uniform_i32(int x) { return __builtin_amdgcn_readfirstlane(x); }

// Weight of a sequence's units of one kv head, by the whole wave (each lane
// its own sequence; long ones by all lanes together).
__device__ __forceinline__ int paged_seq_weight(const PagedShape &sh, const PagedSeq &s) {
  const int nrt = sh.row_tiles(s);
  if (sh.whole) return nrt;
  constexpr int kSerial = 2;
  int w = 0;
  if (nrt <= kSerial)
    for (int rt = 0; rt < nrt; ++rt) w += sh.weight(s, rt);
  const int lane = threadIdx.x & 63;
  for (uint64_t m = __ballot(nrt > kSerial); m; m &= m - 1) {
    const int l = __builtin_ctzll(m), n = __builtin_amdgcn_readlane(nrt, l);
    const PagedSeq o{0, __builtin_amdgcn_readlane(s.qlen, l), __builtin_amdgcn_readlane(s.len, l)};
    int sum = 0;
    for (int rt = lane; rt < n; rt += 64) sum += sh.weight(o, rt);
    sum = wave_sum_i32(sum);
    if (lane == l) w = sum;
  }
  return w;
}

__device__ __forceinline__ PagedSeq paged_seq(const PagedAttnParams &p, int b) {
  return b < p.seqs ? p.sh.seq(p.cu[b], p.cu[b + 1], p.kv_len[b]) : PagedSeq{0, 0, 0};
}

// A block's place in the work: the unit it is at and what is left of its share.
struct PagedWork {
  int id;           // which share
  int b, kvh, rt;   // the unit
  PagedSeq s;
  int nrt;
  int w, w_end, us;  // the share's next weight and end; the unit's first weight
  PagedShares shares;

  // Called by the whole block; false: there is no share for it.  Up to 64
  // sequences every wave sums for itself; more meet in LDS.
  __device__ __forceinline__ bool first(const PagedAttnParams &p) {
    __shared__ int sums[kPgWaves], found[3];
    __shared__ float fsums[kPgWaves];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const PagedShape &sh = p.sh;
    int seq_at, seq_w;  // the sequence's first weight, and all of them
    if (p.seqs <= 64) {
      const PagedSeq my = paged_seq(p, lane);
      const int mine = sh.hkv * paged_seq_weight(sh, my), incl = wave_incl_scan(mine);
      if (!deal(p, __builtin_amdgcn_readlane(incl, 63), wave_sum((float)mine))) return false;
      b = __builtin_ctzll(__ballot(incl > w));
      seq_w = __builtin_amdgcn_readlane(mine, b);
      seq_at = __builtin_amdgcn_readlane(incl, b) - seq_w;
      s.q0 = __builtin_amdgcn_readlane(my.q0, b);
      s.qlen = __builtin_amdgcn_readlane(my.qlen, b);
      s.len = __builtin_amdgcn_readlane(my.len, b);
    } else {
      int mine = 0, incl = 0, total = 0;
      float ftotal = 0.f;
      for (int base = 0; base < p.seqs; base += kPgThreads) {
        mine = sh.hkv * paged_seq_weight(sh, paged_seq(p, base + tid));
        const float f = wave_sum((float)mine);
        __syncthreads();
        if (lane == 0) fsums[wave] = f;
        total += scan(mine, incl, sums, wave, lane);
#pragma unroll
        for (int i = 0; i < kPgWaves; ++i) ftotal += fsums[i];
      }
      if (!deal(p, total, ftotal)) return false;
      int before = 0;
      for (int base = 0; base < p.seqs; base += kPgThreads) {
        int sum = total;
        if (p.seqs > kPgThreads) {
          mine = sh.hkv * paged_seq_weight(sh, paged_seq(p, base + tid));
          sum = scan(mine, incl, sums, wave, lane);
        }
        const int end = before + incl;
        if (w < end && w >= end - mine) {
          found[0] = base + tid;
          found[1] = end - mine;
          found[2] = mine;
        }
        before += sum;
        if (w < before) break;
      }
      __syncthreads();
      b = uniform_i32(found[0]);
      seq_at = uniform_i32(found[1]);
      seq_w = uniform_i32(found[2]);
      load_seq(p);
    }
    nrt = sh.row_tiles(s);
    const int per_head = seq_w / sh.hkv;
    kvh = (w - seq_at) / per_head;
    int r = w - seq_at - kvh * per_head;  // weights of the head's units before w
    if (sh.whole) {
      rt = r;
      us = w;
      return true;
    }
    for (rt = 0;; rt += 64) {
      const int n = rt + lane < nrt ? sh.weight(s, rt + lane) : 0, up = wave_incl_scan(n);
      const uint64_t past = __ballot(up > r);
      if (past) {
        const int l = __builtin_ctzll(past);
        rt += l;
        us = w - (r - (__builtin_amdgcn_readlane(up, l) - __builtin_amdgcn_readlane(n, l)));
        return true;
      }
      r -= __builtin_amdgcn_readlane(up, 63);
    }
  }
  // This block's share of `total` (ftotal: the same sum in floating point, by
  // which lengths in disorder, whose sum passes 2^31, are known: a batch in
  // order stays below by the host's check).
  __device__ __forceinline__ bool deal(const PagedAttnParams &p, int total, float ftotal) {
    if (total <= 0 || ftotal > 2.1e9f) return false;
    shares = PagedShares::deal(total, p.blocks, p.sh.whole);
    if ((int)blockIdx.x >= shares.n) return false;
    // Blocks are dealt to the eight dies in turn: a die takes neighbouring
    // shares, which read the same keys through its L2.
    id = !(shares.n & 7) ? ((int)blockIdx.x & 7) * (shares.n >> 3) + ((int)blockIdx.x >> 3) : (int)blockIdx.x;
    w = shares.start(id);
    w_end = shares.start(id + 1);
    return true;
  }
  // Inclusive sums over the block's threads; returns the block's.
  static __device__ __forceinline__ int scan(int x, int &incl, int *sums, int wave, int lane) {
    incl = wave_incl_scan(x);
    __syncthreads();
    if (lane == 63) sums[wave] = incl;
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int i = 0; i < kPgWaves; ++i) {
      const int t = sums[i];
      if (i < wave) incl += t;
      all += t;
    }
    return uniform_i32(all);
  }
  __device__ __forceinline__ void load_seq(const PagedAttnParams &p) {
    s = paged_seq(p, b);
    s.q0 = uniform_i32(s.q0);
    s.qlen = uniform_i32(s.qlen);
    s.len = uniform_i32(s.len);
  }
  // The unit behind this one; called while w < w_end.
  __device__ __forceinline__ void next(const PagedAttnParams &p) {
    us = w;
    if (++rt < nrt) return;
    rt = 0;
    if (++kvh < p.sh.hkv) return;
    kvh = 0;
    do {
      ++b;
      load_seq(p);
      nrt = p.sh.row_tiles(s);
    } while (nrt == 0 && b < p.seqs);
  }
};

// One unit's rows and keys.
struct PagedUnit {
  int row0, tokens, head0, heads;  // first packed row, tokens, first query head, heads
  int gw;
  int last0;       // last key that the first token sees
  int k0, k1;      // keys that some row sees
  __device__ __forceinline__ PagedUnit(const PagedShape &sh, const PagedSeq &s, int kvh, int rt) {
    const int tok0 = sh.token0(rt), hg = sh.hpt == 1 ? 0 : rt % sh.hpt;
    row0 = s.q0 + tok0;
    tokens = sh.tokens(s, tok0);
    head0 = kvh * sh.G + hg * sh.rows;
    heads = min(sh.gw, sh.G - hg * sh.rows);
    gw = sh.gw;
    last0 = s.len - s.qlen + tok0;
    sh.keys(s, rt, k0, k1);
  }
  // Packed row and query head of row r; false: the unit has no such row.
  __device__ __forceinline__ bool row(int r, int &t, int &h) const {
    const int tok = r / gw, g = r - tok * gw;
    t = row0 + tok;
    h = head0 + g;
    return tok < tokens && g < heads;
  }
};

// This block's part of a unit is [t0, t1) of its tiles: whole, or partial
// rows in slot `partial`: 2 i of block i's first fragment where the unit
// began before it, 2 i + 1 of the unit that goes on behind it.
struct PagedPart {
  int t0, t1, partial;
  __device__ __forceinline__ PagedPart(const PagedAttnParams &p, PagedWork &wk, const PagedUnit &u) {
    const int first = p.sh.first_tile(u.k0), n = p.sh.tiles(u.k0, u.k1);
    if (p.sh.whole) {
      t0 = first;
      t1 = first + n;
      partial = -1;
      ++wk.w;
      return;
    }
    const int end = min(wk.w_end, wk.us + p.sh.fixed + n);
    const int before = p.sh.tiles_before(wk.w - wk.us), upto = p.sh.tiles_before(end - wk.us);
    t0 = first + before;
    t1 = first + upto;  // t0 where the share ends in the unit's fixed weight: the next share has its first tile
    partial = before > 0 ? 2 * wk.id : upto < n ? 2 * wk.id + 1 : -1;
    wk.w = end;
  }
};

// The cut in front of block id's share, if the block before it has the unit's
// first tile.
__device__ __forceinline__ void paged_write_cut(const PagedAttnParams &p, const PagedWork &wk, const PagedUnit &u) {
  if (!p.cuts || threadIdx.x != 0) return;
  PagedCut c = {u.row0, u.tokens, u.head0, u.heads, -1, {0, 0, 0}};
  if (p.sh.tiles_before(wk.w - wk.us) > 0 && p.sh.tiles_before(wk.shares.start(wk.id - 1) - wk.us) == 0)
    c.last = wk.shares.block_of(wk.us + p.sh.fixed + p.sh.tiles(u.k0, u.k1) - 1);
  p.cuts[wk.id] = c;
}
__device__ __forceinline__ void paged_no_cut(const PagedAttnParams &p, int id) {
  if (p.cuts && threadIdx.x == 0) p.cuts[id].last = -1;
}

template <int DT> __device__ __forceinline__ void store4(char *out, int64_t elem, const f32x4_t &o) {
  if constexpr (DT == DT_F32) *reinterpret_cast<f32x4_t *>(out + 4 * elem) = o;
  else *reinterpret_cast<uint2 *>(out + 2 * elem) = make_uint2(pack2<DT>(o[0], o[1]), pack2<DT>(o[2], o[3]));
}

// ---------------------------------------------------------------------------
// Units of 16 rows.
template <int DT, int D> struct RowsGeom {
  static constexpr int EB = Elem<DT>::BYTES, RB = D * EB;  // bytes of a row
  static constexpr int ST = RB / 64;                       // 64-byte steps of a row
  static constexpr int VS = RB + 32;                       // LDS row stride: neighbouring keys 8 banks apart
  static constexpr int ND = D / 16;
  static constexpr int WAVE = 32 * VS;                     // LDS bytes of a wave: 32 V rows, later its 16 x D sums
  static_assert(16 * D * 4 <= WAVE, "a wave's sums fit its V rows");
};

// acc += A B over one 64-byte step.
template <int DT> __device__ __forceinline__ f32x4_t step_16x16(const uint4 &a, const uint4 &b, f32x4_t c) {
  if constexpr (DT == DT_F32) {
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.x), __uint_as_float(b.x), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.y), __uint_as_float(b.y), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.z), __uint_as_float(b.z), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.w), __uint_as_float(b.w), c, 0, 0, 0);
  } else {
    return mfma_16x16x32<DT>(a, b, c);
  }
}

// What a and b lose in hi = pack2(a, b), packed alike.
template <int DT> __device__ __forceinline__ uint32_t pack2_rest(float a, float b, uint32_t hi) {
  if constexpr (DT == DT_BF16) {
    return pack2<DT>(a - __uint_as_float(hi << 16), b - __uint_as_float(hi & 0xffff0000u));
  } else {
    const f16x2_t h = __builtin_bit_cast(f16x2_t, hi);
    return pack2<DT>(a - (float)h[0], b - (float)h[1]);
  }
}

template <int DT, int D>
__global__ void __launch_bounds__(kPgThreads) __attribute__((amdgpu_waves_per_eu(1, 4)))
paged_rows_kernel(PagedAttnParams p) {
  using Geo = RowsGeom<DT, D>;
  constexpr int ST = Geo::ST, VS = Geo::VS, ND = Geo::ND;
  __shared__ __align__(16) char vs[kPgWaves][Geo::WAVE];
  __shared__ float wm[kPgWaves][16], wl[kPgWaves][16];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int col = lane & 15, grp = lane >> 4;
  char *lds = vs[wave];
  PagedWork wk;
  if (!wk.first(p)) {
    paged_no_cut(p, blockIdx.x);
    return;
  }
  bool head = true;
  while (wk.w < wk.w_end) {
    const PagedUnit u(p.sh, wk.s, wk.kvh, wk.rt);
    if (head) paged_write_cut(p, wk, u);
    head = false;
    const PagedPart part(p, wk, u);
    if (part.t0 == part.t1) break;  // the share ends before the unit's first tile
    // The lane's query row (rows the unit has not repeat its first).
    int qt, qh;
    const bool own = u.row(col, qt, qh);
    const char *qp = p.q + (own ? qt : u.row0) * p.q_t + (own ? qh : u.head0) * p.q_h + 16 * grp;
    uint4 qx[ST];
#pragma unroll
    for (int st = 0; st < ST; ++st) qx[st] = load16(qp + 64 * st);
    const int last = u.last0 + (own ? qt - u.row0 : 0);
    const int from = p.sh.window > 0 && last >= p.sh.window ? last - p.sh.window : -1;
    const int32_t *table = p.table + wk.b * p.table_stride;
    const char *kb = p.k + wk.kvh * p.head_b, *vb = p.v + wk.kvh * p.head_b;

    f32x4_t o[ND];
#pragma unroll
    for (int dt = 0; dt < ND; ++dt) o[dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    float m_run = -INFINITY, l_lane = 0.f;

    // The wave's 32 keys of tile t; the lane's are key0 + col and key0 + 16 +
    // col: their pages' numbers (loaded two tiles ahead), then their rows.
    auto key_of = [&](int t, int sub) { return (t << kRowsTileShift) + 32 * wave + 16 * sub + col; };
    auto lookup = [&](int t, int (&page)[2]) {
#pragma unroll
      for (int sub = 0; sub < 2; ++sub) {
        const int key = key_of(t, sub);
        page[sub] = t < part.t1 && key >= u.k0 && key < u.k1 ? table[p.page_div.div(key)] : -1;
      }
    };
    const char *kp[2], *vp[2];
    uint32_t there = 0;  // of the tile in flight: bit 16 sub + k: its key k of sub-tile sub is there
    auto resolve = [&](int t, const int (&page)[2]) {
      there = 0;
#pragma unroll
      for (int sub = 0; sub < 2; ++sub) {
        const int key = key_of(t, sub);
        const bool in = page[sub] >= 0 && page[sub] < p.num_pages;
        const int slot = key - p.page_div.div(key) * p.page_size;
        const int64_t off = page[sub] * p.page_b + slot * p.tok_b + 16 * grp;
        const char *zero = reinterpret_cast<const char *>(paged_zero_row) + 16 * grp;
        kp[sub] = in ? kb + off : zero;
        vp[sub] = in ? vb + off : zero;
        there |= (uint32_t)(__ballot(in) & 0xffffu) << (16 * sub);
      }
    };
    uint4 kx[2][ST], vx[2][ST];
    auto load_k = [&] {
#pragma unroll
      for (int sub = 0; sub < 2; ++sub)
#pragma unroll
        for (int st = 0; st < ST; ++st) kx[sub][st] = load16(kp[sub] + 64 * st);
    };
    auto load_v = [&] {
#pragma unroll
      for (int sub = 0; sub < 2; ++sub)
#pragma unroll
        for (int st = 0; st < ST; ++st) vx[sub][st] = load16(vp[sub] + 64 * st);
    };
    int page[2];
    lookup(part.t0, page);
    resolve(part.t0, page);
    lookup(part.t0 + 1, page);
    load_k();
    load_v();
    for (int t = part.t0; t < part.t1; ++t) {
      const uint32_t seen = there;
      f32x4_t s[2];
#pragma unroll
      for (int sub = 0; sub < 2; ++sub) {
        s[sub] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int st = 0; st < ST; ++st) s[sub] = step_16x16<DT>(kx[sub][st], qx[st], s[sub]);
      }
      const bool more = t + 1 < part.t1;
      if (more) {
        resolve(t + 1, page);
        lookup(t + 2, page);
        load_k();
      }
      // V rows to LDS (this wave's alone; its reads of the tile before come
      // first in the LDS queue).
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
      for (int sub = 0; sub < 2; ++sub)
#pragma unroll
        for (int st = 0; st < ST; ++st)
          *reinterpret_cast<uint4 *>(lds + (16 * sub + col) * VS + 64 * st + 16 * grp) = vx[sub][st];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      if (more) load_v();

      // Scores in base 2; keys that the row does not see are -inf.
      const int key0 = key_of(t, 0) - col;
      const bool edge = u.tokens > 1 && (key0 + 31 > u.last0 ||
                                         (p.sh.window > 0 && key0 + p.sh.window <= u.last0 + u.tokens - 1));
#pragma unroll
      for (int sub = 0; sub < 2; ++sub)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[sub][i] *= p.scale_log2;
      if (edge || seen != ~0u) {
#pragma unroll
        for (int sub = 0; sub < 2; ++sub)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int at = 16 * sub + 4 * grp + i, key = key0 + at;
            if (!((seen >> at) & 1u) || key > last || key <= from) s[sub][i] = -INFINITY;
          }
      }
      // The running max moves only when a score exceeds it by 2^kPgRoom.
      float x = s[0][0];
#pragma unroll
      for (int i = 1; i < 4; ++i) x = fmaxf(x, s[0][i]);
#pragma unroll
      for (int i = 0; i < 4; ++i) x = fmaxf(x, s[1][i]);
      if (__ballot(x > m_run + kPgRoom<DT>)) {
        const float mt = half_wave_max(row_pair_max(x));
        const float m_new = mt > m_run + kPgRoom<DT> ? mt - kPgLift<DT> : m_run;
        const float a = m_run == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_run - m_new);
        l_lane *= a;
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) o[dt] *= a;
        m_run = m_new;
      }
      const float m_neg = m_run == -INFINITY ? 0.f : -m_run;
      float e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        e[i] = __builtin_amdgcn_exp2f(s[i >> 2][i & 3] + m_neg);
        l_lane += e[i];
      }
      if constexpr (DT == DT_F32) {
        const char *at = lds + 4 * grp * VS + 4 * col;
#pragma unroll
        for (int dt = 0; dt < ND; ++dt)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float a = *reinterpret_cast<const float *>(at + (16 * (i >> 2) + (i & 3)) * VS + 64 * dt);
            o[dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(a, e[i], o[dt], 0, 0, 0);
          }
      } else {
        // Probabilities as two operands of the dtype, their rounding and what
        // it left, which together hold them to 2^-16 (fp16 2^-22).  The second
        // product hides under the loads: 64 sequences of up to 8192 keys 101.0
        // us, 100.9 without; a million keys 380.6, 380.1; 301 keys 7.6, 7.6.
        const uint4 pb = make_uint4(pack2<DT>(e[0], e[1]), pack2<DT>(e[2], e[3]), pack2<DT>(e[4], e[5]),
                                    pack2<DT>(e[6], e[7]));
        const uint4 pr = make_uint4(pack2_rest<DT>(e[0], e[1], pb.x), pack2_rest<DT>(e[2], e[3], pb.y),
                                    pack2_rest<DT>(e[4], e[5], pb.z), pack2_rest<DT>(e[6], e[7], pb.w));
        const char *at = lds + (4 * grp + (col >> 2)) * VS + 8 * (col & 3);
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) {
          const uint2 lo =
              __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_t *)(at + 32 * dt)));
          const uint2 hi = __builtin_bit_cast(
              uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_t *)(at + 16 * VS + 32 * dt)));
          const uint4 vt = make_uint4(lo.x, lo.y, hi.x, hi.y);
          o[dt] = mfma_16x16x32<DT>(vt, pb, o[dt]);
          o[dt] = mfma_16x16x32<DT>(vt, pr, o[dt]);
        }
      }
    }

    // The four waves' sums meet in LDS.
    const float l_row = half_wave_sum(row_pair_sum(l_lane));
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    float *os = reinterpret_cast<float *>(lds);
#pragma unroll
    for (int dt = 0; dt < ND; ++dt) *reinterpret_cast<f32x4_t *>(os + col * D + 16 * dt + 4 * grp) = o[dt];
    if (grp == 0) {
      wm[wave][col] = m_run;
      wl[wave][col] = l_row;
    }
    __syncthreads();
    for (int i = tid; i < 16 * (D / 4); i += kPgThreads) {
      const int r = i / (D / 4), d0 = 4 * (i - r * (D / 4));
      int rt, rh;
      if (!u.row(r, rt, rh)) continue;
      float M = wm[0][r];
#pragma unroll
      for (int w = 1; w < kPgWaves; ++w) M = fmaxf(M, wm[w][r]);
      float L = 0.f;
      f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kPgWaves; ++w) {
        const float c = wm[w][r] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(wm[w][r] - M);
        L = fmaf(c, wl[w][r], L);
        acc += c * *reinterpret_cast<const f32x4_t *>(reinterpret_cast<const float *>(vs[w]) + r * D + d0);
      }
      if (part.partial >= 0) {
        const int64_t sr = (int64_t)part.partial * kRowsOfUnit + r;
        *reinterpret_cast<f32x4_t *>(p.ws_o + sr * D + d0) = acc;
        if (d0 == 0) {
          p.ws_m[sr] = M;
          p.ws_l[sr] = L;
        }
      } else {
        // A row that sees no key gets zeros.
        const float inv = L > 0.f ? 1.f / L : 0.f;
        store4<DT>(p.out, ((int64_t)rt * p.hq + rh) * D + d0, acc * inv);
      }
    }
    __syncthreads();  // the next unit's V rows reuse the LDS
    if (wk.w < wk.w_end) wk.next(p);
  }
}

// ---------------------------------------------------------------------------
// Units of 128 rows (16-bit types): 4 waves of 32.
//
// K and V tiles of 64 keys go from their pages straight to LDS, as rows,
// double-buffered, their 16-byte chunks permuted so that operand reads spread
// over the banks (K chunk c of row r at c ^ xk(r), V chunk c at c ^ 4 xv(r):
// the loading lanes fetch the permuted chunk).
//   S^T = K Q^T with 32x32 matrix instructions: lane l gives row l % 32 of a
//   32-key sub-tile of K (A) and its own query row l % 32 (B, in registers
//   for the whole unit), dims 16 st + 8 (l / 32) .. + 7 of step st, and
//   receives keys 8 (i / 4) + 4 (l / 32) + i % 4 (i < 16) for its row.
//   O^T += V^T P^T, 16 keys a step: B is the lane's own probabilities, A the
//   same keys of dim l % 32 from two transposing LDS reads.
// One iteration forms the scores of the next tile beside the exponentials of
// this one, then adds this tile's values beside the next one's maxima, so
// that vector and matrix instructions alternate in one wave's stream.
// Bound: neither unit is full (matrix cores busy 51% of the cycles): 4096 tokens
// over 8192 keys, 12 heads over 2 of 128, 338,000 cycles: 168 us at 2.0 GHz, 200
// after a dozen calls back to back, whose matrix work lowers the clock; a call
// with the merge 174 to 200 us, 770 to 890 TFLOP/s, 1 PFLOP/s on long keys.  Two
// waves a SIMD: the registers hold no third.
template <int KT> struct ChunkGeom {
  static constexpr int D = 32 * KT, CPR = D / 8;
  static constexpr int CP = CPR <= 4 ? 4 : CPR <= 8 ? 8 : CPR <= 16 ? 16 : 32;  // chunks of an LDS row
  static constexpr int RPI = 64 / CP;   // rows of a load instruction
  static constexpr int NJ = CP / 4;     // load instructions of a wave for a tile of K (of V)
  static constexpr int TILE = 64 * CP * 16;  // LDS bytes of a tile
  static constexpr int KS = D / 16, ND = D / 32;
  static __device__ __forceinline__ int xk(int r) { return CP >= 16 ? r & 15 : (r / (16 / CP)) & (CP - 1); }
  static __device__ __forceinline__ int xv(int r) { return CP >= 16 ? r & 3 : CP == 8 ? (r >> 1) & 1 : 0; }
};
constexpr int kChunkTileShift = 6;
constexpr int kPgWaitAll = 0x0070;  // s_waitcnt vmcnt(0) lgkmcnt(0)

// Keeps x's computation where it is written: the compiler otherwise moves it
// behind the next branch, to where x is used, and with it the vector
// instructions that are to issue between matrix instructions.
template <typename T> __device__ __forceinline__ void stay(T &x) { asm volatile("" : "+v"(x)); }

template <int DT, int KT>
__global__ void __launch_bounds__(kPgThreads, KT <= 4 ? 2 : 1) paged_chunk_kernel(PagedAttnParams p) {
  using Geo = ChunkGeom<KT>;
  constexpr int D = Geo::D, CP = Geo::CP, CPR = Geo::CPR, RPI = Geo::RPI, NJ = Geo::NJ, KS = Geo::KS, ND = Geo::ND;
  // Objects of their own, so that the compiler knows that reads of one do not
  // wait for loads into another.
  __shared__ __align__(1024) char kb0[Geo::TILE], kb1[Geo::TILE], vb0[Geo::TILE], vb1[Geo::TILE];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int row = lane & 31, hf = lane >> 5;
  PagedWork wk;
  if (!wk.first(p)) {
    paged_no_cut(p, blockIdx.x);
    return;
  }
  // Loads: the lane's row of the wave's first instruction (the next ones are
  // 4 RPI rows on) and its chunks' bytes; with 32 chunks the rows' K
  // permutation alternates.
  const int lrow = wave * RPI + lane / CP, pc = lane % CP;
  const uint32_t in_group = (uint32_t)(lane / CP) * (uint32_t)p.tok_b;  // the lane's row from its group's first
  const uint32_t kc0 = min(pc ^ Geo::xk(lrow), CPR - 1) * 16, kc1 = min(pc ^ Geo::xk(lrow + 4 * RPI), CPR - 1) * 16;
  const uint32_t vc = min(pc ^ (4 * Geo::xv(lrow)), CPR - 1) * 16;
  // Operand reads: the lane's byte offsets within a tile.
  const int kaddr = row * CP * 16 + ((hf ^ Geo::xk(row)) << 4);
  int vaddr[ND];
#pragma unroll
  for (int dt = 0; dt < ND; ++dt) {
    const int j16 = lane & 15, q = j16 >> 2;  // the transposing read: key q of four, dims 4 (j16 % 4) ..
    const int c = 4 * (dt ^ Geo::xv(q)) + 2 * ((lane >> 4) & 1) + ((j16 & 3) >> 1);
    vaddr[dt] = (4 * hf + q) * CP * 16 + c * 16 + (j16 & 1) * 8;
  }
  const bool one_page = p.page_size % 64 == 0;  // a tile lies in one page
  const float cc = p.scale_log2;
  bool head = true;
  while (wk.w < wk.w_end) {
    const PagedUnit u(p.sh, wk.s, wk.kvh, wk.rt);
    if (head) paged_write_cut(p, wk, u);
    head = false;
    const PagedPart part(p, wk, u);
    if (part.t0 == part.t1) break;  // the share ends before the unit's first tile
    const int32_t *table = p.table + wk.b * p.table_stride;
    const char *kbase = p.k + wk.kvh * p.head_b, *vbase = p.v + wk.kvh * p.head_b;

    // Pages of tile t's keys, a key a lane (-1 past the table).
    auto lookup = [&](int t) {
      const int key = (t << kChunkTileShift) + lane;
      return t < part.t1 && key < p.sh.cap ? table[p.page_div.div(key)] : -1;
    };
    // Where those keys' rows lie in the pool, a key a lane, and which of them
    // are there (and seen by some row of the unit).
    auto locate = [&](int t, int page, int64_t &off, uint64_t &there) {
      const int key = (t << kChunkTileShift) + lane, slot = key - p.page_div.div(key) * p.page_size;
      off = (int64_t)page * p.page_b + (int64_t)slot * p.tok_b;
      there = __ballot(page >= 0 && page < p.num_pages && key >= u.k0 && key < u.k1);
    };
    // Starts the loads of a tile of K or V into LDS: a load instruction's rows
    // lie in one page, so its addresses are that page's (in scalar registers)
    // and the lanes' fixed offsets.  Keys that are not there are given the row
    // of one that is (zeros if there is none): neither their stale rows nor
    // other sequences' are read.
    auto load = [&](int64_t off, uint64_t there, const char *base, char *to, uint32_t c0, uint32_t c1) {
      auto row_at = [&](int r) {
        const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)off, r);
        const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(off >> 32), r);
        return tile_rsrc(base + (int64_t)((uint64_t)hi << 32 | lo), 0xffffffffu);
      };
      auto put = [&](__amdgpu_buffer_rsrc_t rs, int j, uint32_t voff, uint32_t soff) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void_t *)(to + (j * 4 + wave) * 1024), 16,
                                                 (int)(voff + (j & 1 ? c1 : c0)), (int)soff, 0, 0);
      };
      if (there == ~uint64_t(0)) {
        if (one_page) {
          const auto rs = row_at(0);
#pragma unroll
          for (int j = 0; j < NJ; ++j) put(rs, j, in_group, (uint32_t)((j * 4 + wave) * RPI) * (uint32_t)p.tok_b);
        } else {
#pragma unroll
          for (int j = 0; j < NJ; ++j) put(row_at((j * 4 + wave) * RPI), j, in_group, 0);
        }
        return;
      }
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int r0 = (j * 4 + wave) * RPI;
        const uint32_t in = (uint32_t)(there >> r0) & ((1u << RPI) - 1u);  // of the group: consecutive
        if (in) {
          const int lo = __builtin_ctz(in), hi = 31 - __builtin_clz(in);
          put(row_at(r0 + lo), j, (uint32_t)(min(max(lane / CP, lo), hi) - lo) * (uint32_t)p.tok_b, 0);
        } else if (there) {
          put(row_at(__builtin_ctzll(there)), j, 0, 0);
        } else {
          put(tile_rsrc(reinterpret_cast<const char *>(paged_zero_row), 0xffffffffu), j, 0, 0);
        }
      }
    };

    // The lane's query rows, their last keys, and the wave's tokens.
    int qt, qh;
    const bool own = u.row(32 * wave + row, qt, qh);
    uint4 qx[KS];
    const char *qp = p.q + (own ? qt : u.row0) * p.q_t + (own ? qh : u.head0) * p.q_h + 16 * hf;
#pragma unroll
    for (int st = 0; st < KS; ++st) qx[st] = load16(qp + 32 * st);
    const int tok = own ? qt - u.row0 : 0;
    const bool active = 32 * wave < u.tokens * u.gw;
    const int tok_a = min(32 * wave / u.gw, u.tokens - 1), tok_z = min((32 * wave + 31) / u.gw, u.tokens - 1);

    f32x16_t o[ND] = {};
    float m_run = -INFINITY, l_lane = 0.f;  // l_lane: this lane's share of the row sum

    // Hidden keys' scores of tile t become -inf.
    auto hide = [&](f32x16_t(&s)[2], int t, uint64_t there) {
      const int key0 = t << kChunkTileShift;
      const bool edge = key0 + 63 > u.last0 + tok_a || (p.sh.window > 0 && key0 + p.sh.window <= u.last0 + tok_z);
      if (!edge && there == ~uint64_t(0)) return;
      // Keys [lo, hi) of the tile; a window as long as the keys hides none.
      const int hi = u.last0 + tok + 1 - key0, lo = p.sh.window > 0 && hi > 0 ? hi - p.sh.window : 0;
      uint64_t v = hi >= 64 ? ~uint64_t(0) : hi <= 0 ? 0 : (uint64_t(1) << hi) - 1;
      if (lo > 0) v &= lo >= 64 ? 0 : ~uint64_t(0) << lo;
      v = (v & there) >> (4 * hf);
#pragma unroll
      for (int sub = 0; sub < 2; ++sub) {
        const uint32_t bits = (uint32_t)(v >> (32 * sub));
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (!(bits & (1u << (8 * (i >> 2) + (i & 3))))) s[sub][i] = -INFINITY;
      }
    };
    // Raises the running maximum (and rescales the sums) where a score exceeds
    // it by more than 2^kPgRoom.
    auto raise = [&](float x) {
      if (!__ballot(x * cc > m_run + kPgRoom<DT>)) return;
      const float mt = half_wave_max(x) * cc;
      const float m_new = mt > m_run + kPgRoom<DT> ? mt - kPgLift<DT> : m_run;
      const float a = m_run == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_run - m_new);
      l_lane *= a;
#pragma unroll
      for (int dt = 0; dt < ND; ++dt) o[dt] *= a;
      m_run = m_new;
    };
    auto k_op = [&](const char *kb, int i) {
      return *reinterpret_cast<const uint4 *>(kb + (kaddr ^ ((i % KS) << 5)) + (i / KS) * 32 * CP * 16);
    };
    auto v_op = [&](const char *vb, int k, int dt) {
      const char *at = vb + vaddr[dt] + 16 * k * CP * 16;
      const uint2 lo = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_t *)at));
      const uint2 hi =
          __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_t *)(at + 8 * CP * 16)));
      return make_uint4(lo.x, lo.y, hi.x, hi.y);
    };
    auto arrived = [&] {
      asm volatile("" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_waitcnt(kPgWaitAll);
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    };

    // In flight: where tile t + 1's keys lie, the pages of tile t + 2's.
    int pg0 = lookup(part.t0), pg1 = lookup(part.t0 + 1), pg2 = lookup(part.t0 + 2);
    int64_t off0, off1;
    uint64_t th0, th1;
    locate(part.t0, pg0, off0, th0);
    load(off0, th0, kbase, kb0, kc0, kc1);
    load(off0, th0, vbase, vb0, vc, vc);
    locate(part.t0 + 1, pg1, off1, th1);
    if (part.t0 + 1 < part.t1) load(off1, th1, kbase, kb1, kc0, kc1);
    arrived();
    f32x16_t sa[2] = {}, sb[2];
    if (active) {
      constexpr int NR = 2 * KS, kAhead = NR < 6 ? NR : 6;
      uint4 ka[NR];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) ka[i] = k_op(kb0, i);
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        if (i + kAhead < NR) ka[i + kAhead] = k_op(kb0, i + kAhead);
        sa[i / KS] = mfma_32x32x16<DT>(ka[i], qx[i % KS], sa[i / KS]);
        __builtin_amdgcn_sched_barrier(0);
      }
      hide(sa, part.t0, th0);
      float x = sa[0][0];
#pragma unroll
      for (int i = 1; i < 32; ++i) x = fmaxf(x, sa[i >> 4][i & 15]);
      raise(x);
    }
    int t = part.t0;
    // One tile: sc its scores, vr its values; sn, kr the next tile's; kw, vw
    // the buffers of the tiles behind those.
    auto step = [&](f32x16_t(&sc)[2], f32x16_t(&sn)[2], const char *kr, const char *vr, char *kw, char *vw) {
      arrived();
      // The pages' numbers first: behind new loads they would wait for those.
      int64_t off2;
      uint64_t th2;
      locate(t + 2, pg2, off2, th2);
      if (t + 1 < part.t1) load(off1, th1, vbase, vw, vc, vc);
      if (t + 2 < part.t1) load(off2, th2, kbase, kw, kc0, kc1);
      const int pg3 = lookup(t + 3);
      if (active) {
        // Scores of the next tile (of no tile behind the last: not used)
        // beside this one's probabilities, 2^(cc s - m), rounded to the dtype
        // as operands; their sums keep the fp32 values.  An output moves by at
        // most half a step of the dtype times sum p |v|.  A second operand for
        // what the rounding leaves, as the rows kernel has, is a third more
        // matrix instructions where those bound: 4096 tokens over 8192 keys 241
        // us, 197 without; 4096-token prompts of 32 heads over 8 223, 178;
        // chunks and tokens mixed 142, 111; a window over 256-wide heads 54, 48.
        constexpr int NR = 2 * KS, kAhead = NR < 3 ? NR : 3;
        const float m_neg = m_run == -INFINITY ? 0.f : -m_run;
        uint4 ka[NR];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) ka[i] = k_op(kr, i);
        // This phase has the vector instructions: its wave goes before the one
        // that shares the SIMD, whose matrix instructions fill in (4096 tokens
        // over 8192 keys 181 -> 173 us; the other phase first 175, both 177).
        __builtin_amdgcn_s_setprio(1);
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < NR; ++i) {
          if (i + kAhead < NR) ka[i + kAhead] = k_op(kr, i + kAhead);
          sn[i / KS] = mfma_32x32x16<DT>(ka[i], qx[i % KS], i % KS == 0 ? f32x16_t{} : sn[i / KS]);
#pragma unroll
          for (int e = 16 * i / NR; e < 16 * (i + 1) / NR; ++e) {
            const float e0 = __builtin_amdgcn_exp2f(fmaf(sc[e >> 3][2 * (e & 7)], cc, m_neg));
            const float e1 = __builtin_amdgcn_exp2f(fmaf(sc[e >> 3][2 * (e & 7) + 1], cc, m_neg));
            l_lane += e0;
            l_lane += e1;
            w[e] = pack2<DT>(e0, e1);
            stay(w[e]);
          }
          stay(l_lane);
          __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
        uint4 pb[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) pb[k] = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
        constexpr int NV = 4 * ND, vAhead = NV < 4 ? NV : 4;
        uint4 va[NV];
#pragma unroll
        for (int i = 0; i < vAhead; ++i) va[i] = v_op(vr, i / ND, i % ND);
        if (t + 1 < part.t1) hide(sn, t + 1, th1);
        float x = sn[0][0];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          if (i + vAhead < NV) va[i + vAhead] = v_op(vr, (i + vAhead) / ND, (i + vAhead) % ND);
          o[i % ND] = mfma_32x32x16<DT>(va[i], pb[i / ND], o[i % ND]);
#pragma unroll
          for (int e = 32 * i / NV; e < 32 * (i + 1) / NV; ++e) x = fmaxf(x, sn[e >> 4][e & 15]);
          stay(x);
          __builtin_amdgcn_sched_barrier(0);
        }
        if (t + 1 < part.t1) raise(x);
      }
      ++t;
      off1 = off2;
      th1 = th2;
      pg2 = pg3;
    };
    while (t < part.t1) {
      step(sa, sb, kb1, vb0, kb0, vb1);
      if (t >= part.t1) break;
      step(sb, sa, kb0, vb1, kb1, vb0);
    }

    // The wave's rows, through a tile's LDS: a store then takes whole rows
    // (from the accumulators it would take 32 bytes of each of 32 rows).
    __syncthreads();  // every wave has read the last tile
    int ln = lane;  // hidden from the compiler, which would otherwise keep the addresses formed from it
    stay(ln);       // below in registers through every tile
    const int er = ln & 31, eh = ln >> 5;
    int qt_e, qh_e;
    const bool own_e = u.row(32 * wave + er, qt_e, qh_e);
    char *rows = wave == 0 ? kb0 : wave == 1 ? kb1 : wave == 2 ? vb0 : vb1;
    constexpr int RC = D / 4;  // 16-byte chunks of an fp32 row; chunk c of row r at c ^ (r % 8)
    static_assert(32 * RC * 16 <= Geo::TILE, "a wave's rows fit a tile");
#pragma unroll
    for (int dt = 0; dt < ND; ++dt)
#pragma unroll
      for (int n = 0; n < 4; ++n)
        *reinterpret_cast<f32x4_t *>(rows + (er * RC + ((8 * dt + 2 * n + eh) ^ (er & 7))) * 16) =
            f32x4_t{o[dt][4 * n], o[dt][4 * n + 1], o[dt][4 * n + 2], o[dt][4 * n + 3]};
    const float l_row = half_wave_sum(l_lane);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    auto chunk_of = [&](int r, int c) { return *reinterpret_cast<const f32x4_t *>(rows + (r * RC + (c ^ (r & 7))) * 16); };
    if (part.partial >= 0) {
      const int64_t sr = (int64_t)part.partial * p.sh.rows + 32 * wave;
      if (own_e && eh == 0) {
        p.ws_m[sr + er] = m_run;
        p.ws_l[sr + er] = l_row;
      }
      float *po = p.ws_o + sr * D;
#pragma unroll
      for (int i0 = 0; i0 < 32 * RC; i0 += 64) {
        const int i = i0 + ln, r = i / RC;
        if (32 * wave + r < u.tokens * u.gw) *reinterpret_cast<f32x4_t *>(po + 4 * i) = chunk_of(r, i - r * RC);
      }
    } else {
      // A row that sees no key gets zeros.
      const float inv = l_row > 0.f ? 1.f / l_row : 0.f;
      const int64_t at = own_e ? ((int64_t)qt_e * p.hq + qh_e) * D : -1;
#pragma unroll
      for (int i0 = 0; i0 < 32 * RC / 2; i0 += 64) {
        const int i = i0 + ln, r = i / (RC / 2), c = 2 * (i - r * (RC / 2));
        const float f = __shfl(inv, r, 64);
        const int64_t to = __shfl(at, r, 64);
        const f32x4_t x = chunk_of(r, c) * f, y = chunk_of(r, c + 1) * f;
        if (to >= 0)
          *reinterpret_cast<uint4 *>(p.out + (to + 4 * c) * 2) =
              make_uint4(pack2<DT>(x[0], x[1]), pack2<DT>(x[2], x[3]), pack2<DT>(y[0], y[1]), pack2<DT>(y[2], y[3]));
      }
    }
    if (wk.w < wk.w_end) {
      __syncthreads();  // the next unit's first loads reuse the LDS
      wk.next(p);
    }
  }
}

// Merges the units that the shares cut: o = sum_i 2^(m_i - M) o_i / sum_i
// 2^(m_i - M) l_i over a unit's partial rows, M the largest of their maxima.
// A block takes the cuts of neighbouring shares; D / 4 threads a row, kCombineParts
// parts of it in flight together.  SPLIT (units cut into many parts): a row a
// block, its parts dealt to the block's groups of D / 4 threads, whose sums
// meet in LDS; else a row a group.  It reads the
// partial rows once: 13 to 16 us after the 4096 tokens over 8192 keys.
constexpr int kCombineParts = 4;
struct PartialSum {
  float m = -INFINITY, l = 0.f;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
};
// Parts first, first + step, ... < n of row r of the unit cut in front of block id.
__device__ __forceinline__ PartialSum paged_sum_parts(const PagedAttnParams &p, int D, int id, int r, int d0, int n,
                                                      int first, int step) {
  PartialSum s;
  for (int i0 = first; i0 < n; i0 += kCombineParts * step) {
    float ms[kCombineParts], ls[kCombineParts];
    f32x4_t os[kCombineParts];
#pragma unroll
    for (int k = 0; k < kCombineParts; ++k) {
      const bool in = i0 + k * step < n;
      const int i = in ? i0 + k * step : i0;
      const int64_t x = (int64_t)(i == 0 ? 2 * id - 1 : 2 * (id + i - 1)) * p.sh.rows + r;
      ms[k] = in ? p.ws_m[x] : -INFINITY;
      ls[k] = in ? p.ws_l[x] : 0.f;
      os[k] = *reinterpret_cast<const f32x4_t *>(p.ws_o + x * D + d0);
    }
    float m = s.m;
#pragma unroll
    for (int k = 0; k < kCombineParts; ++k) m = fmaxf(m, ms[k]);
    // A part without a weight (l = 0) adds nothing.  One whose scores are all
    // NaN has m = -inf too, but l is NaN, and with any weight stays it.
    const float a = s.l == 0.f ? 0.f : __builtin_amdgcn_exp2f(s.m - m);
    s.l *= a;
    s.o *= a;
#pragma unroll
    for (int k = 0; k < kCombineParts; ++k) {
      if (ls[k] == 0.f) continue;
      const float w = __builtin_amdgcn_exp2f(ms[k] - m);
      s.l = fmaf(w, ls[k], s.l);
      s.o += w * os[k];
    }
    s.m = m;
  }
  return s;
}

template <int DT, bool SPLIT>
__global__ void __launch_bounds__(kPgThreads) paged_combine_kernel(PagedAttnParams p, int D) {
  __shared__ float gm[kPgThreads], gl[kPgThreads];
  __shared__ f32x4_t go[kPgThreads];
  const int tid = threadIdx.x, lane = tid & 63, wide = D / 4, groups = kPgThreads / wide;
  const int group = tid / wide, d0 = 4 * (tid - group * wide), gw = p.sh.gw;
  const int per = (p.blocks + gridDim.x - 1) / gridDim.x, end = min((int)(blockIdx.x + 1) * per, p.blocks);
  for (int base = blockIdx.x * per; base < end; base += 64) {
    for (uint64_t cut = __ballot(base + lane < end && p.cuts[min(base + lane, end - 1)].last >= 0); cut;
         cut &= cut - 1) {
      const int id = base + __builtin_ctzll(cut);
      const PagedCut c = p.cuts[id];
      const int n = c.last - id + 2;  // the part of the block before, then parts id .. last
      const int rows = c.tokens * gw;
      for (int r0 = blockIdx.y * (SPLIT ? 1 : groups); r0 < rows; r0 += gridDim.y * (SPLIT ? 1 : groups)) {
        const int r = SPLIT ? r0 : r0 + group, tok = r / gw, g = r - tok * gw;
        const bool own = group < groups && r < rows && g < c.heads;
        if (SPLIT && r % gw >= c.heads) continue;
        PartialSum s;
        if (own) s = paged_sum_parts(p, D, id, r, d0, n, SPLIT ? group : 0, SPLIT ? groups : 1);
        if constexpr (SPLIT) {
          __syncthreads();
          gm[tid] = s.m;
          gl[tid] = s.l;
          go[tid] = s.o;
          __syncthreads();
          if (group != 0) continue;
          float M = s.m;
          for (int k = 1; k < groups; ++k) M = fmaxf(M, gm[tid + k * wide]);
          PartialSum all;
          for (int k = 0; k < groups; ++k) {
            const float m = gm[tid + k * wide], w = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - M);
            all.l = fmaf(w, gl[tid + k * wide], all.l);
            all.o += w * go[tid + k * wide];
          }
          s = all;
        }
        if (!own) continue;
        const float inv = s.l > 0.f ? 1.f / s.l : 0.f;
        store4<DT>(p.out, ((int64_t)(c.row0 + tok) * p.hq + c.head0 + g) * D + d0, s.o * inv);
      }
    }
  }
}

// ------------------------------------------------------------------- host
// Units of at most this many tiles (by the host's bound of the keys) are never
// divided: one launch, no partial rows.  Chunks: 512 tokens of 32 heads over 8
// 18 us whole, 27 divided; 1000 (16 tiles) 29, 35; 1500 of 12 over 2 (24
// tiles, few units) 39, 33; above head_dim 128, one block a compute unit, 1000
// tokens 44, 32.  Units of 16 rows: 8 sequences of 1000 keys (8 tiles) 18.4,
// 16.7; 301 keys 7, 11.
static int whole_tiles(bool chunk, int head_dim) { return !chunk ? 4 : head_dim <= 128 ? 16 : 8; }
// A unit's fixed cost in tiles.  Without it the shares of short units are the
// longest: 8192 tokens of 12 heads over 2 305 us, 242 with three tiles, 230
// with five, 236 with eight; 4096 of 28 over 4 224, 157, 148, 150.  Units of
// 16 rows: one, two or three tiles alike, 3% less than none.
constexpr int kChunkFixed = 5, kRowsFixed = 1;

struct PagedPlan {
  PagedShape sh;
  int64_t weight;  // a bound of the call's weights
  int blocks;
  bool chunk;  // the chunk kernel
  bool split;  // units are cut into many parts
  int cuts_x, cuts_y;  // the combine's grid
  size_t m_off, l_off, o_off, total;  // workspace: cuts, then these
};

constexpr int chunk_load_rows(int D) { return D <= 32 ? 16 : D <= 64 ? 8 : D <= 128 ? 4 : 2; }
constexpr int kChunkRows = 128;

static PagedPlan paged_plan(const kiv_paged_attention_args_t &a) {
  const kiv_paged_cache_t &c = a.cache;
  const kiv_paged_batch_t &b = a.batch;
  PagedPlan w;
  const int G = a.num_q_heads / c.num_kv_heads, cap = b.table_width * c.page_size;
  const int64_t most_keys = std::min<int64_t>(b.max_kv_len, cap);
  // More rows of a kv head than a unit of the rows kernel has: the chunk
  // kernel, if the rows of one of its load instructions lie in one page and
  // a tile's rows within 2 GiB.  (16 sequences of up to 4096 keys, 8 new
  // tokens of 32 heads over 8: 34 us by the chunk kernel, 48 by units of 16
  // rows; 5 tokens of 28 over 4: 30, 33; one token each: 27, 24; one token
  // over a million keys 362, 364.)
  w.chunk = c.dtype != KIV_DTYPE_F32 && (int64_t)std::min(b.max_q_len, b.total_q) * G > kRowsOfUnit &&
            c.page_size % chunk_load_rows(c.head_dim) == 0 && c.stride[2] >= 0 && c.stride[2] < (1 << 24);
  const int rows = w.chunk ? kChunkRows : kRowsOfUnit, shift = w.chunk ? kChunkTileShift : kRowsTileShift;
  const int window = std::min(a.window, 1 << 30);  // no table is as long
  w.sh = PagedShape::of(b.total_q, c.num_kv_heads, G, rows, cap, shift, window, false,
                        w.chunk ? kChunkFixed : kRowsFixed);
  // More than the call's units and tiles, by what the host knows of them.
  const int64_t units =
      ((int64_t)b.total_q / w.sh.tpu + std::min(b.num_seqs, b.total_q)) * w.sh.hpt * c.num_kv_heads;
  w.weight = units * ((cap >> shift) + 2 + w.sh.fixed);
  const int64_t keys = window > 0 ? std::min<int64_t>(most_keys, (int64_t)window + w.sh.tpu) : most_keys;
  const int64_t tiles = (keys >> shift) + 1;
  // Blocks that a compute unit holds at once: two, or one where a row's
  // operands take a whole wave's registers (32 sequences of up to 8192 keys of
  // 256-wide heads dealt to twice as many 44 us, 37 by this).
  const bool one = w.chunk ? c.head_dim > 128 : c.head_dim * elem_bytes(c.dtype) >= 512;
  const int slots = device_cu_count() * (one ? 1 : 2);
  w.split = false;
  w.cuts_x = w.cuts_y = 0;
  w.m_off = w.l_off = w.o_off = w.total = 0;
  if (tiles <= whole_tiles(w.chunk, c.head_dim)) {
    w.sh.whole = 1;
    w.blocks = (int)std::min<int64_t>(4 * slots, units);
    return w;
  }
  w.blocks = (int)std::max<int64_t>(8, std::min<int64_t>(slots, units * (tiles + 1)) & ~int64_t(7));
  w.split = w.blocks > 6 * units;
  w.cuts_x = (int)std::min<int64_t>(w.blocks, std::max<int64_t>(1, units));
  const int most_rows = (int)std::min<int64_t>(rows, (int64_t)w.sh.gw * std::max(1, std::min(w.sh.tpu, b.max_q_len)));
  const int groups = kPgThreads / (c.head_dim / 4);
  w.cuts_y = w.split ? most_rows : (most_rows + 2 * groups - 1) / (2 * groups);
  auto up = [](size_t x) { return (x + 255) & ~size_t(255); };
  const size_t parts = (size_t)2 * w.blocks * rows;
  w.m_off = up(w.blocks * sizeof(PagedCut));
  w.l_off = w.m_off + up(parts * 4);
  w.o_off = w.l_off + up(parts * 4);
  w.total = w.o_off + parts * c.head_dim * 4;
  return w;
}

static int paged_attention_check(const kiv_paged_attention_args_t *a, const char *who) {
  if (!a) return fail(KIV_ERR_INVALID, "%s: null argument", who);
  const kiv_paged_cache_t &c = a->cache;
  int rc = paged_cache_check(c, who);
  if (rc || (rc = paged_batch_check(a->batch, c, who))) return rc;
  const int D = c.head_dim, kt = D / 32;
  if (D % 32 || !(kt <= 4 || kt == 6 || kt == 8))
    return fail(KIV_ERR_UNSUPPORTED, "%s: head_dim %d unsupported (32, 64, 96, 128, 192, 256)", who, D);
  if (a->num_q_heads < 1 || a->num_q_heads % c.num_kv_heads)
    return fail(KIV_ERR_INVALID, "%s: bad head geometry", who);
  if (a->window < 0) return fail(KIV_ERR_INVALID, "%s: negative window", who);
  if ((int64_t)a->batch.table_width * c.page_size > (1 << 30))
    return fail(KIV_ERR_UNSUPPORTED, "%s: the block table spans over 2^30 keys", who);
  // Hidden scores are -inf behind the scale, and the maximum is taken there:
  // in base 2, so the scale must be finite there too.
  if (!(a->scaling > 0.f) || !(a->scaling * kPgLog2e < INFINITY))
    return fail(KIV_ERR_UNSUPPORTED, "%s: scaling must be positive and finite (at most 2.3e38)", who);
  return KIV_OK;
}

template <typename F> static int with_head_dim(int D, F &&f) {
  using std::integral_constant;
  switch (D) {
    case 32: return f(integral_constant<int, 32>{});
    case 64: return f(integral_constant<int, 64>{});
    case 96: return f(integral_constant<int, 96>{});
    case 128: return f(integral_constant<int, 128>{});
    case 192: return f(integral_constant<int, 192>{});
    default: return f(integral_constant<int, 256>{});
  }
}

}  // namespace kiv

using namespace kiv;

extern "C" {

size_t kiv_paged_attention_workspace_size(const kiv_paged_attention_args_t *a) {
  if (paged_attention_check(a, "kiv_paged_attention_workspace_size")) return 0;
  if (a->batch.total_q == 0 || a->batch.num_seqs == 0) return 0;
  return paged_plan(*a).total;
}

int kiv_paged_attention(const kiv_paged_attention_args_t *a, kiv_stream_t stream) {
  const char *who = "kiv_paged_attention";
  int rc = paged_attention_check(a, who);
  if (rc) return rc;
  const kiv_paged_cache_t &c = a->cache;
  const kiv_paged_batch_t &b = a->batch;
  if (b.total_q == 0 || b.num_seqs == 0) return KIV_OK;
  if (!a->q || !a->out) return fail(KIV_ERR_INVALID, "%s: null pointer", who);
  const int eb = elem_bytes(c.dtype), vec = vec_elems(c.dtype);
  if ((((uintptr_t)a->q | (uintptr_t)a->out) & 15) || a->q_stride[0] % vec || a->q_stride[1] % vec)
    return fail(KIV_ERR_INVALID, "%s: rows must be 16-byte aligned", who);
  const PagedPlan w = paged_plan(*a);
  if (w.weight > 2000000000)
    return fail(KIV_ERR_UNSUPPORTED, "%s: too much work for one call (%lld tiles)", who, (long long)w.weight);
  if (w.total > 0 && (!a->workspace || a->workspace_bytes < w.total || ((uintptr_t)a->workspace & 255)))
    return fail(KIV_ERR_INVALID, "%s: needs a 256-byte aligned workspace of %zu bytes "
                "(kiv_paged_attention_workspace_size)", who, w.total);
  // A unit's rows may be written before another block reads its own query rows.
  const int64_t q_end[2] = {(b.total_q - 1) * a->q_stride[0] * eb, (a->num_q_heads - 1) * a->q_stride[1] * eb};
  const int64_t row = (int64_t)c.head_dim * eb, q0 = (int64_t)(uintptr_t)a->q, o0 = (int64_t)(uintptr_t)a->out;
  const int64_t lo = q0 + std::min<int64_t>(q_end[0], 0) + std::min<int64_t>(q_end[1], 0);
  const int64_t hi = q0 + std::max<int64_t>(q_end[0], 0) + std::max<int64_t>(q_end[1], 0) + row;
  if (o0 < hi && lo < o0 + (int64_t)b.total_q * a->num_q_heads * row)
    return fail(KIV_ERR_INVALID, "%s: out must not overlap the query", who);
  const RowSet out = {a->out, {0, a->num_q_heads * row, row}, {1, b.total_q, a->num_q_heads}, row};
  if (rows_overlap(out, page_rows(c, c.k)) || rows_overlap(out, page_rows(c, c.v)))
    return fail(KIV_ERR_INVALID, "%s: out must not overlap the pages", who);
  PagedAttnParams p;
  p.q = (const char *)a->q;
  p.q_t = a->q_stride[0] * eb;
  p.q_h = a->q_stride[1] * eb;
  p.k = (const char *)c.k;
  p.v = (const char *)c.v;
  p.page_b = c.stride[0] * eb;
  p.head_b = c.stride[1] * eb;
  p.tok_b = c.stride[2] * eb;
  p.cu = b.cu_q;
  p.kv_len = b.kv_len;
  p.table = b.block_table;
  p.table_stride = b.table_stride;
  p.seqs = b.num_seqs;
  p.num_pages = c.num_pages;
  p.page_size = c.page_size;
  p.hq = a->num_q_heads;
  p.page_div = FastDiv::of(c.page_size);
  p.sh = w.sh;
  p.blocks = w.blocks;
  p.scale_log2 = a->scaling * kPgLog2e;
  p.out = (char *)a->out;
  char *ws = (char *)a->workspace;
  p.cuts = w.total > 0 ? (PagedCut *)ws : nullptr;
  p.ws_m = (float *)(ws + w.m_off);
  p.ws_l = (float *)(ws + w.l_off);
  p.ws_o = (float *)(ws + w.o_off);
  hipStream_t st = (hipStream_t)stream;
  const int D = c.head_dim;
  return with_head_dim(D, [&](auto dc) {
    constexpr int DV = decltype(dc)::value;
    const dim3 grid((unsigned)p.blocks), cgrid((unsigned)w.cuts_x, (unsigned)w.cuts_y);
    auto go = [&](auto dtc) {
      constexpr int DTV = decltype(dtc)::value;
      if constexpr (DTV != DT_F32) {
        if (w.chunk)
          hipLaunchKernelGGL((paged_chunk_kernel<DTV, DV / 32>), grid, dim3(kPgThreads), 0, st, p);
      }
      if (!w.chunk) hipLaunchKernelGGL((paged_rows_kernel<DTV, DV>), grid, dim3(kPgThreads), 0, st, p);
      if (w.total == 0) return;
      if (w.split) hipLaunchKernelGGL((paged_combine_kernel<DTV, true>), cgrid, dim3(kPgThreads), 0, st, p, D);
      else hipLaunchKernelGGL((paged_combine_kernel<DTV, false>), cgrid, dim3(kPgThreads), 0, st, p, D);
    };
    if (c.dtype == KIV_DTYPE_F32) go(std::integral_constant<int, DT_F32>{});
    else if (c.dtype == KIV_DTYPE_F16) go(std::integral_constant<int, DT_F16>{});
    else go(std::integral_constant<int, DT_BF16>{});
    KIV_HIP(hipGetLastError());
    return (int)KIV_OK;
  });
}

}  // extern "C"
