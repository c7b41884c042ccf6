// Norms of q and k for each head with the position rotation in the same pass,
// and the append of new K / V rows to a paged cache with both on the way.
//
// A head row x becomes x / sqrt(mean x^2 + eps) * w (in fp32), then each pair
// (a, b) of the first rot_dim entries turns by its angle t = position *
// inv_freq: (a cos t - b sin t, b cos t + a sin t), and is rounded once.
//
// Work: one wave takes rows of one token.  LPR lanes hold a row, each two
// 16-byte chunks that belong to the same pairs (chunk i and chunk i + half, or
// two neighbours where pairs are neighbours), so the rotation needs no
// exchange between lanes and the norm one reduction over LPR lanes.  The
// token's angles are formed once per wave, a pair a lane (64 pairs of a
// 128-wide head at a time), in turns in 64 bits (position 10^6 times a
// frequency of 1 is exact to 10^-10 turns; in fp32 it would be off by 0.06
// radians), and shared through LDS: 2 KiB a wave at head_dim 512.
//
// Bound: memory (each row read and written once): 4096 tokens of 32 rows of 128
// bf16 with norms 15.6 us a call, 4.3 TB/s, 86% of a copy's rate; 3856 tokens'
// K and V rows of 32 heads of 96 into pages 24.7 us, 3.8 TB/s; one token 3.7 us
// on the GPU.  A wave has all its rows' loads in flight before it forms the
// angles (in the paged form behind the lookup of its sequence and page); few
// tokens are dealt a row group a wave, many tokens kRopeBatch row groups a wave,
// whose angles are then formed once (two groups 16.3 us on the 4096 tokens,
// eight 18.7, one 15.9; on the pages 25.8, 31.5, 28.2).
#include <climits>
#include <type_traits>

#include "kiv_common.h"
#include "kiv_internal.h"

namespace kiv {

constexpr int kRopeThreads = 256;
constexpr int kRopeBatch = 4;       // row groups of a wave where there are many tokens
constexpr int kRopeMaxDim = 512;
constexpr int kRopeMaxHeads = 1 << 30;  // of all kinds: rows are counted in 32 bits
constexpr int kRopeFewWaves = 4096;  // waves up to which a wave takes one row group

// Rows of one kind (q, k or v): byte strides.
struct RopeRows {
  const char *src;
  int64_t sb, sh, st;
  char *dst;
  int64_t db, dh, dt;  // paged: db is the page stride
  const float *w;
  float eps;
  int norm, heads;
};

struct RopeParams {
  RopeRows q, k, v;
  int tokens, rows;  // tokens of a batch row; heads of all kinds
  int64_t waves;     // batch * tokens * parts
  int parts, iters;  // waves of a token; row groups of a wave
  int cpr, half;     // chunks of a row; chunks of a rotated half
  float inv_dim;
  const float *inv_freq;
  const int32_t *axes;
  const char *pos;
  int64_t pos_axis, pos_b, pos_t;
  int pos64, num_axes, interleaved;
  float scale;
  // paged
  const int32_t *cu, *kv_len, *table;
  int64_t table_stride;
  int seqs, width, num_pages, page_size;
};

template <int DT, int LPR, int U, bool PAGED>
__global__ void __launch_bounds__(kRopeThreads) norm_rope_kernel(RopeParams p) {
  constexpr int VEC = Elem<DT>::VEC, RPG = 64 / LPR;  // RPG: rows of a group
  __shared__ __align__(16) float angles[kRopeThreads / 64][2][kRopeMaxDim / 2];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int64_t wv = (int64_t)blockIdx.x * (kRopeThreads / 64) + wave;
  if (wv >= p.waves) return;
  const int64_t bt = wv / p.parts;
  const int part = (int)(wv - bt * p.parts);
  int b = PAGED ? 0 : (int)(bt / p.tokens);
  const int t = (int)(bt - (int64_t)b * p.tokens);
  int64_t key = 0, slot_off = -1;  // paged: the token's key index; its row's offset in the pool (-1: none)
  if constexpr (PAGED) {
    // The token's sequence: as many sequences end at or before it.
    int seq = 0;
    for (int base = 0; base < p.seqs; base += 64) {
      const int end = p.cu[min(base + lane, p.seqs - 1) + 1];
      const uint64_t done = __ballot(base + lane < p.seqs && end <= t);
      seq += __popcll(done);
      if (done != ~uint64_t(0)) break;
    }
    if (seq >= p.seqs || t < p.cu[0]) return;
    key = (int64_t)p.kv_len[seq] - p.cu[seq + 1] + t;
    if (key >= 0 && key < (int64_t)p.width * p.page_size) {
      const int at = (int)((uint32_t)key / (uint32_t)p.page_size), slot = (int)key - at * p.page_size;
      const int page = p.table[seq * p.table_stride + at];
      if (page >= 0 && page < p.num_pages) slot_off = (int64_t)page * p.k.db + (int64_t)slot * p.k.dt;
    }
  }

  // The lane's chunks of a row.
  const int item = lane % LPR, sub = lane / LPR;
  const bool turns = item < p.half;
  const int c0 = !turns || p.interleaved ? 2 * item : item, c1 = turns && !p.interleaved ? item + p.half : c0 + 1;
  const bool in0 = c0 < p.cpr, in1 = c1 < p.cpr;
  const int e0 = in0 ? c0 : 0, e1 = in1 ? c1 : 0;

  // All rows' loads, then the angles.
  uint4 x0[U], x1[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int r = (part * p.iters + u) * RPG + sub;
    if (u < p.iters && r < p.rows) {
      const RopeRows &s = r < p.q.heads ? p.q : r < p.q.heads + p.k.heads ? p.k : p.v;
      const int h = r < p.q.heads ? r : r < p.q.heads + p.k.heads ? r - p.q.heads : r - p.q.heads - p.k.heads;
      const char *src = s.src + (int64_t)b * s.sb + (int64_t)h * s.sh + (int64_t)t * s.st;
      x0[u] = load16(src + 16 * e0);
      x1[u] = load16(src + 16 * e1);
    } else {
      x0[u] = x1[u] = make_uint4(0, 0, 0, 0);
    }
  }

  // The token's angles, a pair a lane.
  float *cs = angles[wave][0], *sn = angles[wave][1];
  const int pairs = p.half * VEC;
  for (int i = lane; i < pairs; i += 64) {
    int64_t pos = key;
    if (p.pos) {
      const int axis = p.axes ? min(max(p.axes[i], 0), p.num_axes - 1) : 0;
      const int64_t at = axis * p.pos_axis + b * p.pos_b + t * p.pos_t;
      pos = p.pos64 ? reinterpret_cast<const int64_t *>(p.pos)[at] : reinterpret_cast<const int32_t *>(p.pos)[at];
    }
    double turn = (double)pos * (double)p.inv_freq[i] * 0.15915494309189533577;
    turn -= rint(turn);
    float s, c;
    sincospif((float)(2.0 * turn), &s, &c);
    cs[i] = c * p.scale;
    sn[i] = s * p.scale;
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  float co[VEC], si[VEC];
#pragma unroll
  for (int j = 0; j < VEC; j += 4) {
    const int at = turns ? item * VEC + j : 0;
    const float4 c = *reinterpret_cast<const float4 *>(cs + at), s = *reinterpret_cast<const float4 *>(sn + at);
    co[j] = c.x, co[j + 1] = c.y, co[j + 2] = c.z, co[j + 3] = c.w;
    si[j] = s.x, si[j + 1] = s.y, si[j + 2] = s.z, si[j + 3] = s.w;
  }

#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int r = (part * p.iters + u) * RPG + sub;
    if (u >= p.iters || (part * p.iters + u) * RPG >= p.rows) break;
    const bool is_q = r < p.q.heads, is_v = r >= p.q.heads + p.k.heads;
    const RopeRows &s = is_q ? p.q : !is_v ? p.k : p.v;
    const int h = is_q ? r : !is_v ? r - p.q.heads : r - p.q.heads - p.k.heads;
    float a[VEC], z[VEC];
    unpack_chunk<DT>(x0[u], a);
    unpack_chunk<DT>(x1[u], z);
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {  // lanes past the row hold its first chunk: an infinity there times 0 is NaN
      const float x = in0 ? a[j] : 0.f, y = in1 ? z[j] : 0.f;
      ss = fmaf(x, x, fmaf(y, y, ss));
    }
    ss = group_sum<LPR>(ss);  // every lane of the wave is here
    if (s.norm) {
      const float inv = rsqrtf(fmaf(ss, p.inv_dim, s.eps));
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        a[j] *= inv;
        z[j] *= inv;
      }
      if (s.w) {
#pragma unroll
        for (int j = 0; j < VEC; j += 4) {
          const float4 w0 = *reinterpret_cast<const float4 *>(s.w + e0 * VEC + j);
          const float4 w1 = *reinterpret_cast<const float4 *>(s.w + e1 * VEC + j);
          a[j] *= w0.x, a[j + 1] *= w0.y, a[j + 2] *= w0.z, a[j + 3] *= w0.w;
          z[j] *= w1.x, z[j + 1] *= w1.y, z[j + 2] *= w1.z, z[j + 3] *= w1.w;
        }
      }
    }
    if (turns && !is_v) {
      if (p.interleaved) {
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) {
          const float a0 = a[2 * j], a1 = a[2 * j + 1], z0 = z[2 * j], z1 = z[2 * j + 1];
          a[2 * j] = a0 * co[j] - a1 * si[j];
          a[2 * j + 1] = a1 * co[j] + a0 * si[j];
          z[2 * j] = z0 * co[VEC / 2 + j] - z1 * si[VEC / 2 + j];
          z[2 * j + 1] = z1 * co[VEC / 2 + j] + z0 * si[VEC / 2 + j];
        }
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float u0 = a[j], u1 = z[j];
          a[j] = u0 * co[j] - u1 * si[j];
          z[j] = u1 * co[j] + u0 * si[j];
        }
      }
    }
    // Rows that neither a norm nor a rotation touches keep their bits.
    const bool keep = !s.norm && (is_v || !turns);
    uint4 y0 = x0[u], y1 = x1[u];
    if (!keep) {
      if constexpr (DT == DT_F32) {
        y0 = make_uint4(__float_as_uint(a[0]), __float_as_uint(a[1]), __float_as_uint(a[2]), __float_as_uint(a[3]));
        y1 = make_uint4(__float_as_uint(z[0]), __float_as_uint(z[1]), __float_as_uint(z[2]), __float_as_uint(z[3]));
      } else {
        y0 = make_uint4(pack2<DT>(a[0], a[1]), pack2<DT>(a[2], a[3]), pack2<DT>(a[4], a[5]), pack2<DT>(a[6], a[7]));
        y1 = make_uint4(pack2<DT>(z[0], z[1]), pack2<DT>(z[2], z[3]), pack2<DT>(z[4], z[5]), pack2<DT>(z[6], z[7]));
      }
    }
    if (r >= p.rows || (PAGED && !is_q && slot_off < 0)) continue;
    char *dst = s.dst + (int64_t)h * s.dh + (PAGED && !is_q ? slot_off : (int64_t)b * s.db + (int64_t)t * s.dt);
    if (in0) *reinterpret_cast<uint4 *>(dst + 16 * c0) = y0;
    if (in1) *reinterpret_cast<uint4 *>(dst + 16 * c1) = y1;
  }
}

// none: there is no token to turn (an empty tensor's positions have no address).
static int rotary_check(const kiv_rotary_t &r, int head_dim, int dtype, bool positions_optional, bool none,
                        const char *who) {
  if (r.rot_dim == 0) return KIV_OK;
  const int step = 2 * vec_elems(dtype);
  if (r.rot_dim < 0 || r.rot_dim > head_dim || r.rot_dim % step)
    return fail(KIV_ERR_UNSUPPORTED, "%s: rotated width %d is no multiple of %d up to head_dim %d", who, r.rot_dim,
                step, head_dim);
  if (!r.inv_freq) return fail(KIV_ERR_INVALID, "%s: null inv_freq", who);
  if (none) return KIV_OK;
  if (!r.positions && !positions_optional) return fail(KIV_ERR_INVALID, "%s: null positions", who);
  if (!r.positions && r.axes) return fail(KIV_ERR_INVALID, "%s: several axes need positions", who);
  if (r.positions && r.position_bytes != 4 && r.position_bytes != 8)
    return fail(KIV_ERR_INVALID, "%s: positions are int32 or int64", who);
  if (r.positions && r.num_axes < 1) return fail(KIV_ERR_INVALID, "%s: no position axis", who);
  return KIV_OK;
}

static int norm_check(const kiv_head_norm_t &n, const char *who) {
  if (!n.enabled) return KIV_OK;
  if (!(n.eps >= 0.f)) return fail(KIV_ERR_INVALID, "%s: norm epsilon must not be negative", who);
  if ((uintptr_t)n.weight & 15) return fail(KIV_ERR_INVALID, "%s: norm weights must be 16-byte aligned", who);
  return KIV_OK;
}

static int rows_check(const char *who, int dtype, int head_dim) {
  if (dtype < KIV_DTYPE_F32 || dtype > KIV_DTYPE_BF16) return fail(KIV_ERR_INVALID, "%s: unknown dtype %d", who, dtype);
  if (head_dim < 1 || head_dim > kRopeMaxDim || head_dim % vec_elems(dtype))
    return fail(KIV_ERR_UNSUPPORTED, "%s: head_dim %d unsupported (a multiple of %d up to %d)", who, head_dim,
                vec_elems(dtype), kRopeMaxDim);
  return KIV_OK;
}

static int aligned_check(const char *who, const void *p, const int64_t *stride, int n, int dtype) {
  if (!p) return fail(KIV_ERR_INVALID, "%s: null pointer", who);
  bool ok = !((uintptr_t)p & 15);
  for (int i = 0; i < n; ++i) ok = ok && stride[i] % vec_elems(dtype) == 0;
  if (!ok) return fail(KIV_ERR_INVALID, "%s: rows must be 16-byte aligned", who);
  return KIV_OK;
}

// Rows that are written: apart from each other, and from rows that other
// waves read or write, or the bytes depend on which wave comes first.
static int written_check(const char *who, const char *name, const RowSet &rows) {
  if (rows_fold(rows)) return fail(KIV_ERR_INVALID, "%s: rows of %s share memory", who, name);
  return KIV_OK;
}
static int apart_check(const char *who, const char *name, const RowSet &a, const char *other, const RowSet &b) {
  if (rows_overlap(a, b)) return fail(KIV_ERR_INVALID, "%s: %s must not overlap %s", who, name, other);
  return KIV_OK;
}
// An output may be its input: a wave has read a row before it writes it.
static int in_place_check(const char *who, const char *name, const RowSet &out, const char *input, const RowSet &in) {
  if (!rows_same(out, in) && rows_overlap(out, in))
    return fail(KIV_ERR_INVALID, "%s: %s must be %s or not overlap it", who, name, input);
  return KIV_OK;
}

static void fill_rotary(RopeParams &p, const kiv_rotary_t &r, int dtype) {
  p.half = r.rot_dim / (2 * vec_elems(dtype));
  p.inv_freq = r.inv_freq;
  p.axes = r.axes;
  p.pos = (const char *)r.positions;
  p.pos_axis = r.position_stride[0];
  p.pos_b = r.position_stride[1];
  p.pos_t = r.position_stride[2];
  p.pos64 = r.position_bytes == 8;
  p.num_axes = r.num_axes;
  p.interleaved = r.interleaved != 0;
  p.scale = r.scale;
}

static RopeRows rope_rows(const void *src, int64_t sb, int64_t sh, int64_t st, void *dst, int64_t db, int64_t dh,
                          int64_t dt, const kiv_head_norm_t &n, int heads, int eb) {
  RopeRows r;
  r.src = (const char *)src;
  r.sb = sb * eb;
  r.sh = sh * eb;
  r.st = st * eb;
  r.dst = (char *)dst;
  r.db = db * eb;
  r.dh = dh * eb;
  r.dt = dt * eb;
  r.w = n.weight;
  r.eps = n.eps;
  r.norm = n.enabled != 0;
  r.heads = heads;
  return r;
}

template <bool PAGED>
static int rope_launch(RopeParams &p, int batch, int head_dim, int dtype, hipStream_t st, const char *who) {
  p.cpr = head_dim / vec_elems(dtype);
  p.inv_dim = 1.f / (float)head_dim;
  p.rows = p.q.heads + p.k.heads + p.v.heads;
  const int64_t tokens = (int64_t)batch * p.tokens;
  if (tokens == 0 || p.rows == 0) return KIV_OK;
  int lpr = 2;
  while (lpr < (p.cpr + 1) / 2) lpr *= 2;
  const int groups = (p.rows + 64 / lpr - 1) / (64 / lpr);
  // A row group a wave while that leaves few waves: one token's 36 rows of 128
  // are then five waves' work side by side.
  const bool few = tokens * groups <= kRopeFewWaves;
  const int batch_of = few ? 1 : kRopeBatch;
  p.parts = (groups + batch_of - 1) / batch_of;
  p.iters = (groups + p.parts - 1) / p.parts;
  p.waves = tokens * p.parts;
  const int64_t blocks = (p.waves + kRopeThreads / 64 - 1) / (kRopeThreads / 64);
  if (blocks > INT32_MAX) return fail(KIV_ERR_UNSUPPORTED, "%s: too many tokens", who);
  auto go = [&](auto dtc, auto lc) {
    constexpr int DTV = decltype(dtc)::value, LV = decltype(lc)::value;
    if (few)
      hipLaunchKernelGGL((norm_rope_kernel<DTV, LV, 1, PAGED>), dim3((unsigned)blocks), dim3(kRopeThreads), 0, st, p);
    else
      hipLaunchKernelGGL((norm_rope_kernel<DTV, LV, kRopeBatch, PAGED>), dim3((unsigned)blocks), dim3(kRopeThreads), 0,
                         st, p);
  };
  auto by_lanes = [&](auto dtc) {
    using std::integral_constant;
    switch (lpr) {
      case 2: return go(dtc, integral_constant<int, 2>{});
      case 4: return go(dtc, integral_constant<int, 4>{});
      case 8: return go(dtc, integral_constant<int, 8>{});
      case 16: return go(dtc, integral_constant<int, 16>{});
      case 32: return go(dtc, integral_constant<int, 32>{});
      default: return go(dtc, integral_constant<int, 64>{});
    }
  };
  if (dtype == KIV_DTYPE_F32) by_lanes(std::integral_constant<int, DT_F32>{});
  else if (dtype == KIV_DTYPE_F16) by_lanes(std::integral_constant<int, DT_F16>{});
  else by_lanes(std::integral_constant<int, DT_BF16>{});
  KIV_HIP(hipGetLastError());
  return KIV_OK;
}

int paged_cache_check(const kiv_paged_cache_t &c, const char *who) {
  if (c.dtype < KIV_DTYPE_F32 || c.dtype > KIV_DTYPE_BF16)
    return fail(KIV_ERR_INVALID, "%s: unknown dtype %d", who, c.dtype);
  if (c.num_pages < 1 || c.page_size < 1 || c.num_kv_heads < 1 || c.head_dim < 1)
    return fail(KIV_ERR_INVALID, "%s: bad cache geometry", who);
  if ((int64_t)c.num_pages * c.page_size > INT32_MAX)
    return fail(KIV_ERR_UNSUPPORTED, "%s: the pool holds 2^31 tokens or more", who);
  int rc = aligned_check(who, c.k, c.stride, 3, c.dtype);
  return rc ? rc : aligned_check(who, c.v, c.stride, 3, c.dtype);
}

RowSet page_rows(const kiv_paged_cache_t &c, const void *pages) {
  const int64_t eb = elem_bytes(c.dtype);
  return {pages, {c.stride[0] * eb, c.stride[2] * eb, c.stride[1] * eb}, {c.num_pages, c.page_size, c.num_kv_heads},
          c.head_dim * eb};
}

int paged_batch_check(const kiv_paged_batch_t &b, const kiv_paged_cache_t &c, const char *who) {
  if (b.num_seqs < 0 || b.table_width < 0 || b.total_q < 0)
    return fail(KIV_ERR_INVALID, "%s: negative batch sizes", who);
  if ((int64_t)b.table_width * c.page_size > INT32_MAX)
    return fail(KIV_ERR_UNSUPPORTED, "%s: the block table spans 2^31 keys or more", who);
  if (b.num_seqs > 0 && (!b.cu_q || !b.kv_len || (b.table_width > 0 && !b.block_table)))
    return fail(KIV_ERR_INVALID, "%s: null batch array", who);
  return KIV_OK;
}

}  // namespace kiv

using namespace kiv;

extern "C" {

int kiv_norm_rope(const kiv_norm_rope_args_t *a, kiv_stream_t stream) {
  const char *who = "kiv_norm_rope";
  if (!a) return fail(KIV_ERR_INVALID, "%s: null argument", who);
  int rc = rows_check(who, a->dtype, a->head_dim);
  if (rc) return rc;
  if (a->batch < 0 || a->tokens < 0 || a->num_q_heads < 1 || a->num_kv_heads < 0)
    return fail(KIV_ERR_INVALID, "%s: bad sizes", who);
  if ((int64_t)a->num_q_heads + a->num_kv_heads > kRopeMaxHeads)
    return fail(KIV_ERR_UNSUPPORTED, "%s: over 2^30 heads", who);
  const bool none = a->batch == 0 || a->tokens == 0;
  if ((rc = rotary_check(a->rotary, a->head_dim, a->dtype, false, none, who)) || (rc = norm_check(a->q_norm, who)) ||
      (rc = norm_check(a->k_norm, who)))
    return rc;
  if (none) return KIV_OK;
  if ((rc = aligned_check(who, a->q, a->q_stride, 3, a->dtype)) ||
      (rc = aligned_check(who, a->q_out, a->q_out_stride, 3, a->dtype)))
    return rc;
  if (a->num_kv_heads > 0 && ((rc = aligned_check(who, a->k, a->k_stride, 3, a->dtype)) ||
                              (rc = aligned_check(who, a->k_out, a->k_out_stride, 3, a->dtype))))
    return rc;
  const int eb = elem_bytes(a->dtype);
  auto rows = [&](const void *at, const int64_t *stride, int heads) {
    return RowSet{at, {stride[0] * eb, stride[1] * eb, stride[2] * eb}, {a->batch, heads, a->tokens},
                  (int64_t)a->head_dim * eb};
  };
  const RowSet q = rows(a->q, a->q_stride, a->num_q_heads), k = rows(a->k, a->k_stride, a->num_kv_heads);
  const RowSet q_out = rows(a->q_out, a->q_out_stride, a->num_q_heads);
  const RowSet k_out = rows(a->k_out, a->k_out_stride, a->num_kv_heads);
  if ((rc = written_check(who, "q_out", q_out)) || (rc = written_check(who, "k_out", k_out)) ||
      (rc = in_place_check(who, "q_out", q_out, "q", q)) || (rc = in_place_check(who, "k_out", k_out, "k", k)) ||
      (rc = apart_check(who, "q_out", q_out, "k", k)) || (rc = apart_check(who, "k_out", k_out, "q", q)) ||
      (rc = apart_check(who, "q_out", q_out, "k_out", k_out)))
    return rc;
  RopeParams p = {};
  p.q = rope_rows(a->q, a->q_stride[0], a->q_stride[1], a->q_stride[2], a->q_out, a->q_out_stride[0],
                  a->q_out_stride[1], a->q_out_stride[2], a->q_norm, a->num_q_heads, eb);
  p.k = rope_rows(a->k, a->k_stride[0], a->k_stride[1], a->k_stride[2], a->k_out, a->k_out_stride[0],
                  a->k_out_stride[1], a->k_out_stride[2], a->k_norm, a->num_kv_heads, eb);
  p.tokens = a->tokens;
  fill_rotary(p, a->rotary, a->dtype);
  return rope_launch<false>(p, a->batch, a->head_dim, a->dtype, (hipStream_t)stream, who);
}

int kiv_paged_append(const kiv_paged_append_args_t *a, kiv_stream_t stream) {
  const char *who = "kiv_paged_append";
  if (!a) return fail(KIV_ERR_INVALID, "%s: null argument", who);
  const kiv_paged_cache_t &c = a->cache;
  const kiv_paged_batch_t &b = a->batch;
  int rc = paged_cache_check(c, who);
  if (rc || (rc = rows_check(who, c.dtype, c.head_dim)) || (rc = paged_batch_check(b, c, who)) ||
      (rc = rotary_check(a->rotary, c.head_dim, c.dtype, true, b.total_q == 0 || b.num_seqs == 0, who)) || (rc = norm_check(a->q_norm, who)) ||
      (rc = norm_check(a->k_norm, who)) || (rc = norm_check(a->v_norm, who)))
    return rc;
  if (a->num_q_heads < 0) return fail(KIV_ERR_INVALID, "%s: bad sizes", who);
  if ((int64_t)a->num_q_heads + 2 * (int64_t)c.num_kv_heads > kRopeMaxHeads)
    return fail(KIV_ERR_UNSUPPORTED, "%s: over 2^30 heads", who);
  if (b.total_q == 0 || b.num_seqs == 0) return KIV_OK;
  if ((rc = aligned_check(who, a->k, a->k_stride, 2, c.dtype)) ||
      (rc = aligned_check(who, a->v, a->v_stride, 2, c.dtype)))
    return rc;
  if (a->num_q_heads > 0 && ((rc = aligned_check(who, a->q, a->q_stride, 2, c.dtype)) ||
                             (rc = aligned_check(who, a->q_out, a->q_out_stride, 2, c.dtype))))
    return rc;
  const int eb = elem_bytes(c.dtype);
  auto rows = [&](const void *at, const int64_t *stride, int heads) {  // axes as page_rows has them
    return RowSet{at, {0, stride[0] * eb, stride[1] * eb}, {1, b.total_q, heads}, (int64_t)c.head_dim * eb};
  };
  const RowSet k_pages = page_rows(c, c.k), v_pages = page_rows(c, c.v);
  const RowSet k = rows(a->k, a->k_stride, c.num_kv_heads), v = rows(a->v, a->v_stride, c.num_kv_heads);
  const RowSet q = rows(a->q, a->q_stride, a->num_q_heads), q_out = rows(a->q_out, a->q_out_stride, a->num_q_heads);
  if ((rc = written_check(who, "the pages", k_pages)) || (rc = apart_check(who, "K pages", k_pages, "V pages", v_pages)))
    return rc;
  for (const RowSet &pages : {k_pages, v_pages})
    if ((rc = apart_check(who, "the pages", pages, "k", k)) || (rc = apart_check(who, "the pages", pages, "v", v)) ||
        (rc = apart_check(who, "the pages", pages, "q", q)) || (rc = apart_check(who, "the pages", pages, "q_out", q_out)))
      return rc;
  if ((rc = written_check(who, "q_out", q_out)) || (rc = in_place_check(who, "q_out", q_out, "q", q)) ||
      (rc = apart_check(who, "q_out", q_out, "k", k)) || (rc = apart_check(who, "q_out", q_out, "v", v)))
    return rc;
  RopeParams p = {};
  p.q = rope_rows(a->q, 0, a->q_stride[1], a->q_stride[0], a->q_out, 0, a->q_out_stride[1], a->q_out_stride[0],
                  a->q_norm, a->num_q_heads, eb);
  p.k = rope_rows(a->k, 0, a->k_stride[1], a->k_stride[0], c.k, c.stride[0], c.stride[1], c.stride[2], a->k_norm,
                  c.num_kv_heads, eb);
  p.v = rope_rows(a->v, 0, a->v_stride[1], a->v_stride[0], c.v, c.stride[0], c.stride[1], c.stride[2], a->v_norm,
                  c.num_kv_heads, eb);
  p.tokens = b.total_q;
  fill_rotary(p, a->rotary, c.dtype);
  p.pos_b = 0;
  p.cu = b.cu_q;
  p.kv_len = b.kv_len;
  p.table = b.block_table;
  p.table_stride = b.table_stride;
  p.seqs = b.num_seqs;
  p.width = b.table_width;
  p.num_pages = c.num_pages;
  p.page_size = c.page_size;
  return rope_launch<true>(p, 1, c.head_dim, c.dtype, (hipStream_t)stream, who);
}

}  // extern "C"
