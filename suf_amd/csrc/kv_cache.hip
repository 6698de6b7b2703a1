// Rotary positions on both parties' shares and the append of keys and values
// to a paged cache (sufhip_rotary2, sufhip_kv_append2).
//
// A rotation by public fixed-point factors is linear, so each party turns its
// own shares: per pair u' = u c - v s, v' = u s + v c mod 2^64.  The append
// opens value - mask once, E = x_0 + x_1 - b_0 - b_1, and stores E, b_0, b_1 in
// the token's page.
//
// HBM bounds both: a rotation reads and writes 16 bytes a value and party, an
// append reads 32 and writes 24 bytes a value.  One lane takes one unit of a
// row, two pieces of kP words that the rotation mixes (half layout: kP words
// of each half; neighbours: 2 kP words in a row), for both parties, so nothing
// is exchanged between lanes and an output may replace its input.  kP = 2
// where every piece is 16-byte aligned: 2048 tokens of 32 heads of 128 rotate
// in 52 us against 53 by single words (43 against 46 out of the last cache);
// 2579 tokens append keys and values of 8 heads of 128 in 68 us either way, 57
// against 59 out of the last cache.
//
// Measured: rotation of 2048 x 32 x 128 values 51 us (5.2 TB/s; a copy of
// 2 GiB reaches 4.85), 1021 x 16 x 80 with 32 of them rotated 10.1; one token
// of 12 heads 2.2 (the launch).  Append of 2579 tokens, 8 heads of 128, rotated
// keys and values, 67 us (4.5 TB/s); of eight single tokens, 12 heads, 4.6: a
// row's sequence, its length and its page are loads that wait for one another,
// so the row's own words are asked for first.
#include <hip/hip_runtime.h>

#include <utility>

#include "kv_device.hpp"
#include "suf_hip.h"
#include "sufhip_internal.hpp"
#include "trunc_device.hpp"

namespace sufhip {
namespace {

constexpr int kBlock = 256;
constexpr uint32_t kMaxUnits = 1u << 30;  // units of one launch (32-bit indices)

struct Rot {
  const int32_t* table;
  int positions, half, interleaved, on;
  uint64_t pass_mul;
};

struct Rows {
  const uint64_t* p[2];
  int64_t ts, hs;
};

// The unit q of a row: the first words of its two pieces, the pair it starts
// at (-1: not rotated), and whether the second piece is inside the row.
struct Unit {
  int o0, o1, pair;
  bool two;
};
template <int kP>
__device__ __forceinline__ Unit unit_of(const Rot& r, int dim, int q) {
  const int turned = r.half / kP;
  if (q < turned) {
    const int i = q * kP;
    return r.interleaved ? Unit{2 * i, 2 * i + kP, i, true} : Unit{i, r.half + i, i, true};
  }
  const int o = 2 * r.half + 2 * kP * (q - turned);
  return {o, o + kP, -1, o + kP < dim};
}
inline int units_of(int kP, int half, int dim) {
  return half / kP + (dim - 2 * half + 2 * kP - 1) / (2 * kP);
}

template <int kP>
__device__ __forceinline__ void load_piece(const uint64_t* p, uint64_t* v) {
  if constexpr (kP == 2) {
    const ulonglong2 w = *reinterpret_cast<const ulonglong2*>(p);
    v[0] = w.x;
    v[1] = w.y;
  } else {
    v[0] = *p;
  }
}
template <int kP>
__device__ __forceinline__ void store_piece(uint64_t* p, const uint64_t* v) {
  if constexpr (kP == 2)
    *reinterpret_cast<ulonglong2*>(p) = make_ulonglong2(v[0], v[1]);
  else
    *p = v[0];
}

template <int kP>
__device__ __forceinline__ void load_unit(const uint64_t* row, const Unit& u,
                                          uint64_t (&v)[2 * kP]) {
  load_piece<kP>(row + u.o0, v);
  if (u.two)
    load_piece<kP>(row + u.o1, v + kP);
  else
    for (int k = 0; k < kP; ++k) v[kP + k] = 0;
}
template <int kP>
__device__ __forceinline__ void store_unit(uint64_t* row, const Unit& u,
                                           const uint64_t (&v)[2 * kP]) {
  store_piece<kP>(row + u.o0, v);
  if (u.two) store_piece<kP>(row + u.o1, v + kP);
}

// The factors of a unit's pairs at a position (inside the table).
template <int kP>
__device__ __forceinline__ void load_factors(const Rot& r, const Unit& u, int pos, int64_t (&c)[kP],
                                             int64_t (&s)[kP]) {
  if (u.pair < 0) return;
  const int32_t* t = r.table + 2 * (int64_t(pos) * r.half + u.pair);
  if constexpr (kP == 2) {
    const int4 w = *reinterpret_cast<const int4*>(t);
    c[0] = w.x;
    s[0] = w.y;
    c[1] = w.z;
    s[1] = w.w;
  } else {
    const int2 w = *reinterpret_cast<const int2*>(t);
    c[0] = w.x;
    s[0] = w.y;
  }
}

template <int kP>
__device__ __forceinline__ void turn(const Rot& r, const Unit& u, const int64_t (&c)[kP],
                                     const int64_t (&s)[kP], uint64_t (&v)[2 * kP]) {
  if (u.pair < 0) {
#pragma unroll
    for (int k = 0; k < 2 * kP; ++k) v[k] *= r.pass_mul;
    return;
  }
#pragma unroll
  for (int k = 0; k < kP; ++k) {
    // Neighbours: pair k is words 2 k, 2 k + 1 of the unit; halves: word k of
    // each piece.
    const int a = k, b = kP + k;
    const uint64_t x = r.interleaved ? v[2 * k] : v[a], y = r.interleaved ? v[2 * k + 1] : v[b];
    const uint64_t nx = x * uint64_t(c[k]) - y * uint64_t(s[k]);
    const uint64_t ny = x * uint64_t(s[k]) + y * uint64_t(c[k]);
    if (r.interleaved) {
      v[2 * k] = nx;
      v[2 * k + 1] = ny;
    } else {
      v[a] = nx;
      v[b] = ny;
    }
  }
}

// Truncates both parties' values of a unit by the gate of `epi` (on).
template <int kP>
__device__ __forceinline__ void trunc_unit(const TruncEpi& epi, const EpiHdrs& eh, uint64_t mask,
                                           uint64_t (&v)[2][2 * kP]) {
  uint64_t open[2 * kP], w[2][2 * kP];
#pragma unroll
  for (int k = 0; k < 2 * kP; ++k) {
    open[k] = v[0][k] + v[1][k] + mask;
#pragma unroll
    for (int p = 0; p < 2; ++p) w[p][k] = trunc_table_word(eh.h[p], epi.table[p], epi.f, open[k]);
  }
#pragma unroll
  for (int k = 0; k < 2 * kP; ++k)
#pragma unroll
    for (int p = 0; p < 2; ++p) v[p][k] = trunc_table_out(eh.h[p], epi.f, open[k], w[p][k]);
}

struct RotaryArgs {
  Rows x;
  Rot rot;
  const int32_t* positions;
  uint64_t* out[2];
  int64_t ots, ohs;
  int token0, heads, dim, units;
  uint32_t total;  // tokens of this launch * heads * units
  FastDiv by_units, by_heads;
  TruncEpi epi;
  uint64_t mask;
};

template <int kP, bool kTrunc>
__global__ void __launch_bounds__(kBlock) rotary2_kernel(RotaryArgs a) {
  const uint32_t g = blockIdx.x * kBlock + threadIdx.x;
  if (g >= a.total) return;
  const uint32_t row = div_by(a.by_units, g);
  const uint32_t tl = div_by(a.by_heads, row);
  const int64_t t = a.token0 + int64_t(tl);
  const int64_t h = row - tl * uint32_t(a.heads);
  const Unit u = unit_of<kP>(a.rot, a.dim, int(g - row * uint32_t(a.units)));
  const int pos = a.positions[t];
  uint64_t v[2][2 * kP];
#pragma unroll
  for (int p = 0; p < 2; ++p) load_unit<kP>(a.x.p[p] + t * a.x.ts + h * a.x.hs, u, v[p]);
  if (pos < 0 || pos >= a.rot.positions) return;
  int64_t c[kP], s[kP];
  load_factors<kP>(a.rot, u, pos, c, s);
#pragma unroll
  for (int p = 0; p < 2; ++p) turn<kP>(a.rot, u, c, s, v[p]);
  if constexpr (kTrunc) {
    const EpiHdrs eh = epi_hdrs(a.epi);
    trunc_unit<kP>(a.epi, eh, a.mask, v);
  }
#pragma unroll
  for (int p = 0; p < 2; ++p)
    store_unit<kP>((kTrunc ? a.epi.y[p] : a.out[p]) + t * a.ots + h * a.ohs, u, v[p]);
}

struct AppendPart {
  Rows x;
  const uint64_t* mask[2];
  KvPool pool;
  Rot rot;  // off: half 0, pass_mul 1
  const int32_t* positions;
  int units;
  uint32_t total;
  FastDiv by_units, by_heads;
  TruncEpi epi;
  uint64_t trunc_mask;
};
struct AppendArgs {
  KvBatch b;
  AppendPart part[2];
  uint32_t blocks0;  // workgroups of part 0
};

template <int kP, bool kTrunc>
__device__ __forceinline__ void append_unit(const KvBatch& b, const AppendPart& a, uint32_t g) {
  if (g >= a.total) return;
  const uint32_t row = div_by(a.by_units, g);
  const uint32_t tl = div_by(a.by_heads, row);
  const int64_t t = tl;
  const int h = int(row - tl * uint32_t(a.pool.heads));
  const Unit u = unit_of<kP>(a.rot, a.pool.dim, int(g - row * uint32_t(a.units)));
  const int64_t dense = int64_t(row) * a.pool.dim;
  uint64_t v[2][2 * kP], m[2][2 * kP];
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    load_unit<kP>(a.x.p[p] + t * a.x.ts + h * a.x.hs, u, v[p]);
    load_unit<kP>(a.mask[p] + dense, u, m[p]);
  }
  const int s = seq_of(b, int(tl));
  if (s < 0) return;
  const int64_t at = int64_t(b.lens[s]) - b.cu[s + 1] + t;
  const int64_t place = kv_place(b, a.pool, s, h, at);
  if (place < 0) return;
  if (a.rot.on) {
    const int64_t pos = a.positions ? a.positions[t] : at;
    if (pos < 0 || pos >= a.rot.positions) return;
    int64_t c[kP], sn[kP];
    load_factors<kP>(a.rot, u, int(pos), c, sn);
#pragma unroll
    for (int p = 0; p < 2; ++p) turn<kP>(a.rot, u, c, sn, v[p]);
  }
  if constexpr (kTrunc) {
    if (a.epi.on) {
      const EpiHdrs eh = epi_hdrs(a.epi);
      trunc_unit<kP>(a.epi, eh, a.trunc_mask, v);
      if (a.epi.y[0]) {
        store_unit<kP>(a.epi.y[0] + dense, u, v[0]);
        store_unit<kP>(a.epi.y[1] + dense, u, v[1]);
      }
    }
  }
  uint64_t e[2 * kP];
#pragma unroll
  for (int k = 0; k < 2 * kP; ++k) e[k] = v[0][k] + v[1][k] - m[0][k] - m[1][k];
  store_unit<kP>(a.pool.e + place, u, e);
  store_unit<kP>(a.pool.b[0] + place, u, m[0]);
  store_unit<kP>(a.pool.b[1] + place, u, m[1]);
}

template <int kP, bool kTrunc>
__global__ void __launch_bounds__(kBlock) kv_append2_kernel(AppendArgs a) {
  if (blockIdx.x < a.blocks0)
    append_unit<kP, kTrunc>(a.b, a.part[0], blockIdx.x * kBlock + threadIdx.x);
  else
    append_unit<kP, kTrunc>(a.b, a.part[1], (blockIdx.x - a.blocks0) * kBlock + threadIdx.x);
}

bool at16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Pieces of two words: everything 16-byte aligned and even.
bool rot_even(const Rot& r) { return (r.half & 1) == 0 && at16(r.table); }
bool rows_even(const Rows& r) {
  return at16(r.p[0]) && at16(r.p[1]) && (r.ts & 1) == 0 && (r.hs & 1) == 0;
}

int rot_of(const sufhip_rotary& g, int dim, const char* what, Rot* out) {
  if (!g.d_table && g.positions == 0) {  // no rotation
    *out = {nullptr, 0, 0, 0, 0, 1};
    return SUFHIP_OK;
  }
  if (g.positions < 0 || g.rot < 0 || (g.rot & 1) || g.rot > dim || (g.rot > 0 && !g.d_table) ||
      (reinterpret_cast<uintptr_t>(g.d_table) & 7))
    return kv_fail(what, "a rotary table needs positions >= 0, an even rot in [0, dim] and 8-byte "
                         "alignment");
  *out = {g.d_table, g.positions, g.rot / 2, g.interleaved ? 1 : 0, 1, uint64_t(g.pass_mul)};
  return SUFHIP_OK;
}

// Whether an array of one pool shares a word with one of the other's.
bool pools_meet(const sufhip_kv_pool& a, const sufhip_kv_pool& b) {
  const auto bytes = [](const sufhip_kv_pool& p) {
    return 8 * size_t(p.pages) * size_t(p.kv_heads) * size_t(p.page_tokens) * size_t(p.dim);
  };
  const size_t na = bytes(a), nb = bytes(b);
  const uint64_t* const pa[3] = {a.e, a.b[0], a.b[1]};
  const uint64_t* const pb[3] = {b.e, b.b[0], b.b[1]};
  for (const uint64_t* x : pa)
    for (const uint64_t* y : pb) {
      const uintptr_t u = reinterpret_cast<uintptr_t>(x), v = reinterpret_cast<uintptr_t>(y);
      if (u < v + nb && v < u + na) return true;
    }
  return false;
}

int rows_of(const sufhip_rows2& g, const char* what, Rows* out) {
  if (!g.p[0] || !g.p[1] || g.token_stride < 0 || g.head_stride < 0)
    return kv_fail(what, "rows need both parties' pointers and strides >= 0");
  *out = {{g.p[0], g.p[1]}, g.token_stride, g.head_stride};
  return SUFHIP_OK;
}

// Rows of dim words each at p + t ts + h hs (words), t < tokens, h < heads.
struct Lattice {
  const uint64_t* p;
  int64_t ts, hs;
};

// Whether the extents of two sets of rows meet.
bool extents_meet(const Lattice& a, const Lattice& b, int tokens, int heads, int dim) {
  const auto last = [&](const Lattice& r) {
    return __int128(reinterpret_cast<uintptr_t>(r.p)) +
           8 * ((__int128(tokens) - 1) * r.ts + (__int128(heads) - 1) * r.hs + dim);
  };
  return __int128(reinterpret_cast<uintptr_t>(a.p)) < last(b) &&
         __int128(reinterpret_cast<uintptr_t>(b.p)) < last(a);
}

// Whether a row of one set shares a word with a row of another set of the same
// strides `by` bytes after it; by = 0: with another row of the same set.  Two
// rows i tokens and j heads apart do if |by + 8 (i ts + j hs)| < 8 dim: for each
// step along the shorter axis the two steps along the longer one that come
// nearest decide.
bool rows_meet(__int128 by, int64_t ts, int64_t hs, int tokens, int heads, int dim) {
  __int128 n[2] = {tokens, heads}, step[2] = {8 * __int128(ts), 8 * __int128(hs)};
  const __int128 row = 8 * __int128(dim);
  if (n[0] > n[1]) {
    std::swap(n[0], n[1]);
    std::swap(step[0], step[1]);
  }
  if (by == 0) {
    // Rows side by side, and those as a whole: the usual layouts.
    const int in = n[1] == 1 || (n[0] > 1 && step[0] < step[1]) ? 0 : 1;
    if ((n[in] == 1 || step[in] >= row) &&
        (n[1 - in] == 1 || step[1 - in] >= (n[in] - 1) * step[in] + row))
      return false;
  }
  for (__int128 i = 1 - n[0]; i < n[0]; ++i) {
    const __int128 at = by + i * step[0];
    __int128 j = step[1] == 0 ? 0 : -at / step[1];
    for (__int128 k = j - 1; k <= j + 1; ++k) {
      if (k <= -n[1] || k >= n[1] || (by == 0 && i == 0 && k == 0)) continue;
      const __int128 d = at + k * step[1];
      if (d < row && -d < row) return true;
    }
  }
  return false;
}

// What a rotation's outputs may not be: rows that share words with each other,
// with the other party's, or with input rows other than their own.
int rotary_overlap(const Rows& x, uint64_t* const (&y)[2], int64_t ots, int64_t ohs, int tokens,
                   int heads, int dim, const char* what) {
  const auto apart = [](const void* a, const void* b) {
    return __int128(reinterpret_cast<uintptr_t>(a)) - __int128(reinterpret_cast<uintptr_t>(b));
  };
  const Lattice o[2] = {{y[0], ots, ohs}, {y[1], ots, ohs}};
  if (rows_meet(0, ots, ohs, tokens, heads, dim) || y[0] == y[1] ||
      (extents_meet(o[0], o[1], tokens, heads, dim) &&
       rows_meet(apart(y[0], y[1]), ots, ohs, tokens, heads, dim)))
    return kv_fail(what, "output rows overlap");
  const bool like = (tokens == 1 || x.ts == ots) && (heads == 1 || x.hs == ohs);
  for (int p = 0; p < 2; ++p)
    for (int q = 0; q < 2; ++q) {
      if (!extents_meet({x.p[p], x.ts, x.hs}, o[q], tokens, heads, dim)) continue;
      if (like && (x.p[p] == y[q] ||
                   !rows_meet(apart(x.p[p], y[q]), ots, ohs, tokens, heads, dim)))
        continue;
      return kv_fail(what, "outputs overlap other input rows than their own");
    }
  return SUFHIP_OK;
}

}  // namespace
}  // namespace sufhip

using namespace sufhip;

extern "C" {

int sufhip_rotary2(const sufhip_rotary2_args* args, void* stream) {
  const char* what = "sufhip_rotary2";
  SUFHIP_REQUIRE(args != nullptr, "sufhip_rotary2: null args");
  const sufhip_rotary2_args& g = *args;
  SUFHIP_REQUIRE(g.tokens >= 0 && g.heads >= 0 && g.dim >= 0,
                 "sufhip_rotary2: tokens, heads and dim must be >= 0");
  if (g.tokens == 0 || g.heads == 0 || g.dim == 0) return SUFHIP_OK;
  SUFHIP_REQUIRE(g.d_positions, "sufhip_rotary2: null d_positions");
  RotaryArgs a{};
  if (int rc = rows_of(g.x, what, &a.x)) return rc;
  if (int rc = rot_of(g.rot, g.dim, what, &a.rot)) return rc;
  const size_t n = size_t(g.tokens) * size_t(g.heads) * size_t(g.dim);
  if (int rc = make_epi(g.trunc, n, what, &a.epi)) return rc;
  SUFHIP_REQUIRE(!a.epi.add[0], "sufhip_rotary2: the truncation takes no addend");
  SUFHIP_REQUIRE(a.epi.on || (g.out[0] && g.out[1]),
                 "sufhip_rotary2: outputs (or a truncation) needed");
  SUFHIP_REQUIRE(g.out_token_stride >= 0 && g.out_head_stride >= 0,
                 "sufhip_rotary2: strides must be >= 0");
  a.positions = g.d_positions;
  a.ots = g.out_token_stride;
  a.ohs = g.out_head_stride;
  a.heads = g.heads;
  a.dim = g.dim;
  a.mask = g.mask;
  for (int p = 0; p < 2; ++p) a.out[p] = g.out[p];
  uint64_t* const y[2] = {a.epi.on ? a.epi.y[0] : g.out[0], a.epi.on ? a.epi.y[1] : g.out[1]};
  const bool vec = (g.dim & 1) == 0 && rot_even(a.rot) && rows_even(a.x) &&
                   rows_even(Rows{{y[0], y[1]}, a.ots, a.ohs});
  a.units = units_of(vec ? 2 : 1, a.rot.half, g.dim);
  const uint64_t per_token = uint64_t(g.heads) * uint64_t(a.units);
  SUFHIP_REQUIRE(per_token <= kMaxUnits, "sufhip_rotary2: heads * dim too large");
  if (int rc = rotary_overlap(a.x, y, a.ots, a.ohs, g.tokens, g.heads, g.dim, what)) return rc;
  a.by_units = fast_div(uint32_t(a.units));
  a.by_heads = fast_div(uint32_t(g.heads));
  const int step = int(kMaxUnits / per_token);  // tokens of one launch
  for (int t = 0; t < g.tokens; t += step) {
    const int count = g.tokens - t < step ? g.tokens - t : step;
    a.token0 = t;
    a.total = uint32_t(uint64_t(count) * per_token);
    const dim3 grid(grid_for(a.total, kBlock)), block(kBlock);
    const hipStream_t st = as_stream(stream);
    if (vec && a.epi.on)
      hipLaunchKernelGGL((rotary2_kernel<2, true>), grid, block, 0, st, a);
    else if (vec)
      hipLaunchKernelGGL((rotary2_kernel<2, false>), grid, block, 0, st, a);
    else if (a.epi.on)
      hipLaunchKernelGGL((rotary2_kernel<1, true>), grid, block, 0, st, a);
    else
      hipLaunchKernelGGL((rotary2_kernel<1, false>), grid, block, 0, st, a);
    if (int rc = check_launch("rotary2_kernel")) return rc;
    if (g.tokens - t <= step) break;
  }
  return SUFHIP_OK;
}

int sufhip_kv_append2(const sufhip_kv_append2_args* args, void* stream) {
  const char* what = "sufhip_kv_append2";
  SUFHIP_REQUIRE(args != nullptr, "sufhip_kv_append2: null args");
  AppendArgs a{};
  if (int rc = kv_batch_of(args->batch, what, &a.b)) return rc;
  // No rows: arrays of none may be null.
  const bool empty = a.b.seqs == 0 || a.b.tokens == 0;
  bool vec = true, trunc = false;
  for (int k = 0; k < 2; ++k) {
    const sufhip_kv_append_part& g = args->part[k];
    AppendPart& q = a.part[k];
    if (!g.pool.e) continue;
    if (int rc = kv_pool_of(g.pool, what, &q.pool)) return rc;
    if (int rc = rot_of(g.rot, g.pool.dim, what, &q.rot)) return rc;
    if (empty) continue;
    if (int rc = rows_of(g.x, what, &q.x)) return rc;
    SUFHIP_REQUIRE(g.mask[0] && g.mask[1], "sufhip_kv_append2: null mask");
    const size_t n = size_t(a.b.tokens) * size_t(q.pool.heads) * size_t(q.pool.dim);
    if (int rc = make_epi(g.trunc, n, what, &q.epi, false)) return rc;
    SUFHIP_REQUIRE(!q.epi.add[0], "sufhip_kv_append2: the truncation takes no addend");
    q.mask[0] = g.mask[0];
    q.mask[1] = g.mask[1];
    q.positions = g.d_positions;
    q.trunc_mask = g.trunc_mask;
    trunc = trunc || q.epi.on;
    vec = vec && (q.pool.dim & 1) == 0 && rot_even(q.rot) && rows_even(q.x) &&
          at16(g.mask[0]) && at16(g.mask[1]) && at16(g.pool.e) && at16(g.pool.b[0]) &&
          at16(g.pool.b[1]) && at16(q.epi.y[0]) && at16(q.epi.y[1]);
  }
  if (empty) return SUFHIP_OK;
  uint64_t blocks[2] = {0, 0};
  for (int k = 0; k < 2; ++k) {
    AppendPart& q = a.part[k];
    if (!q.pool.e) continue;
    q.units = units_of(vec ? 2 : 1, q.rot.half, q.pool.dim);
    const uint64_t total = uint64_t(a.b.tokens) * uint64_t(q.pool.heads) * uint64_t(q.units);
    SUFHIP_REQUIRE(total <= kMaxUnits, "sufhip_kv_append2: more than 2^30 pairs in one call");
    q.total = uint32_t(total);
    q.by_units = fast_div(uint32_t(q.units));
    q.by_heads = fast_div(uint32_t(q.pool.heads));
    blocks[k] = grid_for(q.total, kBlock);
  }
  if (blocks[0] + blocks[1] == 0) return SUFHIP_OK;
  SUFHIP_REQUIRE(blocks[0] == 0 || blocks[1] == 0 ||
                     !pools_meet(args->part[0].pool, args->part[1].pool),
                 "sufhip_kv_append2: the parts' pools share memory");
  a.blocks0 = uint32_t(blocks[0]);
  const dim3 grid(unsigned(blocks[0] + blocks[1])), block(kBlock);
  const hipStream_t st = as_stream(stream);
  if (vec && trunc)
    hipLaunchKernelGGL((kv_append2_kernel<2, true>), grid, block, 0, st, a);
  else if (vec)
    hipLaunchKernelGGL((kv_append2_kernel<2, false>), grid, block, 0, st, a);
  else if (trunc)
    hipLaunchKernelGGL((kv_append2_kernel<1, true>), grid, block, 0, st, a);
  else
    hipLaunchKernelGGL((kv_append2_kernel<1, false>), grid, block, 0, st, a);
  return check_launch("kv_append2_kernel");
}

}  // extern "C"
