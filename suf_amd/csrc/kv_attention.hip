// The two products of attention over a paged cache, both parties, exact mod
// 2^64 (sufhip_kv_scores2, sufhip_kv_values2).
//
// With D = (x_0 - a_0) + (x_1 - a_1) a party's share of a product is
//   Z_p = C_p + D B_p + L_p E,   L_0 = A_0 + D,  L_1 = A_1,
// E and B_p read from the cache's pages: four products of u64 matrices.  Each
// is 36 products of int8 digit matrices (digits i, j of weight 256^(i + j) below
// 2^64), 144 matrix instructions for both parties' 16 x 16 results over 64 of
// k; the digits' sums are exact in int32, and joined in 64 bits.
//
// What bounds them: single tokens read the cache once, 24 bytes a cached value,
// at the rate of a large copy; prompts use each cached word for many rows, and
// there the matrix instructions (16 cycles a SIMD) and what forms their digits
// (4 to 5 cycles a vector instruction, of which the other wave of a SIMD
// issues about two under each matrix instruction) share the time with the
// packed elements' traffic, 32 bytes each.
#include <hip/hip_runtime.h>

#include <atomic>

#include "digit_planes.hpp"
#include "kv_device.hpp"
#include "suf_hip.h"
#include "sufhip_internal.hpp"
#include "trunc_device.hpp"

namespace sufhip {
namespace {

struct ProductArgs {
  KvBatch b;
  KvPool pool;
  int heads, group;
  FastDiv by_group;
  const uint64_t* x[2];
  int64_t xts, xhs;
  const uint64_t* a[2];
  const uint64_t* c[2];
  const int32_t* offsets;
  int64_t n;
  uint64_t* out[2];
  TruncEpi epi;
  uint64_t mask;
};

// Both parties' finished values of output element i: to the outputs, or the
// open through the truncation gate.
template <bool kTrunc>
struct Put {
  __device__ __forceinline__ explicit Put(const ProductArgs&) {}
  __device__ __forceinline__ void operator()(const ProductArgs& a, int64_t i, uint64_t z0,
                                             uint64_t z1) const {
    a.out[0][i] = z0;
    a.out[1][i] = z1;
  }
};
template <>
struct Put<true> {
  EpiHdrs eh;
  __device__ __forceinline__ explicit Put(const ProductArgs& a) : eh(epi_hdrs(a.epi)) {}
  __device__ __forceinline__ void operator()(const ProductArgs& a, int64_t i, uint64_t z0,
                                             uint64_t z1) const {
    const uint64_t open = z0 + z1 + a.mask;
    const uint64_t w0 = trunc_table_word(eh.h[0], a.epi.table[0], a.epi.f, open);
    const uint64_t w1 = trunc_table_word(eh.h[1], a.epi.table[1], a.epi.f, open);
    a.epi.y[0][i] = trunc_table_out(eh.h[0], a.epi.f, open, w0);
    a.epi.y[1][i] = trunc_table_out(eh.h[1], a.epi.f, open, w1);
  }
};

// A row's elements by key: where key's words of C are and its outputs go.
// kBuffer: packed arrays of fewer than 2^29 elements as buffers, whose range
// check drops a store past their end and reads zeros there.  Keys without an
// element then need no branch, so the memory operations under way stay counted
// and a wave waits for the words that it uses alone, not for the stores of the
// tile before (32 row tiles of 4 x 2112 keys, 4 cached heads: 426 -> 380 us with
// heads of 128, 222 -> 219 with 64).
constexpr int64_t kBufferMost = (int64_t(1) << 29) - 1;
template <bool kTrunc, bool kBuffer>
struct Elements;
template <bool kTrunc>
struct Elements<kTrunc, false> {
  Put<kTrunc> put_;
  __device__ __forceinline__ explicit Elements(const ProductArgs& a) : put_(a) {}
  __device__ __forceinline__ uint32_t at(int first, int len, int key) const {
    return key < len ? uint32_t(first + key) : ~0u;
  }
  __device__ __forceinline__ uint64_t c(const ProductArgs& a, int p, uint32_t at) const {
    return a.c[p][at == ~0u ? 0 : at];
  }
  __device__ __forceinline__ void put(const ProductArgs& a, uint32_t at, uint64_t z0,
                                      uint64_t z1) const {
    if (at != ~0u) put_(a, at, z0, z1);
  }
};
template <bool kTrunc>
struct Elements<kTrunc, true> {
  EpiHdrs eh;
  __amdgpu_buffer_rsrc_t c_[2], out[2];
  static __device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const uint64_t* p, int64_t n) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint64_t*>(p), 0, int(uint32_t(8 * n)),
                                             0x00020000);
  }
  __device__ __forceinline__ explicit Elements(const ProductArgs& a) {
    if constexpr (kTrunc) eh = epi_hdrs(a.epi);
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      c_[p] = buffer(a.c[p], a.n);
      out[p] = buffer(kTrunc ? a.epi.y[p] : a.out[p], a.n);
    }
  }
  __device__ __forceinline__ uint32_t at(int first, int len, int key) const {
    return key < len ? 8 * uint32_t(first + key) : 0xfffffff8u;
  }
  __device__ __forceinline__ uint64_t c(const ProductArgs&, int p, uint32_t at) const {
    const auto w = __builtin_amdgcn_raw_buffer_load_b64(c_[p], at, 0, 0);
    return uint64_t(w[0]) | uint64_t(w[1]) << 32;
  }
  __device__ __forceinline__ void store(int p, uint32_t at, uint64_t v) const {
    typedef unsigned v2u __attribute__((ext_vector_type(2)));
    __builtin_amdgcn_raw_buffer_store_b64(v2u{unsigned(v), unsigned(v >> 32)}, out[p], at, 0, 0);
  }
  __device__ __forceinline__ void put(const ProductArgs& a, uint32_t at, uint64_t z0,
                                      uint64_t z1) const {
    if constexpr (kTrunc) {
      const uint64_t open = z0 + z1 + a.mask;
      const uint64_t w0 = trunc_table_word(eh.h[0], a.epi.table[0], a.epi.f, open);
      const uint64_t w1 = trunc_table_word(eh.h[1], a.epi.table[1], a.epi.f, open);
      z0 = trunc_table_out(eh.h[0], a.epi.f, open, w0);
      z1 = trunc_table_out(eh.h[1], a.epi.f, open, w1);
    }
    store(0, at, z0);
    store(1, at, z1);
  }
};

// ---- digits ----
//
// v = sum_i d_i 256^i with d_i in [-128, 127]: adding 128 to every byte (with
// its carries) and flipping the bytes' top bits again leaves d_i in byte i.
constexpr uint64_t kBias = 0x8080808080808080ull;

// Planes of 4 values: pl[i] = digit i of v[0..3], lowest byte first.
__device__ __forceinline__ void digits_of4(const uint64_t (&v)[4], uint32_t (&pl)[8]) {
  uint32_t w[2][4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint64_t u = (v[k] + kBias) ^ kBias;
    w[0][k] = uint32_t(u);
    w[1][k] = uint32_t(u >> 32);
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t a = __builtin_amdgcn_perm(w[h][1], w[h][0], 0x05010400u);
    const uint32_t b = __builtin_amdgcn_perm(w[h][1], w[h][0], 0x07030602u);
    const uint32_t c = __builtin_amdgcn_perm(w[h][3], w[h][2], 0x05010400u);
    const uint32_t d = __builtin_amdgcn_perm(w[h][3], w[h][2], 0x07030602u);
    pl[4 * h] = __builtin_amdgcn_perm(c, a, 0x05040100u);
    pl[4 * h + 1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
    pl[4 * h + 2] = __builtin_amdgcn_perm(d, b, 0x05040100u);
    pl[4 * h + 3] = __builtin_amdgcn_perm(d, b, 0x07060302u);
  }
}

// Planes of a lane's 16 values of a matrix-core operand.
__device__ __forceinline__ void digits_of16(const uint64_t (&v)[16], v4i (&pl)[kDigitPlanes]) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const uint64_t f[4] = {v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
    uint32_t d[8];
    digits_of4(f, d);
#pragma unroll
    for (int i = 0; i < kDigitPlanes; ++i) pl[i][q] = int(d[i]);
  }
}

// The value of digit sums S_s: sum_s 256^s S_s mod 2^64.  Sums 4 to 7 reach
// only the high word.
__device__ __forceinline__ uint64_t from_sums(const v4i (&acc)[kDigitPlanes], int r) {
  const uint32_t hi = ((((uint32_t(acc[7][r]) << 8) + uint32_t(acc[6][r])) << 8) +
                       uint32_t(acc[5][r])) * 256u + uint32_t(acc[4][r]);
  uint64_t lo = uint64_t(int64_t(acc[3][r]));
  lo = (lo << 8) + uint64_t(int64_t(acc[2][r]));
  lo = (lo << 8) + uint64_t(int64_t(acc[1][r]));
  lo = (lo << 8) + uint64_t(int64_t(acc[0][r]));
  return lo + (uint64_t(hi) << 32);
}

// ---- left operands in LDS ----
//
// One 16 x 64 tile (16 rows, 64 of k) of the three left operands D, L_0, L_1
// as digit planes of 1 KB (plane i of operand o at o * 8192 + i * 1024), where
// byte j of k group g of row r is byte j of the 16-byte cell below: a lane's
// operand is one cell.  The rows are exchanged within a group so that neither
// the 16-byte reads nor the writes of a wave (all groups of 2 rows) meet on
// LDS banks.
constexpr int kTileBytes = 3 * kDigitPlanes * 1024;
__device__ __forceinline__ int cell(int r, int g) {
  return (16 * g + (r ^ (2 * (g & 1) + 12 * (g >> 1)))) * 16;
}

// kN of a row's k from byte j0 of group g on (kN = 2 or 4, j0 a multiple).
template <int kN>
__device__ __forceinline__ void put_digits(int8_t* plane0, const uint64_t (&v)[kN]) {
  if constexpr (kN == 4) {
    uint32_t pl[8];
    digits_of4(v, pl);
#pragma unroll
    for (int i = 0; i < 8; ++i) *reinterpret_cast<uint32_t*>(plane0 + i * 1024) = pl[i];
  } else {
    const uint64_t u0 = (v[0] + kBias) ^ kBias, u1 = (v[1] + kBias) ^ kBias;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t w0 = uint32_t(u0 >> (32 * h)), w1 = uint32_t(u1 >> (32 * h));
      const uint32_t a = __builtin_amdgcn_perm(w1, w0, 0x05010400u);
      const uint32_t b = __builtin_amdgcn_perm(w1, w0, 0x07030602u);
      int8_t* p = plane0 + 4096 * h;
      *reinterpret_cast<uint16_t*>(p) = uint16_t(a);
      *reinterpret_cast<uint16_t*>(p + 1024) = uint16_t(a >> 16);
      *reinterpret_cast<uint16_t*>(p + 2 * 1024) = uint16_t(b);
      *reinterpret_cast<uint16_t*>(p + 3 * 1024) = uint16_t(b >> 16);
    }
  }
}

// kN words of each array a left operand is formed from.
template <int kN>
struct Raw {
  uint64_t x0[kN], x1[kN], a0[kN], a1[kN];
};
template <int kN>
__device__ __forceinline__ void put_left(int8_t* tile, int r, int g, int j0, const Raw<kN>& v) {
  uint64_t d[kN], l0[kN];
#pragma unroll
  for (int k = 0; k < kN; ++k) {
    d[k] = (v.x0[k] - v.a0[k]) + (v.x1[k] - v.a1[k]);
    l0[k] = v.a0[k] + d[k];
  }
  int8_t* p = tile + cell(r, g) + j0;
  put_digits<kN>(p, d);
  put_digits<kN>(p + 8192, l0);
  put_digits<kN>(p + 16384, v.a1);
}

// Plane i of operand o for lane l (row l % 16, k group l / 16).
__device__ __forceinline__ v4i get_left(const int8_t* tile, int o, int l, int i) {
  return *reinterpret_cast<const v4i*>(tile + o * 8192 + i * 1024 + cell(l & 15, l >> 4));
}

// acc += (left operand o) r over the digit pairs of weight below 256^8.
__device__ __forceinline__ void mul_left(const int8_t* tile, int o, int l,
                                         const v4i (&r)[kDigitPlanes],
                                         v4i (&acc)[kDigitPlanes]) {
#pragma unroll
  for (int i = 0; i < kDigitPlanes; ++i) {
    const v4i x = get_left(tile, o, l, i);
#pragma unroll
    for (int j = 0; i + j < kDigitPlanes; ++j)
      acc[i + j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x, r[j], acc[i + j], 0, 0, 0);
  }
}

// Both parties' digit products of a left tile with the right operands: D with
// the parties' masks, then all of them.
__device__ __forceinline__ void mul_opened(const int8_t* tile, int l,
                                           const v4i (&b0)[kDigitPlanes],
                                           const v4i (&b1)[kDigitPlanes],
                                           v4i (&acc)[2][kDigitPlanes]) {
#pragma unroll
  for (int i = 0; i < kDigitPlanes; ++i) {
    const v4i x = get_left(tile, 0, l, i);
#pragma unroll
    for (int j = 0; i + j < kDigitPlanes; ++j) {
      acc[0][i + j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x, b0[j], acc[0][i + j], 0, 0, 0);
      acc[1][i + j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x, b1[j], acc[1][i + j], 0, 0, 0);
    }
  }
}

__device__ __forceinline__ void mul_tile(const int8_t* tile, int l, const v4i (&e)[kDigitPlanes],
                                         const v4i (&b0)[kDigitPlanes],
                                         const v4i (&b1)[kDigitPlanes],
                                         v4i (&acc)[2][kDigitPlanes]) {
  mul_opened(tile, l, b0, b1, acc);
  mul_left(tile, 1, l, e, acc[0]);
  mul_left(tile, 2, l, e, acc[1]);
}

__device__ __forceinline__ void clear(v4i (&acc)[2][kDigitPlanes]) {
#pragma unroll
  for (int p = 0; p < 2; ++p)
#pragma unroll
    for (int s = 0; s < kDigitPlanes; ++s) acc[p][s] = v4i{0, 0, 0, 0};
}

// A sequence's part of the batch for one cached head: its rows are (token,
// head of the group) in that order, row m at token t0 + m / group.
// kv: its keys, none of which a row of at most n elements can do without.
// Wrong starts (any words, in any order) still give rows of the batch: both
// ends are brought into [0, tokens] before they are subtracted.
struct Seq {
  int s, hk, t0, rows, kv;
};
__device__ __forceinline__ Seq seq_of_head(const ProductArgs& a, int s, int hk) {
  const int lo = a.b.cu[s], hi = a.b.cu[s + 1], kv = a.b.lens[s];
  Seq q;
  q.s = s;
  q.hk = hk;
  q.t0 = min(max(lo, 0), a.b.tokens);
  q.rows = max(min(max(hi, 0), a.b.tokens) - q.t0, 0) * a.group;
  q.kv = int(min(int64_t(kv), a.n));
  return q;
}
__device__ __forceinline__ Seq seq_at(const ProductArgs& a, int z) {
  const int s = z / a.pool.heads;
  return seq_of_head(a, s, z - s * a.pool.heads);
}

// Row m of a sequence: its token, its head, where its packed elements start
// and how many of them have a key (m past the last row: token -1, no
// elements; row_of: without the elements).  A row that does not lie within
// the packed elements has none.
struct Row {
  int t, h, first, len;
};
__device__ __forceinline__ Row row_of(const ProductArgs& a, const Seq& q, int m) {
  if (m >= q.rows) return {-1, 0, 0, 0};
  const int tl = int(div_by(a.by_group, uint32_t(m)));
  return {q.t0 + tl, q.hk * a.group + (m - tl * a.group), 0, 0};
}
// row_at in two halves: the row's offsets on their way, then its elements.
struct RowLoad {
  Row r;
  int from, to;
};
__device__ __forceinline__ RowLoad load_row(const ProductArgs& a, const Seq& q, int m) {
  RowLoad w{row_of(a, q, m), 0, 0};
  const int64_t i = w.r.t < 0 ? 0 : int64_t(w.r.h) * a.b.tokens + w.r.t;
  w.from = a.offsets[i];
  w.to = a.offsets[i + 1];
  return w;
}
__device__ __forceinline__ Row row_from(const ProductArgs& a, const Seq& q, const RowLoad& w) {
  Row r = w.r;
  const int64_t f = w.from, l = int64_t(w.to) - f;
  if (r.t < 0 || f < 0 || l <= 0 || f + l > a.n) return r;
  r.first = w.from;
  r.len = int(l < q.kv ? l : q.kv);
  return r;
}
__device__ __forceinline__ Row row_at(const ProductArgs& a, const Seq& q, int m) {
  return row_from(a, q, load_row(a, q, m));
}

// A key's page number on its way, then the first word of its head in the pool
// (-1: no page holds it).
struct Spot {
  int64_t key;
  int page;
};
__device__ __forceinline__ bool has_entry(const ProductArgs& a, const Seq& q, int64_t key) {
  return key < q.kv && (key >> a.pool.shift) < a.b.max_pages;
}
__device__ __forceinline__ Spot load_spot(const ProductArgs& a, const Seq& q, int64_t key) {
  const int64_t at = has_entry(a, q, key) ? key >> a.pool.shift : 0;
  return {key, a.b.table[int64_t(q.s) * a.b.max_pages + at]};
}
__device__ __forceinline__ int64_t place_at(const ProductArgs& a, const Seq& q, const Spot& w) {
  const bool ok = has_entry(a, q, w.key) && unsigned(w.page) < unsigned(a.pool.pages);
  const int64_t row = ((int64_t(w.page) * a.pool.heads + q.hk) << a.pool.shift) +
                      (w.key & ((1 << a.pool.shift) - 1));
  return ok ? row * a.pool.dim : -1;
}

// ---- even shares ----
//
// Few rows a sequence, and sequences of any lengths: the work is cut into
// units of 64 keys of one item (row tile, column block, cached head of a
// sequence), in that order within each sequence, and every workgroup takes
// the same number of neighbouring units, across items and sequences.  The
// lengths are in device memory, so each workgroup sums them up for itself
// (one load of each length; 256 threads scan).  An item counts one unit more
// than its keys, in front: what a workgroup spends on starting one.
constexpr int kKeyTile = 64;

struct Share {
  int64_t unit, end, per;  // this workgroup's units; units of each workgroup
};

__device__ __forceinline__ int tiles_of(int kv) {
  return kv > kKeyTile ? (kv + kKeyTile - 1) / kKeyTile : 1;
}
__device__ __forceinline__ int64_t units_of(const ProductArgs& a, int s, int blocks) {
  const Seq q = seq_of_head(a, s, 0);
  return int64_t((q.rows + 15) / 16) * blocks * a.pool.heads * (tiles_of(q.kv) + 1);
}

// Sums before each of the 256 threads' sequences into pre[0 .. 256] (a
// workgroup of 256), and the workgroup's share.
__device__ __forceinline__ Share share_of(const ProductArgs& a, int blocks, int64_t (&pre)[260]) {
  const int tid = threadIdx.x, l = tid & 63;
  if (a.b.seqs == 1) {  // nothing to scan
    const int64_t all = units_of(a, 0, blocks);
    const int64_t n = (all + gridDim.x - 1) / gridDim.x, u = int64_t(blockIdx.x) * n;
    return {u, u + n < all ? u + n : all, n};
  }
  const int per = (a.b.seqs + 255) / 256;
  int64_t mine = 0;
  for (int s = tid * per; s < a.b.seqs && s < (tid + 1) * per; ++s) mine += units_of(a, s, blocks);
  int64_t sum = mine;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t v = __shfl_up(sum, d);
    if (l >= d) sum += v;
  }
  if (l == 63) pre[256 + (tid >> 6)] = sum;
  __syncthreads();
  int64_t before = 0, all = 0;
  for (int w = 0; w < 4; ++w) {
    if (w < (tid >> 6)) before += pre[256 + w];
    all += pre[256 + w];
  }
  __syncthreads();
  pre[tid] = before + sum - mine;
  if (tid == 0) pre[256] = all;
  __syncthreads();
  const int64_t n = (all + gridDim.x - 1) / gridDim.x;
  const int64_t u = int64_t(blockIdx.x) * n;
  return {u, u + n < all ? u + n : all, n};
}

// The item of the share's next unit: key tiles [tile, tile + count) of its
// `tiles` are the workgroup's (count 0: none), `first` and `last` the
// workgroups of its first and last ones.  Steps the share past them.
struct Piece {
  Seq q;
  int rt, block, tile, count, tiles, first, last;
};
__device__ __forceinline__ Piece piece_at(const ProductArgs& a, int blocks,
                                          const int64_t (&pre)[260], Share& sh) {
  int s = 0;
  int64_t rem = sh.unit;
  if (a.b.seqs > 1) {
    int b = 0;
#pragma unroll
    for (int step = 128; step; step >>= 1)
      if (pre[b + step] <= sh.unit) b += step;
    const int per = (a.b.seqs + 255) / 256;
    s = b * per;
    rem = sh.unit - pre[b];
    if (per > 1)
      for (int64_t n; s + 1 < a.b.seqs && (n = units_of(a, s, blocks)) <= rem; ++s) rem -= n;
  }
  Piece p;
  p.q = seq_of_head(a, s, 0);
  p.tiles = tiles_of(p.q.kv);
  const int64_t item = rem / (p.tiles + 1);
  const int at = int(rem - item * (p.tiles + 1));  // 0: the unit in front
  // Divided afresh for each piece: the divisors' reciprocals would be kept in
  // registers over the caller's loop.
  int heads = a.pool.heads;
  asm volatile("" : "+s"(heads));
  asm volatile("" : "+s"(blocks));
  const int64_t row = item / heads;
  p.q.hk = int(item - row * heads);
  p.rt = int(row / blocks);
  p.block = int(row - int64_t(p.rt) * blocks);
  const int64_t begin = sh.unit - at + 1;
  p.first = int(begin / sh.per);
  p.last = int((begin + p.tiles - 1) / sh.per);
  const int left = int(min(sh.end - sh.unit, int64_t(p.tiles + 1 - at)));
  sh.unit += left;
  p.tile = at > 0 ? at - 1 : 0;
  p.count = at > 0 ? left : left - 1;
  return p;
}

// ---- scores ----
//
// A wave takes 16 keys of one cached head (the columns of a 16 x 16 tile), a
// workgroup 16 for each of its waves.  The keys' digits are formed in
// registers straight from the pages, the rows' pass through LDS.  k order:
// byte j = 2 i + e of group g stands for dim 8 i + 2 g + e of a 64-wide
// chunk, so each of a lane's 16-byte loads has its neighbours' beside it (64
// contiguous bytes a key).
//
// Every lane loads from its page or, where there is none (past the last key,
// a page number outside the pool), from the pool's first word: a key reaches
// its own column alone, and that column's product is dropped.  Values past a
// head's last meet zero digits of the left operand.  So no load is
// conditional, and the loads of a tile leave together.

// kFull: dim is a multiple of 64.
template <bool kVec, bool kFull>
__device__ __forceinline__ void load_keys(const uint64_t* p, int g, int left, uint64_t (&v)[16]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d = 8 * i + 2 * g;
    if constexpr (kVec) {
      const ulonglong2 w = *reinterpret_cast<const ulonglong2*>(p + (kFull || d < left ? d : 0));
      v[2 * i] = w.x;
      v[2 * i + 1] = w.y;
    } else {
      v[2 * i] = p[d < left ? d : 0];
      v[2 * i + 1] = p[d + 1 < left ? d + 1 : 0];
    }
  }
}

// Words at dims d (+ 8 for the second pair).
template <int kN, bool kVec, bool kFull>
__device__ __forceinline__ void load_left(const uint64_t* p, int d, int left, uint64_t (&v)[kN]) {
#pragma unroll
  for (int h = 0; h < kN / 2; ++h) {
    const int o = d + 8 * h;
    if constexpr (kVec) {
      ulonglong2 w = make_ulonglong2(0, 0);
      if (kFull || o < left) w = *reinterpret_cast<const ulonglong2*>(p + o);
      v[2 * h] = w.x;
      v[2 * h + 1] = w.y;
    } else {
      v[2 * h] = o < left ? p[o] : 0;
      v[2 * h + 1] = o + 1 < left ? p[o + 1] : 0;
    }
  }
}

// kN of a 64-wide chunk of a row's left operands, of 64 / kN threads a row:
// thread part takes group part % 4, bytes kN (part / 4) on.  A thread whose
// words lie past the head's last leaves v as it is (zeros from the start).
template <int kN, bool kVec, bool kFull>
__device__ __forceinline__ void load_raw(const ProductArgs& a, const Row& r, int c, int part,
                                         Raw<kN>& v) {
  const int d = 4 * kN * (part >> 2) + 2 * (part & 3), left = a.pool.dim - 64 * c;
  if (r.t < 0 || d >= left) return;
  const int64_t t = max(r.t, 0);
  const int64_t xo = t * a.xts + int64_t(r.h) * a.xhs + 64 * c;
  const int64_t ao = (t * a.heads + r.h) * a.pool.dim + 64 * c;
  load_left<kN, kVec, kFull || (kVec && kN == 2)>(a.x[0] + xo, d, left, v.x0);
  load_left<kN, kVec, kFull || (kVec && kN == 2)>(a.x[1] + xo, d, left, v.x1);
  load_left<kN, kVec, kFull || (kVec && kN == 2)>(a.a[0] + ao, d, left, v.a0);
  load_left<kN, kVec, kFull || (kVec && kN == 2)>(a.a[1] + ao, d, left, v.a1);
}
// Rows past the last write what their registers hold, or the first token's
// words: a row of the left operand reaches that row of the product alone, and
// it is not stored.
template <int kN>
__device__ __forceinline__ void put_raw(int8_t* tile, int row, int part, const Raw<kN>& v) {
  put_left<kN>(tile, row, part & 3, kN * (part >> 2), v);
}

// The longest row of a tile.
__device__ __forceinline__ int longest(const Row (&rows)[16]) {
  int most = 0;
#pragma unroll
  for (int r = 0; r < 16; ++r) most = rows[r].len > most ? rows[r].len : most;
  return __builtin_amdgcn_readfirstlane(most);
}

// The shortest.
__device__ __forceinline__ int shortest(const Row (&rows)[16]) {
  int least = rows[0].len;
#pragma unroll
  for (int r = 1; r < 16; ++r) least = rows[r].len < least ? rows[r].len : least;
  return __builtin_amdgcn_readfirstlane(least);
}

// Few rows: a workgroup keeps one row tile in LDS and streams its units of
// the keys.  Bound by HBM: an array's 16 words a lane are turned into digits,
// the next unit's loads leave into the same registers, and the matrix cores
// run under them, so a wave has up to 24 KB in flight.  Two workgroups a CU
// (256 registers a wave).  16 sequences of up to 4096 keys, 8 cached heads of
// 128, 4 queries each: 190 us, 852 MB at 4.5 TB/s.  One sequence of 300 keys,
// 12 heads of 64: 11 us, a chain of loads that wait for one another (lengths,
// page numbers, keys: 6 us), one unit's product (3) and the store (1.5); the
// loads of one step leave together and without branches (12.3 with them).
template <bool kVec, bool kFull, bool kTrunc>
__global__ void __launch_bounds__(256, kVec ? 2 : 1)
    kv_scores2_few_kernel(ProductArgs a, int chunks) {
  extern __shared__ __align__(16) int8_t tiles[];
  __shared__ Row rows[16];
  const int w = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6);
  const int dim = a.pool.dim;
  const Put<kTrunc> put(a);
  __shared__ int64_t pre[260];
  Share sh = share_of(a, 1, pre);
  while (sh.unit < sh.end) {
    const Piece pc = piece_at(a, 1, pre, sh);
    const Seq& q = pc.q;
    if (pc.count == 0) continue;
    // The lane's offsets are formed again for each piece: kept over the loop
    // they would take registers that it does not have.
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const int l = tid & 63, g = l >> 4, n = l & 15;
    __syncthreads();
    // The first keys' pages, the rows' words and the rows' offsets are on
    // their way together, the keys' words with the writes to LDS.
    const int tb = pc.tile;
    const auto spot_of = [&](int t) {
      return load_spot(a, q, int64_t(t) * kKeyTile + 16 * w + n);
    };
    const Spot here = spot_of(tb);
    Spot next = spot_of(tb + 1);
    const RowLoad spans = load_row(a, q, 16 * pc.rt + n);
    Raw<4> first{};
    const Row stage = row_of(a, q, 16 * pc.rt + (tid >> 4));
    load_raw<4, kVec, kFull>(a, stage, 0, tid & 15, first);
    int64_t place = place_at(a, q, here);
    uint64_t raw[3][16];
    const auto issue = [&](int k, int64_t place, int c) {
      const uint64_t* src = k == 0 ? a.pool.b[0] : k == 1 ? a.pool.b[1] : a.pool.e;
      load_keys<kVec, kFull>(src + (place < 0 ? 0 : place) + 64 * c, g, dim - 64 * c, raw[k]);
    };
#pragma unroll
    for (int k = 0; k < 3; ++k) issue(k, place, 0);
    if (tid < 16) rows[tid] = row_from(a, q, spans);
    put_raw<4>(tiles, tid >> 4, tid & 15, first);
    for (int c = 1; c < chunks; ++c) {
      Raw<4> v{};
      load_raw<4, kVec, kFull>(a, stage, c, tid & 15, v);
      put_raw<4>(tiles + c * kTileBytes, tid >> 4, tid & 15, v);
    }
    __syncthreads();
    const int all = (longest(rows) + kKeyTile - 1) / kKeyTile;
    const int te = tb + pc.count < all ? tb + pc.count : all;
    if (tb >= te) continue;
    v4i acc[2][kDigitPlanes];
    clear(acc);
    int t = tb, c = 0;
    for (int u = (te - tb) * chunks; u > 0; --u) {
      const bool last = c + 1 == chunks;
      const int64_t np = last ? place_at(a, q, next) : place;
      const int nc = last ? 0 : c + 1;
      // Read again for each chunk: no branch, and older than the loads below.
      next = spot_of(last ? t + 2 : t + 1);
      const int8_t* tile = tiles + c * kTileBytes;
      const int key = t * kKeyTile + 16 * w + n;
      uint64_t cw[2][4];
      int at[4];
      if (last) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const Row& row = rows[4 * g + r];
          at[r] = key < row.len ? row.first + key : -1;
          const int o = at[r] < 0 ? 0 : at[r];
          cw[0][r] = a.c[0][o];
          cw[1][r] = a.c[1][o];
        }
      }
      v4i y[kDigitPlanes];
      digits_of16(raw[0], y);
      issue(0, np, nc);
      mul_left(tile, 0, l, y, acc[0]);
      digits_of16(raw[1], y);
      issue(1, np, nc);
      mul_left(tile, 0, l, y, acc[1]);
      digits_of16(raw[2], y);
      issue(2, np, nc);
      mul_left(tile, 1, l, y, acc[0]);
      mul_left(tile, 2, l, y, acc[1]);
      c = nc;
      if (last) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (at[r] < 0) continue;
          const uint64_t z0 = place < 0 ? 0 : from_sums(acc[0], r);
          const uint64_t z1 = place < 0 ? 0 : from_sums(acc[1], r);
          put(a, at[r], z0 + cw[0][r], z1 + cw[1][r]);
          if constexpr (kTrunc) __builtin_amdgcn_sched_barrier(0);
        }
        clear(acc);
        ++t;
        place = np;
      }
    }
  }
}

// Many rows: a workgroup of 4 kGroups waves keeps the digits of its keys in
// registers, kHeld 64-wide chunks of them, and runs over row tiles.  Each
// thread loads its words of the next row tile, and writes their digits into
// the other half of LDS while the matrix cores work on the present one (one
// barrier a tile).  Two groups of waves over one row tile (128 keys) where a
// 64-wide chunk is all of a head: each thread then forms half as many digits.
// Three prompts (1024, 517 after 200, 33), 12 heads of 64 on 4 cached ones:
// 127 to 138 us on different cards; 342 MB needed, 493 moved, for each of the
// 60 key tiles is loaded by up to 11 workgroups of its row tiles.  Without its
// loads, stores and LDS writes the same work takes seven tenths of that, two
// thirds of it matrix instructions.
template <int kHeld, int kGroups, bool kVec, bool kFull, bool kTrunc, bool kBuffer>
__global__ void __launch_bounds__(256 * kGroups, kGroups) kv_scores2_kernel(ProductArgs a) {
  constexpr int kRows = 256 * kGroups;  // rows looked up at once
  constexpr int kKeys = 64 * kGroups;
  constexpr int kHalf = kHeld * kTileBytes;
  extern __shared__ __align__(16) int8_t tiles[];
  __shared__ Row rows[kRows];
  __shared__ unsigned active;
  const int tid = threadIdx.x, l = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = l >> 4, n = l & 15;
  const int dim = a.pool.dim;
  const Elements<kTrunc, kBuffer> io(a);
  const Seq q = seq_at(a, int(blockIdx.x));
  const int row_tiles = (q.rows + 15) / 16;
  for (int64_t first_key = int64_t(blockIdx.z) * kKeys; first_key < q.kv;
       first_key += int64_t(gridDim.z) * kKeys) {
    const int k0 = int(first_key), key = k0 + 16 * w + n;
    const int64_t place = place_at(a, q, load_spot(a, q, key));
    v4i K[kHeld][3][kDigitPlanes];
    // The lane's offsets are formed again for each key tile: kept over the
    // loop they would take registers that it does not have.
    int lane_g = g;
    asm volatile("" : "+v"(lane_g));
#pragma unroll
    for (int c = 0; c < kHeld; ++c) {
      const int64_t o = (place < 0 ? 0 : place) + 64 * c;
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        uint64_t v[16];
        load_keys<kVec, kFull>((k == 0 ? a.pool.e : a.pool.b[k - 1]) + o, lane_g, dim - 64 * c,
                               v);
        digits_of16(v, K[c][k]);
      }
    }
    for (int rb = blockIdx.y; rb < row_tiles; rb += gridDim.y * (kRows / 16)) {
      // Up to kRows / 16 row tiles, and which of them see these keys.
      __syncthreads();
      const Row mine = row_at(a, q, (rb + (tid >> 4) * int(gridDim.y)) * 16 + (tid & 15));
      rows[tid] = mine;
      if (tid == 0) active = 0;
      const uint64_t seen = __ballot(mine.len > k0);
      __syncthreads();
      if (l == 0) {
        unsigned bits = 0;
        for (int i = 0; i < 4; ++i)
          if ((seen >> (16 * i)) & 0xffff) bits |= 1u << (4 * w + i);
        if (bits) atomicOr(&active, bits);
      }
      __syncthreads();
      unsigned todo = __builtin_amdgcn_readfirstlane(active);
      if (!todo) continue;
      constexpr int kN = 4 / kGroups;
      const int row = tid / (64 / kN), part = tid % (64 / kN);
      Raw<kN> raw[kHeld] = {};
      const auto fetch = [&](unsigned bits) {
        const Row r = rows[(bits ? __builtin_ctz(bits) * 16 : 0) + row];
#pragma unroll
        for (int c = 0; c < kHeld; ++c) load_raw<kN, kVec, kFull>(a, r, c, part, raw[c]);
      };
      const auto write = [&](int it) {
        int8_t* to = tiles + (it & 1) * kHalf;
#pragma unroll
        for (int c = 0; c < kHeld; ++c) put_raw<kN>(to + c * kTileBytes, row, part, raw[c]);
      };
      fetch(todo);
      write(0);
      fetch(todo & (todo - 1));
      for (int it = 0; todo; ++it) {
        const int ti = __builtin_ctz(todo);
        todo &= todo - 1;
        __syncthreads();
        if (todo) {
          write(it + 1);
          fetch(todo & (todo - 1));
        }
        const int8_t* tile = tiles + (it & 1) * kHalf;
        // C's words load under the products; asked for before this tile's
        // writes to LDS they gain nothing (128 to 133 us for three prompts in
        // four places).
        uint64_t cw[2][4];
        uint32_t at[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const Row& row = rows[ti * 16 + 4 * g + r];
          at[r] = io.at(row.first, row.len, key);
          cw[0][r] = io.c(a, 0, at[r]);
          cw[1][r] = io.c(a, 1, at[r]);
        }
        v4i acc[2][kDigitPlanes];
        clear(acc);
#pragma unroll
        for (int c = 0; c < kHeld; ++c)
          mul_opened(tile + c * kTileBytes, l, K[c][1], K[c][2], acc);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int c = 0; c < kHeld; ++c) {
          mul_left(tile + c * kTileBytes, 1, l, K[c][0], acc[0]);
          mul_left(tile + c * kTileBytes, 2, l, K[c][0], acc[1]);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const uint64_t z0 = place < 0 ? 0 : from_sums(acc[0], r);
          const uint64_t z1 = place < 0 ? 0 : from_sums(acc[1], r);
          io.put(a, at[r], z0 + cw[0][r], z1 + cw[1][r]);
          if constexpr (kTrunc) __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
  }
}

// Heads of 65 to 128: the digits of both chunks of a key do not fit in a wave's
// registers beside a second wave on the SIMD, so two groups of four waves take
// a chunk each, of the same 64 keys.  Each forms its own chunk of the left
// operand; of a tile's 4 rows a lane, the first group finishes two and the
// second two, with the other's sums through LDS, after the next tile's
// barrier.  32 row tiles of 4 x 2112 keys, 4 cached heads of 128: 380 us; 460
// with both chunks in one wave a SIMD.
template <bool kFull, bool kTrunc, bool kBuffer>
__global__ void __launch_bounds__(512, 2) kv_scores2_pair_kernel(ProductArgs a) {
  constexpr int kRows = 512, kKeys = 64, kHalf = 2 * kTileBytes;
  extern __shared__ __align__(16) int8_t tiles[];
  __shared__ uint64_t sums[2][2][4][256];
  __shared__ Row rows[kRows];
  __shared__ unsigned active;
  const int tid = threadIdx.x, l = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6), half = w >> 2;
  const int g = l >> 4, n = l & 15;
  const int dim = a.pool.dim, in = tid & 255;
  const Elements<kTrunc, kBuffer> io(a);
  const Seq q = seq_at(a, int(blockIdx.x));
  const int row_tiles = (q.rows + 15) / 16;
  for (int64_t first_key = int64_t(blockIdx.z) * kKeys; first_key < q.kv;
       first_key += int64_t(gridDim.z) * kKeys) {
    const int k0 = int(first_key), key = k0 + 16 * (w & 3) + n;
    const int64_t place = place_at(a, q, load_spot(a, q, key));
    v4i K[3][kDigitPlanes];
    int lane_g = g;
    asm volatile("" : "+v"(lane_g));
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      uint64_t v[16];
      load_keys<true, kFull>((k == 0 ? a.pool.e : a.pool.b[k - 1]) + (place < 0 ? 0 : place) +
                                 64 * half,
                             lane_g, dim - 64 * half, v);
      digits_of16(v, K[k]);
    }
    for (int rb = blockIdx.y; rb < row_tiles; rb += gridDim.y * (kRows / 16)) {
      __syncthreads();
      const Row mine = row_at(a, q, (rb + (tid >> 4) * int(gridDim.y)) * 16 + (tid & 15));
      rows[tid] = mine;
      if (tid == 0) active = 0;
      const uint64_t seen = __ballot(mine.len > k0);
      __syncthreads();
      if (l == 0) {
        unsigned bits = 0;
        for (int i = 0; i < 4; ++i)
          if ((seen >> (16 * i)) & 0xffff) bits |= 1u << (4 * w + i);
        if (bits) atomicOr(&active, bits);
      }
      __syncthreads();
      unsigned todo = __builtin_amdgcn_readfirstlane(active);
      if (!todo) continue;
      Raw<4> raw = {};
      const auto fetch = [&](unsigned bits) {
        load_raw<4, true, kFull>(a, rows[(bits ? __builtin_ctz(bits) * 16 : 0) + (in >> 4)], half,
                                 tid & 15, raw);
      };
      const auto write = [&](int it) {
        put_raw<4>(tiles + (it & 1) * kHalf + half * kTileBytes, in >> 4, tid & 15, raw);
      };
      // The tile before: its C words, where they go, this group's sums.
      uint64_t cw[2][2] = {}, own[2][2] = {};
      uint32_t at[2] = {io.at(0, 0, 0), io.at(0, 0, 0)};  // none yet
      const auto finish = [&](int it) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint64_t z0 = own[0][r] + sums[it & 1][half][r][in];
          const uint64_t z1 = own[1][r] + sums[it & 1][half][2 + r][in];
          io.put(a, at[r], (place < 0 ? 0 : z0) + cw[0][r], (place < 0 ? 0 : z1) + cw[1][r]);
          if constexpr (kTrunc) __builtin_amdgcn_sched_barrier(0);
        }
      };
      fetch(todo);
      write(0);
      fetch(todo & (todo - 1));
      int it = 0;
      for (; todo; ++it) {
        const int ti = __builtin_ctz(todo);
        todo &= todo - 1;
        __syncthreads();
        write(it + 1);
        fetch(todo & (todo - 1));
        finish(it - 1);
        __builtin_amdgcn_sched_barrier(0);
        const int8_t* tile = tiles + (it & 1) * kHalf + half * kTileBytes;
        v4i acc[2][kDigitPlanes];
        clear(acc);
        mul_opened(tile, l, K[1], K[2], acc);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const Row& row = rows[ti * 16 + 4 * g + 2 * half + r];
          at[r] = io.at(row.first, row.len, key);
          cw[0][r] = io.c(a, 0, at[r]);
          cw[1][r] = io.c(a, 1, at[r]);
        }
        mul_left(tile, 1, l, K[0], acc[0]);
        mul_left(tile, 2, l, K[0], acc[1]);
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const uint64_t lo = from_sums(acc[p], r), hi = from_sums(acc[p], 2 + r);
            own[p][r] = half ? hi : lo;
            sums[it & 1][half ^ 1][2 * p + r][in] = half ? lo : hi;
          }
      }
      __syncthreads();
      finish(it - 1);
    }
  }
}

// ---- values ----
//
// A workgroup takes 16 rows, 16 columns a wave, and a share of the keys in
// chunks of 64 (the k of the product).  k order: byte j of group g stands for
// key 16 (j % 4) + 4 (j / 4) + g of a chunk, so that the left operand's loads
// and the pages' (one column of 16 keys a lane) both run over neighbouring
// words, and the 16 keys of one j % 4 are in one page when pages hold 16.
//
// The left operand (one row of packed elements a k) passes through LDS, the
// next chunk's written while the present one multiplies; the pages' words go
// to registers, an array's turned into digits and the next chunk's loaded in
// their place, as for the scores.  Two row tiles a wave (the pages' digits used
// twice, one wave a SIMD) took 190 us where this took 159.
struct ValuesArgs {
  ProductArgs p;
  int blocks;        // column blocks
  int8_t* planes;    // many rows: the values' digits (kPlanesBytes), or null
  int room;          // many rows: key tiles a sequence has digits for
  uint64_t* part;    // few rows: two slots of sums a workgroup
  int4* info;        // few rows: [tokens * heads][blocks]
  uint64_t* out[2];  // the values, before a truncation if one follows
};
constexpr int kSlotWords = 2 * 16 * 64;  // both parties' sums of a 16 x 64 tile

// Chunks whose digit sums stay within int32: 2 products of 8 digit pairs of
// at most 2^14 at 64 of k are 2^24 a chunk.
constexpr int kSumChunks = 64;

// One row tile's product with the columns of a workgroup over chunks
// [c0, c1): digit sums of the lane's column and 4 rows into acc, those of
// earlier chunks, if there were too many for int32, into the lane's words of
// `sums` (true).  The pages' first words are on their way while the caller's
// `rows` arrive (a barrier).  kWide: pages of at least 16 keys.
template <int kWaves, bool kWide>
__device__ __forceinline__ bool values_run(const ProductArgs& a, const Seq& q, const Row (&rows)[16],
                                           int8_t (*tiles)[kTileBytes], uint64_t* sums, int c0,
                                           int c1, int col, v4i (&acc)[2][kDigitPlanes]) {
  constexpr int kN = 16 / kWaves;      // words of a row's chunk a thread forms, in pairs
  constexpr int kP = kWide ? 4 : 16;   // page lookups of a chunk: its runs of 16 keys,
                                       // or a lane's own keys
  // The lane's offsets are formed again in each call: kept over the caller's
  // loop they would take registers that the chunk loop does not have.
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));
  const int l = tid & 63, g = l >> 4;
  const int dim = a.pool.dim, shift = a.pool.shift;
  const int row = tid / (64 / kN), part = tid % (64 / kN);
  bool flushed = false;
  clear(acc);
  const uint32_t lane = 8 * uint32_t((kWide ? g * dim : 0) + (col < dim ? col : 0));
  const int32_t* table = a.b.table + int64_t(q.s) * a.b.max_pages;
  const auto page_of = [&](int c, int j) -> int {
    const int at = j >> shift;
    const bool in = c < c1 && j < q.kv && at < a.b.max_pages;
    const int page = table[in ? at : 0];
    return in ? page : -1;
  };
  const auto key_of = [&](int c, int i) {  // of lookup i
    return c * kKeyTile + (kWide ? 16 * i : 16 * (i & 3) + 4 * (i >> 2) + g);
  };
  const auto lookup = [&](int c, int (&pg)[kP]) {
#pragma unroll
    for (int i = 0; i < kP; ++i) pg[i] = page_of(c, key_of(c, i));
  };
  // First word of each lookup's keys (the pool's first where there is no
  // page) and, kWide, which of the four runs have a page.
  int64_t base[kP];
  unsigned held = 0;
  const auto place = [&](int c, const int (&pg)[kP]) {
    held = 0;
#pragma unroll
    for (int i = 0; i < kP; ++i) {
      const int at = kWide ? __builtin_amdgcn_readfirstlane(pg[i]) : pg[i];
      const bool ok = unsigned(at) < unsigned(a.pool.pages);
      const int64_t head = int64_t(ok ? at : 0) * a.pool.heads + (ok ? q.hk : 0);
      const int in = ok ? key_of(c, i) & ((1 << shift) - 1) : 0;
      base[i] = ((head << shift) + in) * dim;
      held |= ok ? 1u << i : 0u;
    }
  };
  uint64_t raw[3][16];
  const auto issue = [&](int k) {
    const uint64_t* src = k == 0 ? a.pool.b[0] : k == 1 ? a.pool.b[1] : a.pool.e;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const char* at = reinterpret_cast<const char*>(src + base[kWide ? i & 3 : i]);
      raw[k][i] = *reinterpret_cast<const uint64_t*>(
          at + (lane + (kWide ? uint32_t(32 * (i >> 2) * dim) : 0u)));
    }
  };
  // The left operand's words of pair h: keys of bytes j and j + 1, j = kN m +
  // 2 h.  Past the row's end and for keys without a page the row's first
  // element, which `write` drops.
  Row mine;
  const auto key0 = [&](int c, int h) {
    const int j = kN * (part >> 2) + 2 * h;
    return c * kKeyTile + 16 * (j & 3) + 4 * (j >> 2) + (part & 3);
  };
  const auto inside = [&](int c, int h, int k) {
    const int key = key0(c, h) + 16 * k;
    if constexpr (kWide) {
      const int run = (kN == 4 ? 2 * h : (part >> 1) & 2) + k;
      return key < mine.len && ((held >> run) & 1);
    } else {
      return key < mine.len && unsigned(page_of(c, key)) < unsigned(a.pool.pages);
    }
  };
  Raw<2> left[kN / 2];
  const auto fetch = [&](int c, int h) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int key = key0(c, h) + 16 * k;
      const int64_t o = int64_t(mine.first) + (key < mine.len ? key : 0);
      left[h].x0[k] = a.x[0][o];
      left[h].x1[k] = a.x[1][o];
      left[h].a0[k] = a.a[0][o];
      left[h].a1[k] = a.a[1][o];
    }
  };
  const auto write = [&](int c, int h) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (inside(c, h, k)) continue;
      left[h].x0[k] = left[h].x1[k] = left[h].a0[k] = left[h].a1[k] = 0;
    }
    put_left<2>(tiles[c & 1], row, part & 3, kN * (part >> 2) + 2 * h, left[h]);
  };
  int pg[kP];
  lookup(c0, pg);
  place(c0, pg);
  lookup(c0 + 1, pg);
#pragma unroll
  for (int k = 0; k < 3; ++k) issue(k);
  __syncthreads();
  const int chunks = (longest(rows) + kKeyTile - 1) / kKeyTile;
  c1 = c1 < chunks ? c1 : chunks;
  if (c0 >= c1) return flushed;
  mine = rows[row];
#pragma unroll
  for (int h = 0; h < kN / 2; ++h) fetch(c0, h);
#pragma unroll
  for (int h = 0; h < kN / 2; ++h) write(c0, h);
  for (int c = c0; c < c1; ++c) {
    const int8_t* tile = tiles[c & 1];
    __syncthreads();
    place(c + 1, pg);
    lookup(c + 2, pg);
    if constexpr (kN == 4) fetch(c + 1, 1);
    // An array's loads leave when its digits have been used: into their
    // registers, with the other two arrays' still under way.
    v4i y[kDigitPlanes];
    digits_of16(raw[0], y);
    mul_left(tile, 0, l, y, acc[0]);
    __builtin_amdgcn_sched_barrier(0);
    issue(0);
    fetch(c + 1, 0);
    digits_of16(raw[1], y);
    mul_left(tile, 0, l, y, acc[1]);
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (kN == 4) write(c + 1, 1);
    issue(1);
    digits_of16(raw[2], y);
    mul_left(tile, 1, l, y, acc[0]);
    mul_left(tile, 2, l, y, acc[1]);
    __builtin_amdgcn_sched_barrier(0);
    write(c + 1, 0);
    issue(2);
    if ((c - c0) % kSumChunks == kSumChunks - 1) {
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          uint64_t v = from_sums(acc[p], r);
          if (flushed) v += sums[4 * p + r];
          sums[4 * p + r] = v;
        }
      flushed = true;
      clear(acc);
    }
  }
  return flushed;
}

// The values' digits, formed once for all row tiles: 64 keys of 16 columns are
// the planes of b_0, b_1 and E (plane i of array k at (8 k + i) KB), 16 bytes a
// lane in the lanes' order.  Keys without a page are zeros.  k order here:
// byte j of group g stands for key 16 (j / 4) + 4 g + j % 4, so that a thread's
// left words, bytes of one group, are neighbours.
constexpr int kPlanesBytes = 3 * kDigitPlanes * 1024;
__device__ __forceinline__ int8_t* planes_at(const ValuesArgs& va, int z, int tile, int c16) {
  const int per = (va.p.pool.dim + 15) / 16;
  return va.planes + ((int64_t(z) * va.room + tile) * per + c16) * kPlanesBytes;
}

// A workgroup an array and 64 x 64 of its values: short chains of loads (lengths,
// page numbers, words), and many of them.
__global__ void __launch_bounds__(256) kv_values2_digits_kernel(ValuesArgs va) {
  const ProductArgs& a = va.p;
  const int l = threadIdx.x & 63, g = l >> 4, n = l & 15;
  const int k = int(blockIdx.y) % 3;
  const int c16 = 4 * (int(blockIdx.y) / 3) +
                  __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6);
  const int dim = a.pool.dim;
  if (16 * c16 >= dim) return;
  const Seq q = seq_at(a, int(blockIdx.x));
  const int tiles = tiles_of(q.kv);
  if (q.rows == 0 || q.kv <= 0 || tiles > va.room) return;
  const int col = 16 * c16 + n < dim ? 16 * c16 + n : 0;
  const uint64_t* src = (k == 2 ? a.pool.e : a.pool.b[k]) + col;
  for (int t = blockIdx.z; t < tiles; t += gridDim.z) {
    Spot spot[16];
#pragma unroll
    for (int i = 0; i < 16; ++i)
      spot[i] = load_spot(a, q, t * kKeyTile + 16 * (i >> 2) + 4 * g + (i & 3));
    uint64_t v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int64_t at = place_at(a, q, spot[i]);
      v[i] = src[at < 0 ? 0 : at];
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = place_at(a, q, spot[i]) < 0 ? 0 : v[i];
    v4i y[kDigitPlanes];
    digits_of16(v, y);
    int8_t* to = planes_at(va, int(blockIdx.x), t, c16) + 8192 * k + 16 * l;
#pragma unroll
    for (int i = 0; i < kDigitPlanes; ++i) *reinterpret_cast<v4i*>(to + i * 1024) = y[i];
  }
}

// values_run over digits that are there: from `from` (the wave's planes of the
// first chunk, `step` bytes a chunk).  Nothing but the left operand is formed
// here, 2.7 vector instructions for each matrix instruction instead of 5.2.
// The place of the left words' loads and LDS writes among the products does
// not matter (137 to 138 us for three prompts in five orders).
template <int kWaves>
__device__ __forceinline__ bool planes_run(const ProductArgs& a, const Row (&rows)[16],
                                           int8_t (*tiles)[kTileBytes], uint64_t* sums,
                                           const int8_t* from, int step, int c1,
                                           v4i (&acc)[2][kDigitPlanes]) {
  constexpr int kN = 16 / kWaves;
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));
  const int l = tid & 63;
  const uint32_t lane = 16 * uint32_t(l);
  const int row = tid / (64 / kN), part = tid % (64 / kN);
  bool flushed = false;
  clear(acc);
  v4i y[3][kDigitPlanes];
  const auto issue = [&](int k) {
#pragma unroll
    for (int i = 0; i < kDigitPlanes; ++i)
      y[k][i] = *reinterpret_cast<const v4i*>(from + (8 * k + i) * 1024 + lane);
  };
#pragma unroll
  for (int k = 0; k < 3; ++k) issue(k);
  __syncthreads();
  const int chunks = (longest(rows) + kKeyTile - 1) / kKeyTile;
  c1 = c1 < chunks ? c1 : chunks;
  if (c1 <= 0) return flushed;
  // The left operand's words, kN neighbours a thread.  Chunks that all rows
  // reach past need no bounds: two words a load, 8-byte aligned.
  typedef unsigned long long Two __attribute__((ext_vector_type(2), aligned(8)));
  const Row mine = rows[row];
  const int within = shortest(rows);
  const int first = kN == 4 ? 4 * part : 16 * (part >> 3) + 4 * (part & 3) + 2 * ((part >> 2) & 1);
  const uint64_t* at[4];
#pragma unroll
  for (int k = 0; k < 4; ++k)
    at[k] = (k < 2 ? a.x[k] : a.a[k - 2]) + int64_t(mine.first) + first;
  Raw<kN> left;
  const auto fetch = [&](int c) {
    if ((c + 1) * kKeyTile <= within) {
#pragma unroll
      for (int e = 0; e < kN; e += 2) {
        const auto two = [&](const uint64_t* from, uint64_t (&v)[kN]) {
          const Two w = *reinterpret_cast<const Two*>(from + e);
          v[e] = w[0];
          v[e + 1] = w[1];
        };
        two(at[0], left.x0);
        two(at[1], left.x1);
        two(at[2], left.a0);
        two(at[3], left.a1);
      }
    } else {
#pragma unroll
      for (int e = 0; e < kN; ++e) {
        const int key = c * kKeyTile + first + e;
        const int64_t o = int64_t(mine.first) + (key < mine.len ? key : 0);
        left.x0[e] = a.x[0][o];
        left.x1[e] = a.x[1][o];
        left.a0[e] = a.a[0][o];
        left.a1[e] = a.a[1][o];
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) at[k] += kKeyTile;
  };
  const auto write = [&](int c) {
    if ((c + 1) * kKeyTile > within) {
#pragma unroll
      for (int e = 0; e < kN; ++e) {
        if (c * kKeyTile + first + e < mine.len) continue;
        left.x0[e] = left.x1[e] = left.a0[e] = left.a1[e] = 0;
      }
    }
    put_left<kN>(tiles[c & 1], row, part & 3, kN * (part >> 2), left);
  };
  fetch(0);
  write(0);
  fetch(1);
  for (int c = 0; c < c1; ++c) {
    const int8_t* tile = tiles[c & 1];
    __syncthreads();
    if (c + 1 < c1) from += step;
    mul_left(tile, 0, l, y[0], acc[0]);
    __builtin_amdgcn_sched_barrier(0);
    issue(0);
    mul_left(tile, 0, l, y[1], acc[1]);
    __builtin_amdgcn_sched_barrier(0);
    issue(1);
    mul_left(tile, 1, l, y[2], acc[0]);
    write(c + 1);
    fetch(c + 2);
    mul_left(tile, 2, l, y[2], acc[1]);
    __builtin_amdgcn_sched_barrier(0);
    issue(2);
    if (c % kSumChunks == kSumChunks - 1) {
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          uint64_t v = from_sums(acc[p], r);
          if (flushed) v += sums[4 * p + r];
          sums[4 * p + r] = v;
        }
      flushed = true;
      clear(acc);
    }
  }
  return flushed;
}

// Many rows: a workgroup a row tile, cached head and column block.  Three
// prompts (1024, 517 after 200, 33 tokens; 12 heads of 64 on 4 cached ones):
// 123 us and 9 for the digits; 342 MB needed, 419 moved; the matrix cores are
// busy for 31% of it.  The longest item is 16 chunks one after another; without
// the left words' and the digits' traffic a chunk takes six tenths of its time.
template <int kWaves, bool kWide, bool kPlanes>
__global__ void __launch_bounds__(64 * kWaves, kWide ? 2 : 1) kv_values2_kernel(ValuesArgs va) {
  const ProductArgs& a = va.p;
  __shared__ __align__(16) int8_t tiles[2][kTileBytes];
  __shared__ uint64_t sums[64 * kWaves][8];
  __shared__ Row rows[16];
  const int tid = threadIdx.x, l = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = l >> 4, n = l & 15;
  const int dim = a.pool.dim;
  const int col = int(blockIdx.y) * 16 * kWaves + 16 * w + n;
  const Seq q = seq_at(a, int(blockIdx.x));
  // The last row tiles first: with causal rows they are the longest.
  for (int m = (q.rows + 15) / 16 - 1 - int(blockIdx.z); m >= 0; m -= int(gridDim.z)) {
    __syncthreads();
    if (tid < 16) rows[tid] = row_at(a, q, 16 * m + tid);
    v4i acc[2][kDigitPlanes];
    bool flushed;
    if (kPlanes && tiles_of(q.kv) <= va.room) {
      const int per = (dim + 15) / 16;
      const int c16 = min(int(blockIdx.y) * kWaves + w, per - 1);
      flushed = planes_run<kWaves>(a, rows, tiles, sums[tid],
                                   planes_at(va, int(blockIdx.x), 0, c16),
                                   per * kPlanesBytes, tiles_of(q.kv), acc);
    } else {
      flushed = values_run<kWaves, kWide>(a, q, rows, tiles, sums[tid], 0, tiles_of(q.kv), col,
                                          acc);
    }
    if (col >= dim) continue;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const Row at = rows[4 * g + r];
      if (at.t < 0) continue;
      const int64_t o = (int64_t(at.t) * a.heads + at.h) * dim + col;
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        uint64_t v = from_sums(acc[p], r) + a.c[p][o];
        if (flushed) v += sums[tid][4 * p + r];
        va.out[p][o] = v;
      }
    }
  }
}

// Few rows: even shares of the keys' units.  An item that lies within one
// workgroup's share is finished there; the sums of one that does not go to
// the workspace, where slot 2 w holds what workgroup w has of an item that
// began before its share, slot 2 w + 1 of one that goes on after it.  For
// each row and column block `info` keeps the first and last workgroup of its
// item and its row in the tile, from which the join finds the slots.  Sums mod
// 2^64 are the same in any order.  One sequence of 65536 keys, 2 cached heads
// of 128, 4 queries each: 92 us, 420 MB at 4.6 TB/s, the join 5 of them; 16
// sequences of up to 4096 keys 184 us (4.6 TB/s); 300 keys 14 us, 4 of them the
// join's launch.
constexpr int kFewCols = 64;

template <bool kWide>
__global__ void __launch_bounds__(256, kWide ? 2 : 1) kv_values2_few_kernel(ValuesArgs va) {
  const ProductArgs& a = va.p;
  __shared__ __align__(16) int8_t tiles[2][kTileBytes];
  __shared__ uint64_t sums[256][8];
  __shared__ Row rows[16];
  __shared__ int64_t pre[260];
  const int dim = a.pool.dim, blocks = va.blocks;
  Share sh = share_of(a, blocks, pre);
  while (sh.unit < sh.end) {
    const Piece pc = piece_at(a, blocks, pre, sh);
    if (pc.count == 0) continue;
    // As in values_run: offsets formed for each piece.
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const int g = (tid >> 4) & 3, in = 16 * (tid >> 6) + (tid & 15);
    const int col = pc.block * kFewCols + in;
    __syncthreads();
    if (tid < 16) {
      const Row r = row_at(a, pc.q, 16 * pc.rt + tid);
      rows[tid] = r;
      if (pc.tile == 0 && r.t >= 0)
        va.info[(int64_t(r.t) * a.heads + r.h) * blocks + pc.block] =
            make_int4(pc.first, pc.last, tid, 0);
    }
    v4i acc[2][kDigitPlanes];
    const bool flushed = values_run<4, kWide>(a, pc.q, rows, tiles, sums[tid], pc.tile,
                                              pc.tile + pc.count, col, acc);
    const bool whole = pc.count == pc.tiles;
    uint64_t* slot = va.part + (2 * int64_t(blockIdx.x) + (pc.tile == 0 ? 1 : 0)) * kSlotWords;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const Row at = rows[4 * g + r];
      if (at.t < 0 || col >= dim) continue;
      const int64_t o = (int64_t(at.t) * a.heads + at.h) * dim + col;
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        uint64_t v = from_sums(acc[p], r);
        if (flushed) v += sums[tid][4 * p + r];
        if (whole)
          va.out[p][o] = v + a.c[p][o];
        else
          slot[(p * 16 + 4 * g + r) * kFewCols + in] = v;
      }
    }
  }
}

// Joins the items that several workgroups have sums of, and truncates: kOut
// columns of one row a workgroup, the other lanes over the slots.
template <bool kTrunc, int kOut>
__global__ void __launch_bounds__(256) kv_values2_join_kernel(ValuesArgs va) {
  const ProductArgs& a = va.p;
  constexpr int kLanes = 256 / kOut;
  __shared__ uint64_t s[2][kLanes][kOut];
  const int dim = a.pool.dim;
  const int u = threadIdx.x % kOut, lane = threadIdx.x / kOut;
  const Put<kTrunc> put(a);
  const int64_t all = int64_t(a.b.tokens) * a.heads;
  for (int64_t row = blockIdx.x; row < all; row += gridDim.x) {
    if (seq_of(a.b, int(row / a.heads)) < 0) continue;
    const int col = int(blockIdx.y) * kOut + u;
    const int64_t o = row * dim + col;
    const int4 at = va.info ? va.info[row * va.blocks + int(blockIdx.y) * kOut / kFewCols]
                            : make_int4(0, 0, 0, 0);
    if (at.y > at.x) {
      const int64_t in = at.z * kFewCols + col % kFewCols;
      uint64_t z0 = 0, z1 = 0;
#pragma unroll 4
      for (int w = at.x + lane; w <= at.y; w += kLanes) {
        const uint64_t* slot = va.part + (2 * int64_t(w) + (w == at.x ? 1 : 0)) * kSlotWords + in;
        z0 += slot[0];
        z1 += slot[16 * kFewCols];
      }
      __syncthreads();  // the sums of the row before have been used
      s[0][lane][u] = z0;
      s[1][lane][u] = z1;
      __syncthreads();
      if (lane || col >= dim) continue;
      z0 = a.c[0][o];
      z1 = a.c[1][o];
      for (int k = 0; k < kLanes; ++k) {
        z0 += s[0][k][u];
        z1 += s[1][k][u];
      }
      put(a, o, z0, z1);
    } else if (kTrunc && lane == 0 && col < dim) {
      put(a, o, va.out[0][o], va.out[1][o]);
    }
  }
}

int product_args(const sufhip_kv_product2_args* args, bool values, const char* what,
                 ProductArgs* out, bool* empty) {
  if (!args) return kv_fail(what, "null args");
  const sufhip_kv_product2_args& g = *args;
  ProductArgs a{};
  if (int rc = kv_batch_of(g.batch, what, &a.b)) return rc;
  if (int rc = kv_pool_of(g.pool, what, &a.pool)) return rc;
  if (g.pool.pages < 1) return kv_fail(what, "the pool has no pages");
  if (g.heads < 1 || g.heads % g.pool.kv_heads)
    return kv_fail(what, "heads must be a multiple of the pool's kv_heads");
  // Two chunks past the last key are still numbered in 32 bits.
  if (g.n > (size_t(1) << 31) - 256)
    return kv_fail(what, "at most 2^31 - 256 packed elements");
  const size_t rows = size_t(a.b.tokens) * size_t(g.heads);
  if (rows > (1u << 30) || size_t(a.b.seqs) * size_t(a.pool.heads) > (1u << 22))
    return kv_fail(what, "at most 2^30 rows, and 2^22 sequences times cached heads");
  *empty = a.b.seqs == 0 || rows == 0 || (!values && g.n == 0);
  if (*empty) return SUFHIP_OK;
  const size_t n_out = values ? rows * size_t(g.pool.dim) : g.n;
  if (int rc = make_epi(g.trunc, n_out, what, &a.epi)) return rc;
  if (a.epi.add[0]) return kv_fail(what, "the truncation takes no addend");
  if (!g.x.p[0] || !g.x.p[1] || !g.a[0] || !g.a[1] || !g.c[0] || !g.c[1] || !g.d_row_offsets) {
    // Without packed elements the values' left operand is never read.
    if (!(values && g.n == 0 && g.c[0] && g.c[1] && g.d_row_offsets))
      return kv_fail(what, "null operand");
  }
  if (!a.epi.on && (!g.out[0] || !g.out[1]))
    return kv_fail(what, "outputs (or a truncation) needed");
  if (!values && (g.x.token_stride < 0 || g.x.head_stride < 0))
    return kv_fail(what, "strides must be >= 0");
  a.heads = g.heads;
  a.group = g.heads / g.pool.kv_heads;
  a.by_group = fast_div(uint32_t(a.group));
  a.xts = g.x.token_stride;
  a.xhs = g.x.head_stride;
  a.offsets = g.d_row_offsets;
  a.n = int64_t(g.n);
  a.mask = g.mask;
  for (int p = 0; p < 2; ++p) {
    a.x[p] = g.x.p[p];
    a.a[p] = g.a[p];
    a.c[p] = g.c[p];
    a.out[p] = g.out[p];
  }
  // A lookup that is not wanted reads a sequence's first page number; without
  // pages a word that is there, and drops it.
  if (a.b.max_pages == 0) a.b.table = a.b.cu;
  *out = a;
  return SUFHIP_OK;
}

}  // namespace
}  // namespace sufhip

using namespace sufhip;

namespace sufhip {
namespace {

bool at16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
unsigned clip(int64_t v, int64_t most) { return unsigned(v < 1 ? 1 : (v < most ? v : most)); }
// A product of counts, or the largest number: bounds of a launch may be any.
int64_t times(int64_t a, int64_t b) {
  int64_t v;
  return __builtin_mul_overflow(a, b, &v) ? INT64_MAX : v;
}
// Row tiles of a sequence with the bounds' most new tokens (no more than the
// batch has).
int64_t row_tiles_of(const sufhip_kv_batch& b, int group) {
  const int64_t rows = times(b.max_new < b.tokens ? b.max_new : b.tokens, group);
  return rows / 16 + (rows % 16 != 0);
}

// Compute units of the current device (256 without one: sizes asked for on a
// host alone); asked of the runtime once a device.
int cu_total() {
  static std::atomic<int> known[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0) {
    (void)hipGetLastError();
    return 256;
  }
  if (dev < 64)
    if (const int n = known[dev].load(std::memory_order_relaxed)) return n;
  int cus = 0;
  if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess ||
      cus < 1) {
    (void)hipGetLastError();
    return 256;
  }
  if (dev < 64) known[dev].store(cus, std::memory_order_relaxed);
  return cus;
}

// Dynamic LDS past the 64 KB that a kernel may take unasked.
template <typename F>
int allow_lds(F* f, size_t lds) {
  if (lds > 64 * 1024)
    SUFHIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(f),
                                     hipFuncAttributeMaxDynamicSharedMemorySize, int(lds)),
                 "dynamic LDS");
  return SUFHIP_OK;
}

template <bool kVec, bool kFull, bool kTrunc>
int launch_scores_few(const ProductArgs& a, const dim3& grid, int chunks, hipStream_t st) {
  const size_t lds = size_t(chunks) * kTileBytes;
  if (int rc = allow_lds(kv_scores2_few_kernel<kVec, kFull, kTrunc>, lds)) return rc;
  hipLaunchKernelGGL((kv_scores2_few_kernel<kVec, kFull, kTrunc>), grid, dim3(256), lds, st, a,
                     chunks);
  return check_launch("kv_scores2_few_kernel");
}

template <int kHeld, int kGroups, bool kVec, bool kFull, bool kTrunc, bool kBuffer>
int launch_scores_many(const ProductArgs& a, const dim3& grid, hipStream_t st) {
  const size_t lds = 2 * size_t(kHeld) * kTileBytes;
  if (int rc = allow_lds(kv_scores2_kernel<kHeld, kGroups, kVec, kFull, kTrunc, kBuffer>, lds))
    return rc;
  hipLaunchKernelGGL((kv_scores2_kernel<kHeld, kGroups, kVec, kFull, kTrunc, kBuffer>), grid,
                     dim3(256 * kGroups), lds, st, a);
  return check_launch("kv_scores2_kernel");
}

template <bool kFull, bool kTrunc, bool kBuffer>
int launch_scores_pair(const ProductArgs& a, const dim3& grid, hipStream_t st) {
  const size_t lds = 4 * size_t(kTileBytes);
  if (int rc = allow_lds(kv_scores2_pair_kernel<kFull, kTrunc, kBuffer>, lds)) return rc;
  hipLaunchKernelGGL((kv_scores2_pair_kernel<kFull, kTrunc, kBuffer>), grid, dim3(512), lds, st, a);
  return check_launch("kv_scores2_pair_kernel");
}

// Many rows, heads of up to 128.
template <bool kVec, bool kFull, bool kTrunc, bool kBuffer>
int launch_scores_many(const ProductArgs& a, const dim3& grid, hipStream_t st) {
  if (a.pool.dim <= 64)
    return launch_scores_many<1, kVec ? 2 : 1, kVec, kFull, kTrunc, kBuffer>(a, grid, st);
  if constexpr (kVec)
    return launch_scores_pair<kFull, kTrunc, kBuffer>(a, grid, st);
  else
    return launch_scores_many<2, 1, kVec, kFull, kTrunc, kBuffer>(a, grid, st);
}

template <bool kVec, bool kFull, bool kTrunc>
int launch_scores(const ProductArgs& a, const sufhip_kv_batch& b, hipStream_t st) {
  const int chunks = (a.pool.dim + 63) / 64;
  const int64_t row_tiles = row_tiles_of(b, a.group);
  const int64_t zs = int64_t(a.b.seqs) * a.pool.heads;
  const int cus = cu_total();
  // One row tile a sequence streams the keys; with more, keys held as digits
  // are used for all of them (4 cached heads of 64, 8 x 4 rows over 4 x 2048
  // keys, two row tiles: 42 us streamed, 29 held; 24 row tiles: 284 and 155).
  // Heads past 128 do not fit in registers.
  if (row_tiles <= 1 || chunks > 2) {
    const int64_t tiles =
        b.max_keys > kKeyTile ? (int64_t(b.max_keys) + kKeyTile - 1) / kKeyTile : 1;
    const dim3 grid(
        clip(times(times(zs, row_tiles < 1 ? 1 : row_tiles), tiles + 1), 2 * int64_t(cus)));
    return launch_scores_few<kVec, kFull, kTrunc>(a, grid, chunks, st);
  }
  constexpr int kGroups = kVec ? 2 : 1;  // of one chunk's kernel
  const int groups = chunks == 1 ? kGroups : 1;
  const int64_t key_tiles = (int64_t(b.max_keys) + 64 * groups - 1) / (64 * groups);
  // Row tiles are spread over workgroups until four of them share a CU (three
  // prompts: 134 us then, 145 with eight, 175 with sixteen).
  const int64_t want = (4 * int64_t(cus) + key_tiles * zs) / (key_tiles * zs + 1);
  const dim3 grid(unsigned(zs), clip(want < row_tiles ? want : row_tiles, 65535),
                  clip(key_tiles, 65535));
  return a.n <= kBufferMost ? launch_scores_many<kVec, kFull, kTrunc, true>(a, grid, st)
                             : launch_scores_many<kVec, kFull, kTrunc, false>(a, grid, st);
}

template <bool kVec, bool kFull>
int launch_scores(const ProductArgs& a, const sufhip_kv_batch& b, hipStream_t st) {
  return a.epi.on ? launch_scores<kVec, kFull, true>(a, b, st)
                  : launch_scores<kVec, kFull, false>(a, b, st);
}

// How a values call is laid out: even shares of the keys over two workgroups a
// CU (few), or a workgroup an item (row tile, cached head, column block).  An
// item is one chain over its keys, so even shares win while items are fewer
// than half the CUs, and, whatever their number, with one row tile a sequence,
// where lengths differ most; from there on the items fill the chip and need no
// join, as do short chains.  Us, even shares / items (4 cached heads of 64, new
// tokens x 8 heads; keys in all):
//   4 x 2048 keys:  32 items 41 / 131    96: 84 / 140   192: 139 / 145   384: 257 / 222
//   1 x 300:         8 items 15 / 25     48: 24 / 32     96: 32 / 32
//   8 x 100:        64 items 19 / 17    192: 31 / 18    768: 66 / 50
// Items form the values' digits once for all of a sequence's row tiles
// (planes), if those are several and the chains pay for the launch; in each
// item / once:
//   4 x 2048 keys:  heads of 64, 12 row tiles 144 / 119, 24: 221 / 192
//                   heads of 128, 6 row tiles 201 / 153, 24: 395 / 313
//   8 x 100 keys:   heads of 64, 4 row tiles 18 / 23, 24: 51 / 52
// The digits take 24 bytes a value of max_keys for every sequence: not more
// than twice what the pool itself holds nor 2 GiB (beside caches of tens of
// them), or they are formed in each item.
constexpr int kFewMinTiles = 4;
constexpr int kPlanesMinRows = 4;
constexpr int64_t kPlanesMost = int64_t(1) << 31;
struct ValuesPlan {
  bool wide, few;
  int waves, blocks;
  int64_t row_tiles, zs, groups, room;
  size_t part_bytes, info_bytes, planes_bytes;
};
ValuesPlan plan_values(const sufhip_kv_batch& b, const sufhip_kv_pool& p, int heads) {
  ValuesPlan v{};
  v.wide = p.page_tokens >= 16;
  v.row_tiles = row_tiles_of(b, heads / p.kv_heads);
  if (v.row_tiles < 1) v.row_tiles = 1;
  v.zs = int64_t(b.seqs) * p.kv_heads;
  const int64_t tiles = b.max_keys > kKeyTile ? (int64_t(b.max_keys) + kKeyTile - 1) / kKeyTile : 1;
  const int64_t items = times(times(v.zs, v.row_tiles), (p.dim + 63) / 64);
  v.few = tiles >= kFewMinTiles && (v.row_tiles == 1 || items <= cu_total() / 2);
  v.waves = v.few || !v.wide || p.dim <= 64 ? 4 : 8;
  v.blocks = (p.dim + 16 * v.waves - 1) / (16 * v.waves);
  if (v.few) {
    v.groups = clip(times(times(times(v.zs, v.row_tiles), v.blocks), tiles + 1), 2 * cu_total());
    v.part_bytes = size_t(v.groups) * 2 * kSlotWords * 8;
    v.info_bytes = size_t(b.tokens) * size_t(heads) * size_t(v.blocks) * 16;
  } else if (v.row_tiles >= kPlanesMinRows && tiles >= kFewMinTiles &&
             times(times(b.seqs, tiles), kKeyTile) <= 2 * int64_t(p.pages) * p.page_tokens &&
             times(times(v.zs, tiles), (p.dim + 15) / 16) <= kPlanesMost / kPlanesBytes) {
    v.room = tiles;
    v.planes_bytes = size_t(v.zs) * size_t(tiles) * size_t((p.dim + 15) / 16) * kPlanesBytes;
  }
  return v;
}

template <int kWaves, bool kWide>
void launch_values(const ValuesArgs& va, const dim3& grid, hipStream_t st) {
  if (va.planes)
    hipLaunchKernelGGL((kv_values2_kernel<kWaves, kWide, true>), grid, dim3(64 * kWaves), 0, st,
                       va);
  else
    hipLaunchKernelGGL((kv_values2_kernel<kWaves, kWide, false>), grid, dim3(64 * kWaves), 0, st,
                       va);
}
void launch_values(const ValuesArgs& va, const ValuesPlan& v, const dim3& grid, hipStream_t st) {
  if (!v.wide)
    launch_values<4, false>(va, grid, st);
  else if (v.waves == 4)
    launch_values<4, true>(va, grid, st);
  else
    launch_values<8, true>(va, grid, st);
}

template <int kOut>
void launch_join(const ValuesArgs& va, hipStream_t st) {
  const dim3 grid(clip(int64_t(va.p.b.tokens) * va.p.heads, 1 << 20),
                  unsigned((va.p.pool.dim + kOut - 1) / kOut));
  if (va.p.epi.on)
    hipLaunchKernelGGL((kv_values2_join_kernel<true, kOut>), grid, dim3(256), 0, st, va);
  else
    hipLaunchKernelGGL((kv_values2_join_kernel<false, kOut>), grid, dim3(256), 0, st, va);
}

}  // namespace
}  // namespace sufhip

extern "C" {

int sufhip_kv_scores2(const sufhip_kv_product2_args* args, void* stream) {
  ProductArgs a{};
  bool empty = false;
  if (int rc = product_args(args, false, "sufhip_kv_scores2", &a, &empty)) return rc;
  if (empty) return SUFHIP_OK;
  const bool vec = (a.pool.dim & 1) == 0 && at16(a.pool.e) && at16(a.pool.b[0]) &&
                   at16(a.pool.b[1]) && at16(a.x[0]) && at16(a.x[1]) && at16(a.a[0]) &&
                   at16(a.a[1]) && (a.xts & 1) == 0 && (a.xhs & 1) == 0;
  const hipStream_t st = as_stream(stream);
  if (!vec) return launch_scores<false, false>(a, args->batch, st);
  return a.pool.dim % 64 ? launch_scores<true, false>(a, args->batch, st)
                         : launch_scores<true, true>(a, args->batch, st);
}

size_t sufhip_kv_values2_work_bytes(const sufhip_kv_batch* batch, const sufhip_kv_pool* pool,
                                    int heads) {
  if (!batch || !pool || pool->kv_heads < 1 || pool->dim < 1 || heads < 1 || batch->tokens < 1 ||
      batch->seqs < 1 || heads % pool->kv_heads)
    return 0;
  const ValuesPlan v = plan_values(*batch, *pool, heads);
  return v.part_bytes + v.info_bytes + v.planes_bytes;
}

int sufhip_kv_values2(const sufhip_kv_product2_args* args, void* stream) {
  ValuesArgs va{};
  bool empty = false;
  if (int rc = product_args(args, true, "sufhip_kv_values2", &va.p, &empty)) return rc;
  if (empty) return SUFHIP_OK;
  const ValuesPlan v = plan_values(args->batch, args->pool, args->heads);
  const hipStream_t st = as_stream(stream);
  va.blocks = v.blocks;
  for (int p = 0; p < 2; ++p) va.out[p] = va.p.epi.on ? va.p.epi.y[p] : va.p.out[p];
  const size_t need = v.part_bytes + v.info_bytes + v.planes_bytes;
  SUFHIP_REQUIRE(need == 0 || (args->d_work && at16(args->d_work) && args->work_bytes >= need),
                 "sufhip_kv_values2: d_work smaller than its work bytes, or not 16-byte aligned");
  if (v.few) {
    va.part = static_cast<uint64_t*>(args->d_work);
    va.info = reinterpret_cast<int4*>(static_cast<char*>(args->d_work) + v.part_bytes);
    const dim3 grid{unsigned(v.groups)};
    if (v.wide)
      hipLaunchKernelGGL(kv_values2_few_kernel<true>, grid, dim3(256), 0, st, va);
    else
      hipLaunchKernelGGL(kv_values2_few_kernel<false>, grid, dim3(256), 0, st, va);
    if (int rc = check_launch("kv_values2_few_kernel")) return rc;
    // Slots of an item: over four, more lanes take them.
    if ((v.groups - 1) / 4 >= times(times(v.zs, v.row_tiles), v.blocks))
      launch_join<16>(va, st);
    else
      launch_join<64>(va, st);
    return check_launch("kv_values2_join_kernel");
  }
  if (v.planes_bytes) {
    va.planes = static_cast<int8_t*>(args->d_work);
    va.room = int(v.room);
    hipLaunchKernelGGL(kv_values2_digits_kernel,
                       dim3(unsigned(v.zs), unsigned(3 * ((va.p.pool.dim + 63) / 64)),
                            clip(v.room, 65535)),
                       dim3(256), 0, st, va);
    if (int rc = check_launch("kv_values2_digits_kernel")) return rc;
  }
  const dim3 grid(unsigned(v.zs), unsigned(v.blocks), clip(v.row_tiles, 65535));
  launch_values(va, v, grid, st);
  if (int rc = check_launch("kv_values2_kernel")) return rc;
  if (!va.p.epi.on) return SUFHIP_OK;
  launch_join<64>(va, st);
  return check_launch("kv_values2_join_kernel");
}

}  // extern "C"
