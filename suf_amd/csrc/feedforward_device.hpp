// Shared by the kernels of a decoder's feed-forward parts (rmsnorm.hip,
// linear.hip, expert_mix.hip): rows with strides, their digits, gates folded
// into an epilogue, and the host's checks.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <string>

#include "chain_device.hpp"
#include "digit_planes.hpp"
#include "suf_hip.h"
#include "sufhip_internal.hpp"
#include "trunc_device.hpp"

namespace sufhip {

struct Mat2 {
  const uint64_t* p[2];
  int64_t stride;
};

constexpr int kMaxRows = 1 << 24;

// All eight balanced base-256 digits of v at once: with 128 added to every
// byte, carries and all, byte i is digit i plus 128, and the flipped top bit
// takes the 128 off again.
__device__ __forceinline__ uint64_t digit_bytes(uint64_t v) {
  constexpr uint64_t k128 = 0x8080808080808080ull;
  return (v + k128) ^ k128;
}

// Digits i = 0..7 of four neighbours v[0..3], digit i of all four in d[i]: a
// 4 x 4 byte transpose of each half, eight v_perm a half.
__device__ __forceinline__ void digits_of4(const uint64_t (&v)[4], uint32_t (&d)[8]) {
  uint64_t b[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) b[q] = digit_bytes(v[q]);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t w[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) w[q] = uint32_t(b[q] >> (32 * h));
    // v_perm(hi, lo, sel): selector bytes 0-3 are lo's, 4-7 hi's.
    const uint32_t a0 = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u);  // bytes 0, 1 of w0, w1
    const uint32_t a1 = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u);  // bytes 2, 3
    const uint32_t c0 = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u);
    const uint32_t c1 = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
    d[4 * h + 0] = __builtin_amdgcn_perm(c0, a0, 0x05040100u);
    d[4 * h + 1] = __builtin_amdgcn_perm(c0, a0, 0x07060302u);
    d[4 * h + 2] = __builtin_amdgcn_perm(c1, a1, 0x05040100u);
    d[4 * h + 3] = __builtin_amdgcn_perm(c1, a1, 0x07060302u);
  }
}

// Byte offset of digit 0 of (row, column c) of a sufhip_digits2 with `rows`
// rows; party p's rows start at p * rows.  Digit i is 32 i further.
__device__ __forceinline__ size_t digit_off(size_t row, int c, size_t rows) {
  return (size_t(c >> 5) * (2 * rows) + row) * 256 + size_t(c & 31);
}

// One value's digits, byte by byte.
__device__ __forceinline__ void put_digits(int8_t* digits, size_t rows, size_t row, int c, int p,
                                           uint64_t v) {
  int8_t* at = digits + digit_off(size_t(p) * rows + row, c, rows);
  const uint64_t b = digit_bytes(v);
#pragma unroll
  for (int i = 0; i < 8; ++i) at[32 * i] = int8_t(b >> (8 * i));
}

// Both parties' outputs of gate e at the open value.
__device__ __forceinline__ void gate2(const TruncEpi& e, const EpiHdrs& eh, uint64_t open,
                                      uint64_t (&y)[2]) {
  const uint64_t w0 = trunc_table_word(eh.h[0], e.table[0], e.f, open);
  const uint64_t w1 = trunc_table_word(eh.h[1], e.table[1], e.f, open);
  y[0] = trunc_table_out(eh.h[0], e.f, open, w0);
  y[1] = trunc_table_out(eh.h[1], e.f, open, w1);
}

// Gates of up to kLdsGateBits bits with their tables in LDS, for streaming
// kernels: read from memory, each of a wave's 64 places in a 32 KB table is a
// line of the L1 cache to fetch, which four tables do not fit (the large
// norm's outputs, 1999 x 2048: 94 -> 54 us).
constexpr int kLdsGateBits = 12;
typedef uint64_t LdsGate[2][1 << kLdsGateBits];

// Both parties' tables of gate e; the caller syncs.
__device__ __forceinline__ void stage_gate(const TruncEpi& e, LdsGate& t) {
  const int n = 1 << (e.f - 1);  // pairs
#pragma unroll
  for (int p = 0; p < 2; ++p)
    for (int i = threadIdx.x; i < n; i += blockDim.x)
      reinterpret_cast<uint4*>(t[p])[i] = e.table[p][i];
}

__device__ __forceinline__ void gate2(const TruncEpi& e, const EpiHdrs& eh, const LdsGate& t,
                                      uint64_t open, uint64_t (&y)[2]) {
  const uint64_t at = open & ((uint64_t(1) << e.f) - 1);
  const uint64_t w0 = t[0][at], w1 = t[1][at];
  y[0] = trunc_table_out(eh.h[0], e.f, open, w0);
  y[1] = trunc_table_out(eh.h[1], e.f, open, w1);
}

// ---- host ----

inline int ff_fail(const char* what, const std::string& msg) {
  set_error(std::string(what) + ": " + msg);
  return SUFHIP_ERR_INVALID;
}

// Strides up to here reach any row of 2^24 within an address's 64 bits.
constexpr int64_t kMaxStride = int64_t(1) << 35;

inline int mat2_of(const sufhip_matrix2& g, int rows, const char* what, const char* name,
                   Mat2* out) {
  if (!g.p[0] || !g.p[1]) return ff_fail(what, std::string(name) + " is null");
  if (rows > 1 && (g.row_stride < 0 || g.row_stride > kMaxStride))
    return ff_fail(what, std::string(name) + ": row strides are in [0, 2^35]");
  *out = {{g.p[0], g.p[1]}, g.row_stride};
  return SUFHIP_OK;
}

// One party's rows as a set of words.
struct RowSet {
  const uint64_t* p;
  int64_t stride;
  int rows, cols;
};

inline const uint64_t* set_end(const RowSet& s) {
  return s.p + int64_t(s.rows - 1) * (s.rows > 1 ? s.stride : 0) + s.cols;
}

// Whether two sets may share a word.  Exact for rows of one stride (columns of
// one wider matrix do not meet), by the extents otherwise.
inline bool sets_meet(const RowSet& a, const RowSet& b) {
  if (a.rows < 1 || b.rows < 1 || a.cols < 1 || b.cols < 1) return false;
  if (a.p >= set_end(b) || b.p >= set_end(a)) return false;
  const bool one = a.rows == 1 && b.rows == 1;
  const int64_t st = a.rows > 1 ? a.stride : b.stride;
  if (one || st <= 0 || (a.rows > 1 && b.rows > 1 && a.stride != b.stride)) return true;
  // Words of a lie at a.p + r st + [0, a.cols), of b likewise: compare columns.
  int64_t d = (b.p - a.p) % st;
  if (d < 0) d += st;
  return d < a.cols || d + b.cols > st;
}

inline bool same_set(const RowSet& a, const RowSet& b) {
  return a.p == b.p && a.rows == b.rows && a.cols == b.cols &&
         (a.rows <= 1 || a.stride == b.stride);
}

// An output's stride: its rows must not meet each other.
inline bool bad_out_stride(int64_t stride, int rows, int cols) {
  return rows > 1 && (stride < cols || stride > kMaxStride);
}

inline RowSet row_set(const Mat2& m, int p, int rows, int cols) {
  return {m.p[p], m.stride, rows, cols};
}

inline int digits2_of(const sufhip_digits2& g, int rows, int cols, const char* what,
                      const char* name) {
  if ((reinterpret_cast<uintptr_t>(g.d_digits) & 15) != 0)
    return ff_fail(what, std::string(name) + " must be 16-byte aligned");
  if (g.rows != rows || g.cols != cols)
    return ff_fail(what, std::string(name) + " is of other rows or columns");
  return SUFHIP_OK;
}

// Whether `bytes` bytes from p on may share a word with a set (by its extent).
inline bool range_meets(const void* p, size_t bytes, const RowSet& s) {
  if (s.rows < 1 || s.cols < 1) return false;
  const char* a = static_cast<const char*>(p);
  return a < reinterpret_cast<const char*>(set_end(s)) &&
         reinterpret_cast<const char*>(s.p) < a + bytes;
}

// A stretch of memory; without bytes it meets nothing.
struct Range {
  const void* p;
  size_t bytes;
};
inline bool ranges_meet(const Range& a, const Range& b) {
  const char *pa = static_cast<const char*>(a.p), *pb = static_cast<const char*>(b.p);
  return a.p && b.p && a.bytes && b.bytes && pa < pb + b.bytes && pb < pa + a.bytes;
}
inline bool range_meets(const Range& r, const RowSet& s) {
  return r.p && r.bytes && s.p && range_meets(r.p, r.bytes, s);
}

// A gate folded into an operator: its own outputs and addend are not used.
inline int gate_of(const sufhip_trunc_epilogue& g, size_t n, const char* what, TruncEpi* out) {
  sufhip_trunc_epilogue t = g;
  if (t.add[0] || t.add[1]) return ff_fail(what, "the truncations take no addend");
  t.y[0] = t.y[1] = nullptr;
  return make_epi(&t, n, what, out, false);
}

// What a call's gates, LUTs and triples are read from, and nothing that it
// writes may meet.
struct Material {
  Range r[64];
  RowSet t[24];
  int n = 0, m = 0;

  void add(const void* p, size_t bytes) { r[n++] = {p, bytes}; }
  void gate(const uint8_t* const (&key)[2], const uint4* const (&table)[2], int f) {
    for (int p = 0; p < 2; ++p) {
      add(key[p], sufhip_trunc_key_bytes(SUFHIP_TRUNC_GAPARS, f));
      add(table[p], size_t(8) << f);
    }
  }
  void gate(const TruncEpi& e) {
    if (e.on) gate(e.key, e.table, e.f);
  }
  // Triples of n < 2^31 elements; one with an index may read all its rows.
  void chain(const ChainArgs& c, int prods, size_t lut_key_bytes) {
    for (int p = 0; p < 2; ++p) add(c.lut[p], lut_key_bytes);
    for (int k = 0; k < prods; ++k) {
      gate(c.tkey[k], c.ttab[k], c.tf[k]);
      for (const sufhip_term2* w : {&c.a[k], &c.b[k], &c.c[k]})
        for (int p = 0; p < 2; ++p) {
          if (w->index)
            add(w->p[p], w->len * w->stride * 8);
          else
            t[m++] = {w->p[p] + w->off, int64_t(w->stride), int(c.n), 1};
        }
    }
  }

  bool meets(const RowSet& w) const {
    for (int i = 0; i < n; ++i)
      if (range_meets(r[i], w)) return true;
    for (int i = 0; i < m; ++i)
      if (sets_meet(t[i], w)) return true;
    return false;
  }
  bool meets(const Range& w) const {
    for (int i = 0; i < n; ++i)
      if (ranges_meet(r[i], w)) return true;
    for (int i = 0; i < m; ++i)
      if (range_meets(w, t[i])) return true;
    return false;
  }
};

}  // namespace sufhip
