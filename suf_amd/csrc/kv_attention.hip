// The two products of attention over a paged cache, both parties, exact mod
// 2^64 (sufhip_kv_scores2, sufhip_kv_values2).
//
// With D = (x_0 - a_0) + (x_1 - a_1) a party's share of a product is
//   Z_p = C_p + D B_p + L_p E,   L_0 = A_0 + D,  L_1 = A_1,
// E and B_p read from the cache's pages.
#include <hip/hip_runtime.h>

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

// The packed elements of row (h, t): where they start and how many of them
// have a key (kv keys in the sequence).
struct Span {
  int first, len;
};
__device__ __forceinline__ Span span_of(const ProductArgs& a, int h, int t, int kv) {
  const int64_t r = int64_t(h) * a.b.tokens + t;
  const int64_t f = a.offsets[r], l = int64_t(a.offsets[r + 1]) - f;
  if (f < 0 || l <= 0 || f + l > a.n) return {0, 0};
  return {int(f), int(l < kv ? l : kv)};
}

// Both parties' finished values of output element i.
__device__ __forceinline__ void put2(const ProductArgs& a, const EpiHdrs& eh, int64_t i,
                                     uint64_t z0, uint64_t z1) {
  if (a.epi.on) {
    put_open(a.epi, eh, nullptr, size_t(i), z0 + z1 + a.mask);
  } else {
    a.out[0][i] = z0;
    a.out[1][i] = z1;
  }
}

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

// acc += l r over the digit pairs of weight below 256^8.
__device__ __forceinline__ void mul_digits(const v4i (&l)[kDigitPlanes],
                                           const v4i (&r)[kDigitPlanes],
                                           v4i (&acc)[kDigitPlanes]) {
#pragma unroll
  for (int i = 0; i < kDigitPlanes; ++i)
#pragma unroll
    for (int j = 0; i + j < kDigitPlanes; ++j)
      acc[i + j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(l[i], r[j], acc[i + j], 0, 0, 0);
}

// ---- left operands in LDS ----
//
// One 16 x 64 tile (16 rows, 64 of k) of the three left operands D, L_0, L_1
// as digit planes: byte j of k group g of row r of plane i of operand o at
// o * 8192 + i * 1024 + (r * 4 + g) * 16 + j, so a lane's operand is one
// 16-byte read and a wave reads a plane's 1 KB in order.
constexpr int kTileBytes = 3 * kDigitPlanes * 1024;

__device__ __forceinline__ void put_left(int8_t* tile, int r, int g, int q, const uint64_t (&x0)[4],
                                         const uint64_t (&x1)[4], const uint64_t (&a0)[4],
                                         const uint64_t (&a1)[4]) {
  uint64_t d[4], l0[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    d[k] = (x0[k] - a0[k]) + (x1[k] - a1[k]);
    l0[k] = a0[k] + d[k];
  }
  uint32_t pl[8];
  uint32_t* w = reinterpret_cast<uint32_t*>(tile) + (r * 4 + g) * 4 + q;
  digits_of4(d, pl);
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i * 256] = pl[i];
  digits_of4(l0, pl);
#pragma unroll
  for (int i = 0; i < 8; ++i) w[2048 + i * 256] = pl[i];
  digits_of4(a1, pl);
#pragma unroll
  for (int i = 0; i < 8; ++i) w[4096 + i * 256] = pl[i];
}

// Operand o's planes for lane l (row l % 16, k group l / 16).
__device__ __forceinline__ void get_left(const int8_t* tile, int o, int l,
                                         v4i (&pl)[kDigitPlanes]) {
  const int8_t* p = tile + o * 8192 + ((l & 15) * 4 + (l >> 4)) * 16;
#pragma unroll
  for (int i = 0; i < kDigitPlanes; ++i) pl[i] = *reinterpret_cast<const v4i*>(p + i * 1024);
}

// Both parties' digit products of a left tile with the right operands.
__device__ __forceinline__ void mul_tile(const int8_t* tile, int l, const v4i (&e)[kDigitPlanes],
                                         const v4i (&b0)[kDigitPlanes],
                                         const v4i (&b1)[kDigitPlanes],
                                         v4i (&acc)[2][kDigitPlanes]) {
  v4i x[kDigitPlanes];
  get_left(tile, 0, l, x);
  mul_digits(x, b0, acc[0]);
  mul_digits(x, b1, acc[1]);
  get_left(tile, 1, l, x);
  mul_digits(x, e, acc[0]);
  get_left(tile, 2, l, x);
  mul_digits(x, e, acc[1]);
}

__device__ __forceinline__ void clear(v4i (&acc)[2][kDigitPlanes]) {
#pragma unroll
  for (int p = 0; p < 2; ++p)
#pragma unroll
    for (int s = 0; s < kDigitPlanes; ++s) acc[p][s] = v4i{0, 0, 0, 0};
}

// A sequence's part of the batch for one cached head: its rows are (token,
// head of the group) in that order, row m at token t0 + m / group.
struct Seq {
  int s, hk, t0, rows, kv;
};
__device__ __forceinline__ Seq seq_at(const ProductArgs& a, int64_t z) {
  Seq q;
  q.s = int(z / a.pool.heads);
  q.hk = int(z - int64_t(q.s) * a.pool.heads);
  const int lo = a.b.cu[q.s], hi = a.b.cu[q.s + 1];
  q.t0 = lo > 0 ? lo : 0;
  const int t1 = hi < a.b.tokens ? hi : a.b.tokens;
  q.rows = t1 > q.t0 ? (t1 - q.t0) * a.group : 0;
  q.kv = a.b.lens[q.s];
  return q;
}

// ---- scores ----
//
// A workgroup of 4 waves takes 64 keys of one cached head, 16 to a wave (the
// columns of a 16 x 16 tile), and runs over row tiles.  The keys' digits are
// formed once, in registers, straight from the pages; the row tiles' pass
// through LDS.  k order: byte j = 2 i + e of group g stands for dim 8 i + 2 g
// + e of a 64-wide chunk, so each of a lane's 16-byte loads has its
// neighbours' beside it (64 contiguous bytes a key).
constexpr int kKeyTile = 64;
constexpr int kRowGroup = 16;  // row tiles whose spans are read at once

template <bool kVec>
__device__ __forceinline__ void load_keys(const uint64_t* p, bool ok, int g, int left,
                                          uint64_t (&v)[16]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d = 8 * i + 2 * g;
    if constexpr (kVec) {
      ulonglong2 w = make_ulonglong2(0, 0);
      if (ok && d < left) w = *reinterpret_cast<const ulonglong2*>(p + d);
      v[2 * i] = w.x;
      v[2 * i + 1] = w.y;
    } else {
      v[2 * i] = ok && d < left ? p[d] : 0;
      v[2 * i + 1] = ok && d + 1 < left ? p[d + 1] : 0;
    }
  }
}

template <bool kVec>
__device__ __forceinline__ void load_left4(const uint64_t* p, int d, int left, uint64_t (&v)[4]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int o = d + 8 * h;
    if constexpr (kVec) {
      ulonglong2 w = make_ulonglong2(0, 0);
      if (o < left) w = *reinterpret_cast<const ulonglong2*>(p + o);
      v[2 * h] = w.x;
      v[2 * h + 1] = w.y;
    } else {
      v[2 * h] = o < left ? p[o] : 0;
      v[2 * h + 1] = o + 1 < left ? p[o + 1] : 0;
    }
  }
}

// kHeld: 64-wide chunks of the keys held as digits over all row tiles (0:
// any number of chunks, loaded for each row tile again).
template <int kHeld, bool kVec>
__global__ void __launch_bounds__(256, kHeld == 2 ? 1 : 2) kv_scores2_kernel(ProductArgs a,
                                                                             int chunks) {
  extern __shared__ __align__(16) int8_t tiles[];
  __shared__ int first[kRowGroup * 16];
  __shared__ int len[kRowGroup * 16];
  __shared__ unsigned active;
  const int tid = threadIdx.x, l = tid & 63, w = tid >> 6;
  const int g = l >> 4, n = l & 15;
  const int dim = a.pool.dim;
  const EpiHdrs eh = epi_hdrs(a.epi);
  for (int64_t z = blockIdx.z; z < int64_t(a.b.seqs) * a.pool.heads; z += gridDim.z) {
    const Seq q = seq_at(a, z);
    const int row_tiles = (q.rows + 15) / 16;
    for (int64_t k0 = int64_t(blockIdx.x) * kKeyTile; k0 < q.kv;
         k0 += int64_t(gridDim.x) * kKeyTile) {
      const int64_t key = k0 + 16 * w + n;
      const int64_t place = key < q.kv ? kv_place(a.b, a.pool, q.s, q.hk, key) : -1;
      const bool ok = place >= 0;
      constexpr int kC = kHeld ? kHeld : 1;
      v4i K[kC][3][kDigitPlanes];
      auto load_chunk = [&](int c, v4i (&to)[3][kDigitPlanes]) {
        uint64_t v[3][16];
        const int64_t o = place + 64 * c;
        load_keys<kVec>(a.pool.e + o, ok, g, dim - 64 * c, v[0]);
        load_keys<kVec>(a.pool.b[0] + o, ok, g, dim - 64 * c, v[1]);
        load_keys<kVec>(a.pool.b[1] + o, ok, g, dim - 64 * c, v[2]);
#pragma unroll
        for (int o3 = 0; o3 < 3; ++o3) digits_of16(v[o3], to[o3]);
      };
      if constexpr (kHeld > 0) {
#pragma unroll
        for (int c = 0; c < kC; ++c) load_chunk(c, K[c]);
      }
      for (int rb = blockIdx.y; rb < row_tiles; rb += gridDim.y * kRowGroup) {
        // Spans of up to 16 row tiles, and which of them see these keys.
        __syncthreads();
        {
          const int m = (rb + (tid >> 4) * int(gridDim.y)) * 16 + (tid & 15);
          Span sp{0, 0};
          if (m < q.rows && m >= 0) {
            const int tl = m / a.group;
            sp = span_of(a, q.hk * a.group + (m - tl * a.group), q.t0 + tl, q.kv);
          }
          first[tid] = sp.first;
          len[tid] = sp.len;
          if (tid == 0) active = 0;
          const uint64_t seen = __ballot(sp.len > k0);
          __syncthreads();
          if (l == 0) {
            unsigned bits = 0;
            for (int i = 0; i < 4; ++i)
              if ((seen >> (16 * i)) & 0xffff) bits |= 1u << (4 * w + i);
            if (bits) atomicOr(&active, bits);
          }
        }
        __syncthreads();
        for (unsigned todo = active; todo; todo &= todo - 1) {
          const int ti = __builtin_ctz(todo);
          const int m0 = (rb + ti * int(gridDim.y)) * 16;
          // The tile's left operands: thread (row, part) takes 4 of k in each
          // chunk.  Rows past the last stay as they are: a row of the left
          // operand reaches that row of the product alone.
          {
            const int r = tid >> 4, m = m0 + r, lg = tid & 3, lq = (tid >> 2) & 3;
            if (m < q.rows) {
              const int tl = m / a.group, t = q.t0 + tl;
              const int h = q.hk * a.group + (m - tl * a.group);
              const int64_t xo = int64_t(t) * a.xts + int64_t(h) * a.xhs;
              const int64_t ao = (int64_t(t) * a.heads + h) * dim;
              for (int c = 0; c < chunks; ++c) {
                const int d = 16 * lq + 2 * lg, left = dim - 64 * c;
                uint64_t x0[4], x1[4], a0[4], a1[4];
                load_left4<kVec>(a.x[0] + xo + 64 * c, d, left, x0);
                load_left4<kVec>(a.x[1] + xo + 64 * c, d, left, x1);
                load_left4<kVec>(a.a[0] + ao + 64 * c, d, left, a0);
                load_left4<kVec>(a.a[1] + ao + 64 * c, d, left, a1);
                put_left(tiles + c * kTileBytes, r, lg, lq, x0, x1, a0, a1);
              }
            }
          }
          // The product's shares of C for this lane's elements.
          uint64_t cw[2][4];
          int at[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int row = 4 * g + r;
            at[r] = key < len[ti * 16 + row] ? first[ti * 16 + row] + int(key) : -1;
          }
          const auto load_c = [&] {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              cw[0][r] = at[r] >= 0 ? a.c[0][at[r]] : 0;
              cw[1][r] = at[r] >= 0 ? a.c[1][at[r]] : 0;
            }
          };
          if constexpr (kHeld > 0) load_c();
          __syncthreads();
          v4i acc[2][kDigitPlanes];
          clear(acc);
          if constexpr (kHeld > 0) {
#pragma unroll
            for (int c = 0; c < kC; ++c)
              mul_tile(tiles + c * kTileBytes, l, K[c][0], K[c][1], K[c][2], acc);
          } else {
            for (int c = 0; c < chunks; ++c) {
              load_chunk(c, K[0]);
              mul_tile(tiles + c * kTileBytes, l, K[0][0], K[0][1], K[0][2], acc);
            }
            load_c();
          }
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (at[r] >= 0)
              put2(a, eh, at[r], from_sums(acc[0], r) + cw[0][r], from_sums(acc[1], r) + cw[1][r]);
          __syncthreads();
        }
      }
    }
  }
}

// ---- values ----
//
// A workgroup takes 16 rows, 16 columns a wave, and a share of the keys in
// chunks of 64 (the k of the product).  k order: byte j of group g stands for
// key 16 (j % 4) + 4 (j / 4) + g of a chunk, so that the left operand's loads
// (4 keys a thread) and the pages' (one column of 16 keys a lane) both run
// over neighbouring words.
struct ValuesArgs {
  ProductArgs p;
  int splits, cols;   // shares of the keys; columns of a workgroup
  uint64_t* part;     // splits > 1: [splits][2][tokens * heads][dim] sums
};

// Chunks whose digit sums stay within int32: 2 products of 8 digit pairs of
// at most 2^14 at 64 of k are 2^24 a chunk.
constexpr int kSumChunks = 64;

template <int kWaves>
__global__ void __launch_bounds__(64 * kWaves, 2) kv_values2_kernel(ValuesArgs va) {
  const ProductArgs& a = va.p;
  __shared__ __align__(16) int8_t tile[kTileBytes];
  __shared__ int64_t base[kKeyTile];
  __shared__ int first[16];
  __shared__ int len[16];
  const int tid = threadIdx.x, l = tid & 63, w = tid >> 6;
  const int g = l >> 4, n = l & 15;
  const int dim = a.pool.dim;
  const EpiHdrs eh = epi_hdrs(a.epi);
  const int blocks = (dim + va.cols - 1) / va.cols;
  const int split = int(blockIdx.x) % va.splits;
  const int col = (int(blockIdx.x) / va.splits) * va.cols + 16 * w + n;
  if (int(blockIdx.x) / va.splits >= blocks) return;
  for (int64_t z = blockIdx.z; z < int64_t(a.b.seqs) * a.pool.heads; z += gridDim.z) {
    const Seq q = seq_at(a, z);
    for (int64_t m0 = int64_t(blockIdx.y) * 16; m0 < q.rows; m0 += int64_t(gridDim.y) * 16) {
      __syncthreads();
      if (tid < 16) {
        const int m = int(m0) + tid;
        Span sp{0, 0};
        if (m < q.rows) {
          const int tl = m / a.group;
          sp = span_of(a, q.hk * a.group + (m - tl * a.group), q.t0 + tl, q.kv);
        }
        first[tid] = sp.first;
        len[tid] = sp.len;
      }
      __syncthreads();
      int most = 0;
#pragma unroll
      for (int r = 0; r < 16; ++r) most = len[r] > most ? len[r] : most;
      const int chunks = (most + kKeyTile - 1) / kKeyTile;
      const int per = (chunks + va.splits - 1) / va.splits;
      const int c0 = split * per, c1 = c0 + per < chunks ? c0 + per : chunks;
      uint64_t sum[2][4] = {};
      v4i acc[2][kDigitPlanes];
      clear(acc);
      for (int c = c0; c < c1; ++c) {
        const int64_t k0 = int64_t(c) * kKeyTile;
        __syncthreads();
        if (tid < kKeyTile) {
          const int64_t key = k0 + tid;
          base[tid] = key < q.kv ? kv_place(a.b, a.pool, q.s, q.hk, key) : -1;
        }
        for (int u = tid; u < 256; u += 64 * kWaves) {
          const int r = u >> 4, part = u & 15, ln = len[r];
          if (m0 + r < q.rows) {
            uint64_t x0[4], x1[4], a0[4], a1[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int64_t key = k0 + 16 * i + part;
              const bool in = key < ln;
              const int64_t o = int64_t(first[r]) + key;
              x0[i] = in ? a.x[0][o] : 0;
              x1[i] = in ? a.x[1][o] : 0;
              a0[i] = in ? a.a[0][o] : 0;
              a1[i] = in ? a.a[1][o] : 0;
            }
            put_left(tile, r, part & 3, part >> 2, x0, x1, a0, a1);
          }
        }
        __syncthreads();
        v4i K[3][kDigitPlanes];
        {
          uint64_t v[3][16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const int64_t o = base[16 * (j & 3) + 4 * (j >> 2) + g];
            const bool in = o >= 0 && col < dim;
            v[0][j] = in ? a.pool.e[o + col] : 0;
            v[1][j] = in ? a.pool.b[0][o + col] : 0;
            v[2][j] = in ? a.pool.b[1][o + col] : 0;
          }
#pragma unroll
          for (int o3 = 0; o3 < 3; ++o3) digits_of16(v[o3], K[o3]);
        }
        mul_tile(tile, l, K[0], K[1], K[2], acc);
        if (c - c0 + 1 == c1 - c0 || (c - c0) % kSumChunks == kSumChunks - 1) {
#pragma unroll
          for (int p = 0; p < 2; ++p)
#pragma unroll
            for (int r = 0; r < 4; ++r) sum[p][r] += from_sums(acc[p], r);
          clear(acc);
        }
      }
      if (col >= dim) continue;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int m = int(m0) + 4 * g + r;
        if (m >= q.rows) continue;
        const int tl = m / a.group;
        const int64_t row = int64_t(q.t0 + tl) * a.heads + q.hk * a.group + (m - tl * a.group);
        const int64_t o = row * dim + col;
        if (va.splits > 1) {
          const int64_t all = int64_t(a.b.tokens) * a.heads * dim;
          va.part[2 * split * all + o] = sum[0][r];
          va.part[(2 * split + 1) * all + o] = sum[1][r];
        } else {
          put2(a, eh, o, sum[0][r] + a.c[0][o], sum[1][r] + a.c[1][o]);
        }
      }
    }
  }
}

// Adds the splits' sums: 32 outputs a workgroup, 8 lanes over the splits.
__global__ void __launch_bounds__(256) kv_values2_join_kernel(ValuesArgs va) {
  const ProductArgs& a = va.p;
  __shared__ uint64_t s[2][8][32];
  const int64_t all = int64_t(a.b.tokens) * a.heads * a.pool.dim;
  const int u = threadIdx.x & 31, lane = threadIdx.x >> 5;
  const EpiHdrs eh = epi_hdrs(a.epi);
  for (int64_t o0 = int64_t(blockIdx.x) * 32; o0 < all; o0 += int64_t(gridDim.x) * 32) {
    const int64_t o = o0 + u;
    uint64_t z0 = 0, z1 = 0;
    if (o < all)
      for (int k = lane; k < va.splits; k += 8) {
        z0 += va.part[2 * k * all + o];
        z1 += va.part[(2 * k + 1) * all + o];
      }
    __syncthreads();
    s[0][lane][u] = z0;
    s[1][lane][u] = z1;
    __syncthreads();
    if (lane == 0 && o < all && seq_of(a.b, int(o / (int64_t(a.heads) * a.pool.dim))) >= 0) {
      z0 = a.c[0][o];
      z1 = a.c[1][o];
      for (int k = 0; k < 8; ++k) {
        z0 += s[0][k][u];
        z1 += s[1][k][u];
      }
      put2(a, eh, o, z0, z1);
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
  if (g.heads < 1 || g.heads % g.pool.kv_heads)
    return kv_fail(what, "heads must be a multiple of the pool's kv_heads");
  if (g.n > 0x7fffffffu) return kv_fail(what, "at most 2^31 - 1 packed elements");
  const size_t rows = size_t(a.b.tokens) * size_t(g.heads);
  if (rows > (1u << 30)) return kv_fail(what, "at most 2^30 rows");
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

int cu_total() {
  int cus = 256, dev = 0;
  if (hipGetDevice(&dev) != hipSuccess ||
      hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess) {
    (void)hipGetLastError();
    cus = 256;
  }
  return cus;
}

template <int kHeld, bool kVec>
int launch_scores(const ProductArgs& a, const dim3& grid, int chunks, hipStream_t st) {
  const size_t lds = size_t(chunks) * kTileBytes;
  const void* f = reinterpret_cast<const void*>(kv_scores2_kernel<kHeld, kVec>);
  if (lds > 48 * 1024)
    SUFHIP_CHECK(hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, int(lds)),
                 "kv_scores2_kernel LDS");
  hipLaunchKernelGGL((kv_scores2_kernel<kHeld, kVec>), grid, dim3(256), lds, st, a, chunks);
  return check_launch("kv_scores2_kernel");
}

// Shares of the keys: as many as fill the chip twice, each of two chunks of
// keys at least.
int values_splits(int64_t groups, int64_t max_keys, int cus) {
  const int64_t want = (4 * int64_t(cus) + groups - 1) / groups;
  const int64_t most = max_keys / (2 * kKeyTile);
  const int64_t n = want < most ? want : most;
  return n < 1 ? 1 : int(n < 1024 ? n : 1024);
}

struct ValuesPlan {
  int cols, waves, blocks, splits;
  int64_t row_tiles, zs;
};
ValuesPlan plan_values(const sufhip_kv_batch& b, const sufhip_kv_pool& p, int heads) {
  ValuesPlan v{};
  v.waves = p.dim <= 64 ? 4 : 8;
  v.cols = 16 * v.waves;
  v.blocks = (p.dim + v.cols - 1) / v.cols;
  const int64_t rows = int64_t(b.max_new) * (heads / p.kv_heads);
  v.row_tiles = rows < 1 ? 1 : (rows + 15) / 16;
  v.zs = int64_t(b.seqs) * p.kv_heads;
  v.splits = values_splits(v.row_tiles * v.zs * v.blocks, b.max_keys, cu_total());
  return v;
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
  const int chunks = (a.pool.dim + 63) / 64;
  const int64_t key_tiles = (int64_t(args->batch.max_keys) + kKeyTile - 1) / kKeyTile;
  const int64_t row_tiles = (int64_t(args->batch.max_new) * a.group + 15) / 16;
  const int64_t zs = int64_t(a.b.seqs) * a.pool.heads;
  // Row tiles are spread over workgroups until four of them share a CU.
  const int64_t want = (4 * 4 * int64_t(cu_total()) + key_tiles * zs) / (key_tiles * zs + 1);
  const dim3 grid(clip(key_tiles, 1 << 20), clip(want < row_tiles ? want : row_tiles, 65535),
                  clip(zs, 65535));
  const hipStream_t st = as_stream(stream);
  const bool reuse = row_tiles > int64_t(grid.y);  // a workgroup runs over several row tiles
  if (chunks == 1)
    return vec ? launch_scores<1, true>(a, grid, chunks, st)
               : launch_scores<1, false>(a, grid, chunks, st);
  if (chunks == 2 && reuse)
    return vec ? launch_scores<2, true>(a, grid, chunks, st)
               : launch_scores<2, false>(a, grid, chunks, st);
  return vec ? launch_scores<0, true>(a, grid, chunks, st)
             : launch_scores<0, false>(a, grid, chunks, st);
}

size_t sufhip_kv_values2_work_bytes(const sufhip_kv_batch* batch, const sufhip_kv_pool* pool,
                                    int heads) {
  if (!batch || !pool || pool->kv_heads < 1 || pool->dim < 1 || heads < 1 || batch->tokens < 1 ||
      batch->seqs < 1 || heads % pool->kv_heads)
    return 0;
  const ValuesPlan v = plan_values(*batch, *pool, heads);
  if (v.splits <= 1) return 0;
  return size_t(v.splits) * 16 * size_t(batch->tokens) * size_t(heads) * size_t(pool->dim);
}

int sufhip_kv_values2(const sufhip_kv_product2_args* args, void* stream) {
  ValuesArgs va{};
  bool empty = false;
  if (int rc = product_args(args, true, "sufhip_kv_values2", &va.p, &empty)) return rc;
  if (empty) return SUFHIP_OK;
  const ValuesPlan v = plan_values(args->batch, args->pool, args->heads);
  va.splits = v.splits;
  va.cols = v.cols;
  if (v.splits > 1) {
    const size_t need = sufhip_kv_values2_work_bytes(&args->batch, &args->pool, args->heads);
    SUFHIP_REQUIRE(args->d_work && at16(args->d_work) && args->work_bytes >= need,
                   "sufhip_kv_values2: d_work smaller than its work bytes, or not 16-byte aligned");
    va.part = static_cast<uint64_t*>(args->d_work);
  }
  const dim3 grid(unsigned(v.splits * v.blocks), clip(v.row_tiles, 65535), clip(v.zs, 65535));
  const hipStream_t st = as_stream(stream);
  if (v.waves == 4)
    hipLaunchKernelGGL((kv_values2_kernel<4>), grid, dim3(256), 0, st, va);
  else
    hipLaunchKernelGGL((kv_values2_kernel<8>), grid, dim3(512), 0, st, va);
  if (int rc = check_launch("kv_values2_kernel")) return rc;
  if (v.splits == 1) return SUFHIP_OK;
  const int64_t all = int64_t(va.p.b.tokens) * va.p.heads * va.p.pool.dim;
  hipLaunchKernelGGL(kv_values2_join_kernel, dim3(clip((all + 31) / 32, 1 << 20)), dim3(256), 0, st,
                     va);
  return check_launch("kv_values2_join_kernel");
}

}  // extern "C"
