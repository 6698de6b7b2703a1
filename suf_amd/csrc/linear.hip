// Share x public weight for both parties and any number of rows, dense or
// grouped by expert, with the bias, the truncation, an activation and a
// residual in its epilogue (sufhip_linear2), on the int8 matrix cores (gfx950
// v_mfma_i32_16x16x64_i8 and 32x32x32_i8), exact mod 2^64.
//
// Both operands in balanced base-256 digits: x = sum_{i<8} x_i 256^i, W =
// sum_{j<J} w_j 256^j, so that X W = sum_{s<8} 256^s S_s mod 2^64 with S_s =
// sum_{i+j=s} X_i W_j: 15 int8 products for J = 2.  |S_s| <= J K 2^14 < 2^31, so
// sums in int32 are exact and are joined in 64 bits once, at the end.
//
// Rows of a matrix tile: 4 (t >> 1) + 2 p + (t & 1) for token t of party p.  An
// accumulator's four neighbouring rows are then two tokens of both parties, so
// a lane holds both shares of its outputs and opens them without an exchange.
//
// W's planes: [expert][N / 64][K / 32][J][64][32] bytes (N padded to 64
// columns, K to 64 rows): a wave's column tile is one contiguous stream.
#include <hip/hip_runtime.h>

#include "chain_device.hpp"
#include "feedforward_device.hpp"

namespace sufhip {
namespace {

typedef int v4acc __attribute__((ext_vector_type(4)));
typedef int v16acc __attribute__((ext_vector_type(16)));
typedef uint64_t u64x2u __attribute__((ext_vector_type(2), aligned(8)));

constexpr int kCols = 64;         // columns of a weight tile
constexpr int kTileBytes = 2048;  // of one digit and 32 k

struct LinArgs {
  Mat2 x;
  const int8_t* xd;  // digits of x, or NULL
  int x_rows, rows, K, N, kb, groups, experts;
  const int8_t* w;
  size_t expert_bytes;
  const int64_t* bias;
  const int32_t* map;
  const int32_t* offsets;
  int tiles, slices;
  uint64_t* part;  // several k-slices: [slices][2][rows][N] sums
  uint64_t* zhat;  // the masked opens [rows][N], for the epilogue's launch
  uint64_t mask;
  TruncEpi epi;
  Mat2 res;
  uint64_t* out[2];
  int64_t out_stride;
  int8_t* digits;  // the outputs as digits (the epilogue's launch)
};

// The expert of output row i and whether it has one.
__device__ __forceinline__ int expert_of(const LinArgs& a, int row) {
  if (!a.offsets) return 0;
  int lo = 0, hi = a.experts;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.offsets[mid] <= row)
      lo = mid;
    else
      hi = mid;
  }
  return a.offsets[lo] <= row && row < a.offsets[lo + 1] ? lo : -1;
}

// Row tile number ti, of `per` rows: its expert and rows.  Every lane of the
// wave takes part; experts are counted 64 at a time.
struct RowTile {
  int e, begin, end;
};
__device__ __forceinline__ RowTile row_tile(const LinArgs& a, int ti, int per) {
  if (!a.offsets) {
    const int begin = ti * per;
    const int end = begin + per < a.rows ? begin + per : a.rows;
    return {begin < a.rows ? 0 : -1, begin, end};
  }
  const int lane = threadIdx.x & 63;
  int base = 0;
  for (int e0 = 0; e0 < a.experts; e0 += 64) {
    const int e = e0 + lane;
    int lo = 0, hi = 0;
    if (e < a.experts) {
      lo = a.offsets[e];
      hi = a.offsets[e + 1];
      lo = lo < 0 ? 0 : (lo > a.rows ? a.rows : lo);
      hi = hi < lo ? lo : (hi > a.rows ? a.rows : hi);
    }
    const int n = (hi - lo + per - 1) / per;
    int incl = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int v = __shfl_up(incl, d, 64);
      if (lane >= d) incl += v;
    }
    const unsigned long long over = __ballot(base + incl > ti);
    if (over) {
      const int f = __builtin_ctzll(over);
      const int first = base + __shfl(incl - n, f, 64);
      const int flo = __shfl(lo, f, 64), fhi = __shfl(hi, f, 64);
      const int begin = flo + (ti - first) * per;
      return {e0 + f, begin, begin + per < fhi ? begin + per : fhi};
    }
    base += __shfl(incl, 63, 64);
  }
  return {-1, 0, 0};
}

// Both shares of output (row, col) where a launch finishes them: bias, then
// the k-slices' sums, the masked open, or the truncation and the residual.
__device__ __forceinline__ void put_output(const LinArgs& a, const EpiHdrs& eh, int slice, int e,
                                           int row, int col, uint64_t y0, uint64_t y1) {
  const size_t i = size_t(row) * a.N + col;
  if (a.slices > 1) {
    const size_t mn = size_t(a.rows) * a.N;
    a.part[size_t(slice) * 2 * mn + i] = y0;
    a.part[(size_t(slice) * 2 + 1) * mn + i] = y1;
    return;
  }
  if (a.bias) y0 += uint64_t(a.bias[size_t(e) * a.N + col]);
  if (a.zhat) {
    a.zhat[i] = y0 + y1 + a.mask;
    return;
  }
  uint64_t y[2] = {y0, y1};
  if (a.epi.on) gate2(a.epi, eh, y0 + y1 + a.mask, y);
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    if (a.res.p[0]) y[p] += a.res.p[p][int64_t(row) * a.res.stride + col];
    a.out[p][int64_t(row) * a.out_stride + col] = y[p];
  }
}

// Few rows: a workgroup of four waves takes one row tile (kT / 2 tokens of both
// parties), 128 columns, 32 a wave, and one k-slice.  W goes straight into
// registers, each word read once; X's digits, which the four waves share, are
// formed on the way into LDS (or come as digits), 64 k at a time, the next
// chunk's loads in flight under this one's products.
template <int kT, int J, bool kDigits>
__global__ void __launch_bounds__(256, J <= 2 ? 2 : 1) linear_skinny_kernel(LinArgs a) {
  constexpr int kTok = kT / 2;
  constexpr int kC = kT == 16 ? 2 : 1;      // column fragments of a wave
  constexpr int kR = kT == 16 ? 4 : 16;     // accumulator registers of one
  constexpr int kSteps = kT == 16 ? 1 : 2;  // matrix steps of a chunk
  constexpr int kPieces = kT / 8;           // of 16 bytes, a thread stores in a chunk
  typedef typename std::conditional<kT == 16, v4acc, v16acc>::type Acc;
  __shared__ __align__(16) int8_t lds[2][kSteps * 8 * 1024];  // [step][digit][lane] of 16 k
  const int l = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
  const int total = int(gridDim.x);
  int id = int(blockIdx.x);
  // Row tiles of the same weights run on one XCD, one after the other.
  if (total % 8 == 0) id = (id % 8) * (total / 8) + id / 8;
  const int ti = id % a.tiles, rest = id / a.tiles;
  const int slice = rest % a.slices, c0 = rest / a.slices * 128 + 32 * w;
  const RowTile rt = row_tile(a, ti, kTok);
  if (rt.e < 0 || rt.begin >= rt.end) return;  // the whole workgroup
  const EpiHdrs eh = epi_hdrs(a.epi);
  // The row that this thread brings to LDS: a run of kT / 4 words of it, or
  // (digits) its pieces of 16 bytes.
  const int r = kDigits ? l % kT : int(threadIdx.x) / (256 / kT);
  const int kq = int(threadIdx.x) % (256 / kT) * (kT / 4);  // first word in the chunk
  const int p = (r >> 1) & 1, t = 2 * (r >> 2) + (r & 1);
  int xr = rt.begin + t;
  bool live = xr < rt.end;
  if (live && a.map) xr = a.map[xr];
  live = live && xr >= 0 && xr < a.x_rows;
  const uint64_t* xrow =
      kDigits ? nullptr : (p ? a.x.p[1] : a.x.p[0]) + (live ? int64_t(xr) * a.x.stride : 0) + kq;
  const int8_t* drow = kDigits ? a.xd + (live ? (size_t(p) * a.x_rows + xr) * 256 : 0) : nullptr;
  const size_t dstep = size_t(2) * a.x_rows * 256;
  // This wave's columns; past the last weight tile it repeats the last one.
  const int g = c0 / kCols < a.groups ? c0 / kCols : a.groups - 1;
  const int8_t* wl = a.w + size_t(rt.e) * a.expert_bytes + size_t(g) * a.kb * (J * kTileBytes) +
                     (c0 % kCols) * 32 +
                     (kT == 16 ? (l >> 5) * (J * kTileBytes) + (l & 15) * 32 + ((l >> 4) & 1) * 16
                               : (l & 31) * 32 + (l >> 5) * 16);
  const int chunks = a.kb / 2;
  const int q0 = int(int64_t(chunks) * slice / a.slices);
  const int q1 = int(int64_t(chunks) * (slice + 1) / a.slices);
  struct Wreg {
    v4i v[kSteps][kC][J];
  };
  u64x2u xw[kDigits ? 1 : kT / 8];
  v4i xd[kDigits ? kPieces : 1];
  auto load_w = [&](Wreg& g, int q) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int c = 0; c < kC; ++c)
#pragma unroll
        for (int j = 0; j < J; ++j)
          g.v[s][c][j] = load16(wl + (size_t(q) * 2 + s) * (J * kTileBytes) + j * kTileBytes +
                                c * (kT * 32));
  };
  auto load_x = [&](int q) {
    if constexpr (kDigits) {
#pragma unroll
      for (int u = 0; u < kPieces; ++u) {
        // Piece threadIdx + 256 u: step, digit and lane of the fragment.
        const int piece = int(threadIdx.x) + 256 * u;
        const int i = (piece >> 6) & 7;
        const int sixteen = kT == 16 ? l / 16 : 2 * (piece >> 9) + l / 32;
        const int kb = 2 * q + (sixteen >> 1);
        xd[u] = v4i{0, 0, 0, 0};
        if (live && 32 * kb < a.K)
          xd[u] = load16(drow + size_t(kb) * dstep + 32 * i + 16 * (sixteen & 1));
      }
    } else {
      const int k = 64 * q + kq;
#pragma unroll
      for (int u = 0; u < kT / 8; ++u) xw[u] = u64x2u{0, 0};
      if (live && k + kT / 4 <= a.K) {
#pragma unroll
        for (int u = 0; u < kT / 8; ++u)
          xw[u] = *reinterpret_cast<const u64x2u*>(xrow + 64 * q + 2 * u);
      } else if (live) {
#pragma unroll
        for (int u = 0; u < kT / 8; ++u) {
          if (k + 2 * u < a.K) xw[u][0] = xrow[64 * q + 2 * u];
          if (k + 2 * u + 1 < a.K) xw[u][1] = xrow[64 * q + 2 * u + 1];
        }
      }
    }
  };
  auto store_x = [&](int buf) {
    if constexpr (kDigits) {
#pragma unroll
      for (int u = 0; u < kPieces; ++u)
        *reinterpret_cast<v4i*>(&lds[buf][(int(threadIdx.x) + 256 * u) * 16]) = xd[u];
    } else {
      const int lane = (kT == 16 ? kq >> 4 : (kq >> 4) & 1) * kT + r;
      int8_t* at = &lds[buf][(kT == 16 ? 0 : kq >> 5) * 8192 + lane * 16 + (kq & 15)];
      uint32_t d[kT / 16][8];
#pragma unroll
      for (int u = 0; u < kT / 16; ++u) {
        const uint64_t v[4] = {xw[2 * u][0], xw[2 * u][1], xw[2 * u + 1][0], xw[2 * u + 1][1]};
        digits_of4(v, d[u]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (kT == 16)
          *reinterpret_cast<uint32_t*>(at + 1024 * i) = d[0][i];
        else
          *reinterpret_cast<uint2*>(at + 1024 * i) = make_uint2(d[0][i], d[1][i]);
      }
    }
  };
  Acc acc[kC][8];
#pragma unroll
  for (int c = 0; c < kC; ++c)
#pragma unroll
    for (int s = 0; s < 8; ++s)
#pragma unroll
      for (int q = 0; q < kR; ++q) acc[c][s][q] = 0;
  auto products = [&](const Wreg& g, int buf) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      v4i d[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        d[i] = *reinterpret_cast<const v4i*>(&lds[buf][s * 8192 + i * 1024 + 16 * l]);
#pragma unroll
      for (int c = 0; c < kC; ++c)
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
          for (int i = 0; i + j < 8; ++i) {
            if constexpr (kT == 16)
              acc[c][i + j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(d[i], g.v[s][c][j],
                                                                    acc[c][i + j], 0, 0, 0);
            else
              acc[c][i + j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(d[i], g.v[s][c][j],
                                                                    acc[c][i + j], 0, 0, 0);
          }
    }
  };
  auto step = [&](int q, const Wreg& cur, Wreg& next) {
    if (q + 1 < q1) {
      load_w(next, q + 1);
      load_x(q + 1);
    }
    products(cur, (q - q0) & 1);
    if (q + 1 < q1) store_x((q + 1 - q0) & 1);
    __syncthreads();
  };
  if (q0 < q1) {
    Wreg wa, wb;
    load_w(wa, q0);
    load_x(q0);
    store_x(0);
    __syncthreads();
    for (int q = q0; q < q1; q += 2) {
      step(q, wa, wb);
      if (q + 1 < q1) step(q + 1, wb, wa);
    }
  }
#pragma unroll
  for (int c = 0; c < kC; ++c) {
    const int col = c0 + c * kT + l % kT;
    if (col >= a.N) continue;
#pragma unroll
    for (int b = 0; b < kR / 4; ++b) {
      uint64_t v[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        v[q] = 0;
#pragma unroll
        for (int s = 0; s < 8; ++s) v[q] += uint64_t(int64_t(acc[c][s][4 * b + q])) << (8 * s);
      }
      const int pairs = kT == 16 ? l / 16 : 2 * b + l / 32;  // of tokens, in the tile
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = rt.begin + 2 * pairs + h;
        if (row < rt.end) put_output(a, eh, slice, rt.e, row, col, v[h], v[2 + h]);
      }
    }
  }
}

// acc += a b with the accumulator in the accumulation registers for the whole
// loop.  (The compiler keeps 256 of them in vector registers and copies them
// to and from the others in every step.)  The wait before it covers a vector
// instruction's write of an operand; between two products into one
// accumulator lie at least six others.
__device__ __forceinline__ void mfma_acc(v16acc& acc, v4i a, v4i b) {
  asm volatile("s_nop 1\n\tv_mfma_i32_32x32x32_i8 %0, %1, %2, %0" : "+a"(acc) : "v"(a), "v"(b));
}

// Between mfma_acc and other uses of the accumulators: the last products' (or
// the zeros') writes are done.  The ties keep every such use behind the wait.
template <int kC, int kS>
__device__ __forceinline__ void acc_settle(v16acc (&acc)[kC][kS]) {
  asm volatile("s_nop 15\n\ts_nop 15" ::);
#pragma unroll
  for (int c = 0; c < kC; ++c)
#pragma unroll
    for (int s = 0; s < kS; ++s) asm volatile("" : "+a"(acc[c][s]));
}

// Many rows: a workgroup takes 32 tokens of both parties (two tiles of 32
// rows) and 128 columns; wave (m, n) tile m and column tile n, 32 x 64 values
// in 256 accumulator registers.  A k-block's operands, X's digits (gathered a
// row at a time) and W's, pass through LDS in the fragments' order, the next
// block's loads in flight under this one's products.
constexpr int kBigTok = 32;

template <int J>
__global__ void __launch_bounds__(256, 1) linear_tile_kernel(LinArgs a) {
  constexpr int kBlocks = 16 + 4 * J;  // of 1 KB: X (tile, digit), W (column tile, digit, half)
  __shared__ __align__(16) int8_t lds[2][kBlocks * 1024];
  const int l = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
  const int total = int(gridDim.x);
  int id = int(blockIdx.x);
  // An XCD takes neighbouring column tiles of the same rows.
  if (total % 8 == 0) id = (id % 8) * (total / 8) + id / 8;
  const int gpairs = (a.groups + 1) / 2;
  const int gp = id % gpairs, rest = id / gpairs;
  const int slice = rest % a.slices, ti = rest / a.slices;
  const RowTile rt = row_tile(a, ti, kBigTok);
  if (rt.e < 0 || rt.begin >= rt.end) return;  // the whole workgroup
  const EpiHdrs eh = epi_hdrs(a.epi);
  const int m = w >> 1, n = w & 1;
  // Loads of this thread: four X fragments of row tile m (digits 4 n .. 4 n +
  // 3) and J of W's blocks, at its place in the fragment.
  const int r = l & 31, half = l >> 5;
  const int p = (r >> 1) & 1, t = 2 * (r >> 2) + (r & 1);
  int xr = rt.begin + 16 * m + t;
  bool live = xr < rt.end;
  if (live && a.map) xr = a.map[xr];
  live = live && xr >= 0 && xr < a.x_rows;
  // A row that is not there reads row 0 and is zeros in LDS.
  const int8_t* xl = a.xd + (live ? (size_t(p) * a.x_rows + xr) * 256 : 0) + half * 16 + n * 128;
  const size_t xstep = size_t(2) * a.x_rows * 256;
  const int kb_x = (a.K + 31) / 32;
  const int8_t* wl[J];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int b = w * J + j;  // column tile, digit, half of its columns
    int g = 2 * gp + b / (2 * J);
    if (g >= a.groups) g = a.groups - 1;
    wl[j] = a.w + size_t(rt.e) * a.expert_bytes + size_t(g) * a.kb * (J * kTileBytes) +
            ((b >> 1) % J) * kTileBytes + (b & 1) * 1024 + (l & 31) * 32 + half * 16;
  }
  const int b0 = int(int64_t(kb_x) * slice / a.slices);
  const int b1 = int(int64_t(kb_x) * (slice + 1) / a.slices);
  // Registers for the k-blocks on their way to LDS (two ahead of the products)
  // and for the fragments of this step and the next.
  struct Staged {
    v4i x[4], w[J];
  };
  struct Frags {
    v4i x[8], w[2][J];
  };
  auto load_one = [&](Staged& g, int kb, int q) {
    kb = kb < b1 ? kb : b1 - 1;
    if (q < 4)
      g.x[q] = load16(xl + size_t(kb) * xstep + 32 * q);
    else
      g.w[q - 4] = load16(wl[q - 4] + size_t(kb) * (J * kTileBytes));
  };
  auto store_one = [&](const Staged& g, int kb, int q) {
    int8_t* at = lds[(kb - b0) & 1] + 16 * l;
    if (q < 4)  // zeros for a row that is not there and past the last k-block
      *reinterpret_cast<v4i*>(at + (m * 8 + n * 4 + q) * 1024) =
          live && kb < b1 ? g.x[q] : v4i{0, 0, 0, 0};
    else
      *reinterpret_cast<v4i*>(at + (16 + w * J + q - 4) * 1024) = g.w[q - 4];
  };
  auto read_one = [&](Frags& f, int kb, int q) {
    const int8_t* at = lds[(kb - b0) & 1] + 16 * l;
    if (q < 8)
      f.x[q] = *reinterpret_cast<const v4i*>(at + (m * 8 + q) * 1024);
    else
      f.w[(q - 8) / J][(q - 8) % J] = *reinterpret_cast<const v4i*>(
          at + (16 + (n * J + (q - 8) % J) * 2 + (q - 8) / J) * 1024);
  };
  constexpr int kMoves = 4 + J, kReads = 8 + 2 * J;
  auto load = [&](Staged& g, int kb) {
#pragma unroll
    for (int q = 0; q < kMoves; ++q) load_one(g, kb, q);
  };
  auto store = [&](const Staged& g, int kb) {
#pragma unroll
    for (int q = 0; q < kMoves; ++q) store_one(g, kb, q);
  };
  v16acc acc[2][8];
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int s = 0; s < 8; ++s)
#pragma unroll
      for (int q = 0; q < 16; ++q) acc[c][s][q] = 0;
  // Step kb (its fragments in f): between its products the next step's
  // fragments are read, the k-block after that is stored and another load of
  // two steps ahead is issued.  Buffer kb & 1 held this step's k-block, whose
  // readers passed the barrier at the end of the last step.
  auto step = [&](int kb, const Frags& f, Frags& next, Staged& g) {
    constexpr int kMfmas = 2 * (8 * J - J * (J - 1) / 2);
    constexpr int kChores = kReads + 2 * kMoves;
    int at = 0, done = 0;
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int i = 0; i + j < 8; ++i) {
          mfma_acc(acc[c][i + j], f.x[i], f.w[c][j]);
          ++at;
#pragma unroll
          for (; done < at * kChores / kMfmas; ++done) {
            if (done < kReads)
              read_one(next, kb + 1, done);
            else if (done < kReads + kMoves)
              store_one(g, kb + 2, done - kReads);
            else
              load_one(g, kb + 4, done - kReads - kMoves);
          }
        }
    __syncthreads();
  };
  // Steps in pairs; past the last k-block X is zeros.
  Staged ga, gb;
  Frags fa, fb;
  load(ga, b0);
  load(gb, b0 + 1);
  store(ga, b0);
  load(ga, b0 + 2);
  store(gb, b0 + 1);
  load(gb, b0 + 3);
  __syncthreads();
#pragma unroll
  for (int q = 0; q < kReads; ++q) read_one(fa, b0, q);
  __syncthreads();  // buffer 0 is stored to in the first step
  acc_settle(acc);
  for (int kb = b0; kb < b1; kb += 2) {
    step(kb, fa, fb, ga);
    step(kb + 1, fb, fa, gb);
  }
  acc_settle(acc);
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int col = (2 * gp + n) * kCols + 32 * c + (l & 31);
    if (col >= a.N) continue;
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      uint64_t v[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        v[q] = 0;
#pragma unroll
        for (int s = 0; s < 8; ++s) v[q] += uint64_t(int64_t(acc[c][s][4 * b + q])) << (8 * s);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = rt.begin + 16 * m + 2 * (2 * b + half) + h;
        if (row < rt.end) put_output(a, eh, slice, rt.e, row, col, v[h], v[2 + h]);
      }
    }
  }
}

// The epilogue's own launch, where k-slices have to be summed, an activation
// follows or the outputs go out as digits.  An activation's keystream binds a
// large one (two AES blocks an element for a cubic): then workgroups of 1024
// lanes with the four-table AES (128 KB of LDS), one a CU, else 512 lanes on
// two tables.
template <bool kWide>
struct EpiCfg {
  static constexpr int kBlock = 512;
  using Aes = AesLds2<32>;
  static constexpr int kTabWords = Aes::kSpanWords;
};
template <>
struct EpiCfg<true> {
  static constexpr int kBlock = 1024;
  using Aes = AesLds4;
  static constexpr int kTabWords = Aes::kWords;
};

// The ReLU's rows (c0, c1) at the masked open xh, both parties: c0 + c1 xh.
template <class Aes>
__device__ __forceinline__ void relu2(const ChainArgs& A, const ChainLds& L, const ChainKeyInfo& K,
                                      const Aes& aes, size_t i, uint64_t (&y)[2]) {
  const uint64_t xh = y[0] + y[1] + A.lut_mask;
  uint32_t st[2][4];
  int iv[2];
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const uint64_t xm = xh & K.m[p];
    int lo = 0, hi = A.intervals;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if ((L.cuts[p][mid] & K.m[p]) <= xm)
        lo = mid + 1;
      else
        hi = mid;
    }
    iv[p] = lo - 1 < 0 ? 0 : lo - 1;
    const uint64_t ctr = K.nonce[p] ^ (uint64_t(i) << 32) ^ (uint64_t(iv[p]) * 2);
    st[p][0] = uint32_t(ctr);
    st[p][1] = uint32_t(ctr >> 32);
    st[p][2] = st[p][3] = 0;
  }
  {
    uint32_t one[1][4] = {{st[0][0], st[0][1], st[0][2], st[0][3]}};
    const uint4* const rk[1] = {L.rk[0]};
    aes.template encrypt_n<1>(one, rk);
#pragma unroll
    for (int q = 0; q < 4; ++q) st[0][q] = one[0][q];
  }
  const bool shared = K.same_ks && iv[0] == iv[1];
  if (!shared) {
    uint32_t one[1][4] = {{st[1][0], st[1][1], st[1][2], st[1][3]}};
    const uint4* const rk[1] = {L.rk[1]};
    aes.template encrypt_n<1>(one, rk);
#pragma unroll
    for (int q = 0; q < 4; ++q) st[1][q] = one[0][q];
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q) st[1][q] = st[0][q];
  }
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const uint64_t k0 = uint64_t(st[p][0]) | uint64_t(st[p][1]) << 32;
    const uint64_t k1 = uint64_t(st[p][2]) | uint64_t(st[p][3]) << 32;
    const uint64_t* row = L.pay[p] + size_t(iv[p]) * 2;
    const uint64_t c0 = K.party[p] == 0 ? k0 : row[0] - k0;
    const uint64_t c1 = K.party[p] == 0 ? k1 : row[1] - k1;
    y[p] = c0 + c1 * xh;
  }
}

struct EpiArgs {
  LinArgs a;
  ChainArgs act;
};
static_assert(sizeof(EpiArgs) <= 4096, "kernel argument blocks must fit in 4 KB");

template <int kAct, bool kWide>
__global__ void __launch_bounds__(EpiCfg<kWide>::kBlock) linear_epilogue_kernel(EpiArgs A) {
  using Cfg = EpiCfg<kWide>;
  using EpiAes = typename Cfg::Aes;
  constexpr int kEpiBlock = Cfg::kBlock;
  const LinArgs& a = A.a;
  constexpr bool kLut = kAct != SUFHIP_ACT_NONE;
  constexpr int W = kAct == SUFHIP_ACT_CUBIC ? 4 : 2;
  __shared__ __align__(16) uint32_t tab[kLut ? Cfg::kTabWords : 4];
  __shared__ ChainLds L;
  __shared__ TruncHdr th[3][2];
  if constexpr (kLut) {
    typename EpiAes::template Filler<kEpiBlock> tf;
    ChainStager<kEpiBlock, 2> cs;
    tf.load(kTDev.v);
    cs.load(A.act, W);
    if constexpr (kAct == SUFHIP_ACT_CUBIC) {
      TruncHdrStager<3> hs;
      hs.load(A.act, 0);
      hs.store(th);
    }
    cs.store(A.act, W, L);
    tf.store(tab);
    __syncthreads();
    chain_compare(A.act, L);
    __syncthreads();
  }
  const EpiAes aes = EpiAes::make(tab);
  ChainKeyInfo K{};
  if constexpr (kLut) K = chain_key_info(A.act, L);
  const EpiHdrs eh = epi_hdrs(a.epi);
  const size_t mn = size_t(a.rows) * a.N;
  for (size_t i = size_t(blockIdx.x) * kEpiBlock + threadIdx.x; i < mn;
       i += size_t(gridDim.x) * kEpiBlock) {
    const int row = int(uint32_t(i) / uint32_t(a.N)), col = int(uint32_t(i) % uint32_t(a.N));
    const int e = expert_of(a, row);
    if (e < 0) continue;
    uint64_t y[2] = {0, 0}, open;
    if (a.slices > 1) {
      int z = 0;
      for (; z + 4 <= a.slices; z += 4) {  // a group's loads before its sums
        uint64_t v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = a.part[(size_t(z) * 2 + u) * mn + i];
#pragma unroll
        for (int u = 0; u < 8; ++u) y[u & 1] += v[u];
      }
      for (; z < a.slices; ++z) {
        y[0] += a.part[size_t(z) * 2 * mn + i];
        y[1] += a.part[(size_t(z) * 2 + 1) * mn + i];
      }
      if (a.bias) y[0] += uint64_t(a.bias[size_t(e) * a.N + col]);
      open = y[0] + y[1] + a.mask;
    } else {
      open = a.zhat[i];
    }
    if (a.epi.on) gate2(a.epi, eh, open, y);
    if constexpr (kAct == SUFHIP_ACT_RELU) relu2(A.act, L, K, aes, i, y);
    if constexpr (kAct == SUFHIP_ACT_CUBIC) {
      const Two x{{y[0], y[1]}};
      const Two o = chain_eval<SUFHIP_CHAIN_CUBIC, EpiAes>(
          A.act, L, K, aes, i, x, plain_loader<SUFHIP_CHAIN_CUBIC>{&A.act, i}, th);
      y[0] = o.v[0];
      y[1] = o.v[1];
    }
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      if (a.res.p[0]) y[p] += a.res.p[p][int64_t(row) * a.res.stride + col];
      if (a.out[0]) a.out[p][int64_t(row) * a.out_stride + col] = y[p];
      if (a.digits) put_digits(a.digits, size_t(a.rows), size_t(row), col, p, y[p]);
    }
    if (a.digits && col == a.N - 1) {  // up to the next multiple of 32
      for (int c = a.N; c % 32; ++c) {
        put_digits(a.digits, size_t(a.rows), size_t(row), c, 0, 0);
        put_digits(a.digits, size_t(a.rows), size_t(row), c, 1, 0);
      }
    }
  }
}

// x -> digits; a lane takes 16 neighbours of a row.
__global__ void __launch_bounds__(256)
    split_rows_kernel(Mat2 x, int rows, int cols, int8_t* digits) {
  const int per = (cols + 31) / 32 * 2;  // sixteens of a row
  const size_t items = size_t(2) * rows * per;
  for (size_t it = size_t(blockIdx.x) * 256 + threadIdx.x; it < items;
       it += size_t(gridDim.x) * 256) {
    const int h = int(it % per);
    const size_t row = it / per;  // p rows + r
    const int p = row >= size_t(rows) ? 1 : 0;
    const int c0 = 16 * h;
    const uint64_t* src = (p ? x.p[1] : x.p[0]) + int64_t(row - size_t(p) * rows) * x.stride + c0;
    u64x2u v[8];
    if (c0 + 16 <= cols) {
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] = *reinterpret_cast<const u64x2u*>(src + 2 * q);
    } else {
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        v[q][0] = c0 + 2 * q < cols ? src[2 * q] : 0;
        v[q][1] = c0 + 2 * q + 1 < cols ? src[2 * q + 1] : 0;
      }
    }
    v4i d[8];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint64_t f[4] = {v[2 * q][0], v[2 * q][1], v[2 * q + 1][0], v[2 * q + 1][1]};
      uint32_t o[8];
      digits_of4(f, o);
#pragma unroll
      for (int i = 0; i < 8; ++i) d[i][q] = int(o[i]);
    }
    int8_t* at = digits + digit_off(row, c0, size_t(rows));
#pragma unroll
    for (int i = 0; i < 8; ++i) *reinterpret_cast<v4i*>(at + 32 * i) = d[i];
  }
}

// W [experts][K][N] -> planes; a lane takes four neighbouring k of a column.
__global__ void __launch_bounds__(256)
    split_weights_kernel(const int64_t* W, int experts, int K, int N, int kb, int groups, int J,
                         int8_t* planes) {
  const size_t cols = size_t(groups) * kCols, quads = size_t(kb) * 8;
  const size_t items = size_t(experts) * quads * cols;
  for (size_t it = size_t(blockIdx.x) * 256 + threadIdx.x; it < items;
       it += size_t(gridDim.x) * 256) {
    const int n = int(it % cols);
    const size_t rest = it / cols;
    const int k = int(rest % quads) * 4;
    const size_t e = rest / quads;
    uint64_t v[4];
#pragma unroll
    for (int q = 0; q < 4; ++q)
      v[q] = n < N && k + q < K ? uint64_t(W[(e * K + k + q) * size_t(N) + n]) : 0;
    uint32_t d[8];
    digits_of4(v, d);
    int8_t* at = planes + ((e * groups + n / kCols) * kb + (k >> 5)) * size_t(J) * kTileBytes +
                 size_t(n % kCols) * 32 + (k & 31);
    for (int j = 0; j < J; ++j)
      *reinterpret_cast<uint32_t*>(at + size_t(j) * kTileBytes) = d[j];
  }
}

int device_cus() {
  int dev = 0, cus = 256;
  if (hipGetDevice(&dev) == hipSuccess)
    (void)hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev);
  return cus;
}

// How a call runs.
struct Plan {
  bool tile;       // linear_tile_kernel, else linear_skinny_kernel of t rows
  int t;
  int tiles;       // row tiles of the grid (an upper bound with experts)
  int col_tiles;
  int slices;
  bool epilogue;   // the epilogue's own launch
  size_t digits_bytes, words;  // the workspace: x's digits, sums or opens
};

bool extents_ok(int experts, int K, int N, int digits) {
  return experts >= 1 && experts <= 4096 && K >= 1 && K <= 65536 && N >= 1 && N <= kMaxRows &&
         digits >= 1 && digits <= 4 && size_t(digits) * size_t(K) < (size_t(1) << 17);
}

Plan plan_linear(const sufhip_linear2_args& g) {
  Plan p{};
  const int groups = (g.w.N + kCols - 1) / kCols;
  const int kb = (g.w.K + 63) / 64 * 2;
  const int experts = g.d_offsets ? g.w.experts : 1;
  const int each = (g.rows + experts - 1) / experts;  // rows of an expert, on average
  p.tile = each > 32;
  p.t = each <= 8 ? 16 : 32;
  const int per = p.tile ? kBigTok : p.t / 2;
  // Every expert may end inside a tile, and has one only if it has a row.
  p.tiles = g.d_offsets ? g.rows / per + (experts < g.rows ? experts : g.rows)
                        : (g.rows + per - 1) / per;
  const int cus = device_cus();
  p.col_tiles = (groups + 1) / 2;
  const int64_t wgs = int64_t(p.tiles) * p.col_tiles;
  const int most = p.tile ? kb / 8 : kb / 4;
  int64_t s = p.tile ? cus / wgs : (2 * cus + wgs - 1) / wgs;
  if (s > most) s = most;
  if (s > 16) s = 16;
  p.slices = s < 1 ? 1 : int(s);
  p.epilogue = p.slices > 1 || g.act != SUFHIP_ACT_NONE || g.out_digits.d_digits;
  p.digits_bytes =
      p.tile && !g.x_digits.d_digits ? sufhip_digits2_bytes(g.x_rows, g.w.K) : 0;
  const size_t mn = size_t(g.rows) * size_t(g.w.N);
  p.words = !p.epilogue ? 0 : (p.slices > 1 ? size_t(p.slices) * 2 * mn : mn);
  return p;
}

// The extents that a plan needs.
int check_extents(const sufhip_linear2_args& g, const char* what) {
  if (!extents_ok(g.w.experts, g.w.K, g.w.N, g.w.digits))
    return ff_fail(what, "needs 1 <= experts <= 4096, 1 <= K <= 65536, 1 <= N <= 2^24, digits in "
                         "[1, 4] and digits K < 2^17");
  if (g.rows < 0 || g.x_rows < 0 || g.rows > kMaxRows || g.x_rows > kMaxRows)
    return ff_fail(what, "rows and x_rows in [0, 2^24]");
  if (uint64_t(g.rows) * uint64_t(g.w.N) >= (uint64_t(1) << 31))
    return ff_fail(what, "rows N must stay below 2^31");
  return SUFHIP_OK;
}

template <int J>
void launch_skinny(const LinArgs& a, int t, unsigned grid, hipStream_t s) {
  if (t == 16) {
    if (a.xd)
      hipLaunchKernelGGL((linear_skinny_kernel<16, J, true>), dim3(grid), dim3(256), 0, s, a);
    else
      hipLaunchKernelGGL((linear_skinny_kernel<16, J, false>), dim3(grid), dim3(256), 0, s, a);
  } else {
    if (a.xd)
      hipLaunchKernelGGL((linear_skinny_kernel<32, J, true>), dim3(grid), dim3(256), 0, s, a);
    else
      hipLaunchKernelGGL((linear_skinny_kernel<32, J, false>), dim3(grid), dim3(256), 0, s, a);
  }
}

int launch_split(const Mat2& x, int rows, int cols, int8_t* digits, hipStream_t s) {
  const size_t items = size_t(2) * rows * ((cols + 31) / 32 * 2);
  size_t grid = (items + 255) / 256;
  if (grid > 8192) grid = 8192;
  hipLaunchKernelGGL(split_rows_kernel, dim3(unsigned(grid)), dim3(256), 0, s, x, rows, cols,
                     digits);
  return check_launch("split_rows_kernel");
}

}  // namespace
}  // namespace sufhip

using namespace sufhip;

extern "C" {

size_t sufhip_digits2_bytes(int rows, int cols) {
  if (rows < 1 || cols < 1 || rows > kMaxRows || cols > kMaxRows) return 0;
  return size_t((cols + 31) / 32) * 2 * size_t(rows) * 256;
}

int sufhip_digits2_split(const sufhip_matrix2* x, const sufhip_digits2* out, void* stream) {
  const char* what = "sufhip_digits2_split";
  SUFHIP_REQUIRE(x && out, "sufhip_digits2_split: null argument");
  if (out->rows == 0 || out->cols == 0) return SUFHIP_OK;
  if (sufhip_digits2_bytes(out->rows, out->cols) == 0 || !out->d_digits)
    return ff_fail(what, "rows and cols in [1, 2^24], and a buffer");
  if (int rc = digits2_of(*out, out->rows, out->cols, what, "out")) return rc;
  Mat2 m;
  if (int rc = mat2_of(*x, out->rows, out->cols, what, "x", &m)) return rc;
  for (int p = 0; p < 2; ++p)
    if (range_meets(out->d_digits, sufhip_digits2_bytes(out->rows, out->cols),
                    row_set(m, p, out->rows, out->cols)))
      return ff_fail(what, "out meets x");
  return launch_split(m, out->rows, out->cols, out->d_digits, as_stream(stream));
}

size_t sufhip_linear_planes_bytes(int experts, int K, int N, int digits) {
  if (!extents_ok(experts, K, N, digits)) return 0;
  return size_t(experts) * size_t((N + kCols - 1) / kCols) * size_t((K + 63) / 64 * 2) *
         size_t(digits) * kTileBytes;
}

int sufhip_linear_prepare(const int64_t* d_W, int experts, int K, int N, int digits,
                          int8_t* d_planes, void* stream) {
  const char* what = "sufhip_linear_prepare";
  if (!extents_ok(experts, K, N, digits))
    return ff_fail(what, "needs 1 <= experts <= 4096, 1 <= K <= 65536, 1 <= N <= 2^24, digits in "
                         "[1, 4] and digits K < 2^17");
  SUFHIP_REQUIRE(d_W && d_planes, "sufhip_linear_prepare: null pointer");
  SUFHIP_REQUIRE((reinterpret_cast<uintptr_t>(d_planes) & 15) == 0,
                 "sufhip_linear_prepare: planes must be 16-byte aligned");
  const int kb = (K + 63) / 64 * 2, groups = (N + kCols - 1) / kCols;
  const size_t items = size_t(experts) * kb * 8 * groups * kCols;
  size_t grid = (items + 255) / 256;
  if (grid > 65536) grid = 65536;
  hipLaunchKernelGGL(split_weights_kernel, dim3(unsigned(grid)), dim3(256), 0, as_stream(stream),
                     d_W, experts, K, N, kb, groups, digits, d_planes);
  return check_launch("split_weights_kernel");
}

size_t sufhip_linear2_work_bytes(const sufhip_linear2_args* args) {
  if (!args || check_extents(*args, "sufhip_linear2_work_bytes") != SUFHIP_OK) return 0;
  if (args->rows == 0 || args->x_rows == 0) return 0;
  const Plan p = plan_linear(*args);
  return p.digits_bytes + p.words * 8;
}

int sufhip_linear2(const sufhip_linear2_args* args, void* stream) {
  const char* what = "sufhip_linear2";
  SUFHIP_REQUIRE(args, "sufhip_linear2: null args");
  const sufhip_linear2_args& g = *args;
  if (int rc = check_extents(g, what)) return rc;
  if (g.rows == 0) return SUFHIP_OK;
  if (g.x_rows == 0) return ff_fail(what, "x has no rows");
  if (!g.w.d_planes || (reinterpret_cast<uintptr_t>(g.w.d_planes) & 15) != 0)
    return ff_fail(what, "the weights' planes are null or not 16-byte aligned");
  if (!g.d_offsets && g.w.experts > 1) return ff_fail(what, "several experts need d_offsets");
  if (!g.d_rows && g.rows > g.x_rows) return ff_fail(what, "more rows than x has need d_rows");
  LinArgs a{};
  a.x_rows = g.x_rows;
  a.rows = g.rows;
  a.K = g.w.K;
  a.N = g.w.N;
  a.kb = (g.w.K + 63) / 64 * 2;
  a.groups = (g.w.N + kCols - 1) / kCols;
  a.experts = g.w.experts;
  a.w = g.w.d_planes;
  a.expert_bytes = sufhip_linear_planes_bytes(1, g.w.K, g.w.N, g.w.digits);
  a.bias = g.w.d_bias;
  a.map = g.d_rows;
  a.offsets = g.d_offsets;
  a.mask = g.mask;
  if (g.x_digits.d_digits) {
    if (int rc = digits2_of(g.x_digits, g.x_rows, g.w.K, what, "x_digits")) return rc;
    a.xd = g.x_digits.d_digits;
  } else if (int rc = mat2_of(g.x, g.x_rows, g.w.K, what, "x", &a.x)) {
    return rc;
  }
  const size_t mn = size_t(g.rows) * size_t(g.w.N);
  if (g.trunc)
    if (int rc = gate_of(*g.trunc, mn, what, &a.epi)) return rc;
  ChainArgs act{};
  if (g.act == SUFHIP_ACT_RELU) {
    const sufhip_relu_key& k = g.relu;
    if (k.intervals < 1 || k.intervals > kChainMaxIntervals || !k.key[0] || !k.key[1] ||
        k.key_bytes != sufhip_interval_lut_key_bytes(k.intervals, 2) ||
        (reinterpret_cast<uintptr_t>(k.key[0]) & 7) != 0 ||
        (reinterpret_cast<uintptr_t>(k.key[1]) & 7) != 0)
      return ff_fail(what, "relu needs both keys, 8-byte aligned, of (intervals <= 64, 2 words)");
    act.lut[0] = k.key[0];
    act.lut[1] = k.key[1];
    act.intervals = k.intervals;
    act.lut_mask = k.mask;
    act.own_ks = keystream_per_party() ? 1u : 0u;
  } else if (g.act == SUFHIP_ACT_CUBIC) {
    if (!g.cubic || g.cubic->kind != SUFHIP_CHAIN_CUBIC || g.cubic->n != mn)
      return ff_fail(what, "cubic must be a SUFHIP_CHAIN_CUBIC chain with n = rows N");
    if (int rc = make_chain_args(*g.cubic, false, what, &act)) return rc;
    if (!act.plain)
      return ff_fail(what, "cubic's triples must be plain arrays, all of stride 1 or all of 3");
  } else if (g.act != SUFHIP_ACT_NONE) {
    return ff_fail(what, "unknown activation");
  }
  if (g.act != SUFHIP_ACT_NONE && !g.trunc) return ff_fail(what, "an activation needs trunc");
  if ((g.residual.p[0] == nullptr) != (g.residual.p[1] == nullptr))
    return ff_fail(what, "one share of the residual is missing");
  if (g.residual.p[0])
    if (int rc = mat2_of(g.residual, g.rows, g.w.N, what, "residual", &a.res)) return rc;
  if ((g.out[0] == nullptr) != (g.out[1] == nullptr))
    return ff_fail(what, "give both share outputs or neither");
  if (!g.out[0] && !g.out_digits.d_digits) return ff_fail(what, "no output");
  if (g.out_digits.d_digits)
    if (int rc = digits2_of(g.out_digits, g.rows, g.w.N, what, "out_digits")) return rc;
  a.digits = g.out_digits.d_digits;
  a.out_stride = g.out_stride;
  const Plan plan = plan_linear(g);
  const size_t need = plan.digits_bytes + plan.words * 8;
  if (need && (!g.d_work || (reinterpret_cast<uintptr_t>(g.d_work) & 15) != 0 ||
               g.work_bytes < need))
    return ff_fail(what, "the workspace is null, not 16-byte aligned or too small");
  const size_t dig_bytes = g.out_digits.d_digits ? sufhip_digits2_bytes(g.rows, g.w.N) : 0;
  const size_t xd_bytes = a.xd ? sufhip_digits2_bytes(g.x_rows, g.w.K) : 0;
  if (g.out[0]) {
    if (g.out_stride < 0 || rows_overlap(g.out_stride, g.rows, g.w.N))
      return ff_fail(what, "output rows overlap");
    RowSet o[2];
    for (int p = 0; p < 2; ++p) {
      a.out[p] = g.out[p];
      o[p] = {g.out[p], g.out_stride, g.rows, g.w.N};
    }
    if (sets_meet(o[0], o[1])) return ff_fail(what, "the two shares of out meet");
    for (int p = 0; p < 2; ++p) {
      for (int q = 0; q < 2; ++q) {
        if (!a.xd && sets_meet(o[p], row_set(a.x, q, g.x_rows, g.w.K)))
          return ff_fail(what, "out meets x");
        if (a.res.p[0]) {
          const RowSet r = row_set(a.res, q, g.rows, g.w.N);
          if (sets_meet(o[p], r) && !(p == q && same_set(o[p], r)))
            return ff_fail(what, "out meets the residual without being it");
        }
      }
      if ((a.xd && range_meets(a.xd, xd_bytes, o[p])) ||
          (need && range_meets(g.d_work, need, o[p])) ||
          (dig_bytes && range_meets(g.out_digits.d_digits, dig_bytes, o[p])))
        return ff_fail(what, "out meets a buffer of digits or the workspace");
    }
  }
  auto bytes_meet = [](const void* x, size_t nx, const void* y, size_t ny) {
    const char *cx = static_cast<const char*>(x), *cy = static_cast<const char*>(y);
    return nx && ny && cx < cy + ny && cy < cx + nx;
  };
  if (dig_bytes) {
    const void* d = g.out_digits.d_digits;
    bool bad = bytes_meet(d, dig_bytes, a.xd, xd_bytes) ||
               bytes_meet(d, dig_bytes, g.d_work, need);
    for (int q = 0; q < 2; ++q)
      bad = bad || (!a.xd && range_meets(d, dig_bytes, row_set(a.x, q, g.x_rows, g.w.K))) ||
            (a.res.p[0] && range_meets(d, dig_bytes, row_set(a.res, q, g.rows, g.w.N)));
    if (bad) return ff_fail(what, "out_digits meets an input or the workspace");
  }
  hipStream_t s = as_stream(stream);
  int8_t* work = static_cast<int8_t*>(g.d_work);
  if (plan.digits_bytes) {
    if (int rc = launch_split(a.x, g.x_rows, g.w.K, work, s)) return rc;
    a.xd = work;
  }
  uint64_t* words = reinterpret_cast<uint64_t*>(work + plan.digits_bytes);
  a.tiles = plan.tiles;
  a.slices = plan.slices;
  if (plan.slices > 1)
    a.part = words;
  else if (plan.epilogue)
    a.zhat = words;
  if (plan.tile) {
    const unsigned grid = unsigned(int64_t(plan.tiles) * plan.slices * plan.col_tiles);
    switch (g.w.digits) {
      case 1: hipLaunchKernelGGL(linear_tile_kernel<1>, dim3(grid), dim3(256), 0, s, a); break;
      case 2: hipLaunchKernelGGL(linear_tile_kernel<2>, dim3(grid), dim3(256), 0, s, a); break;
      case 3: hipLaunchKernelGGL(linear_tile_kernel<3>, dim3(grid), dim3(256), 0, s, a); break;
      default: hipLaunchKernelGGL(linear_tile_kernel<4>, dim3(grid), dim3(256), 0, s, a); break;
    }
    if (int rc = check_launch("linear_tile_kernel")) return rc;
  } else {
    const unsigned grid = unsigned(int64_t(plan.tiles) * plan.slices * plan.col_tiles);
    switch (g.w.digits) {
      case 1: launch_skinny<1>(a, plan.t, grid, s); break;
      case 2: launch_skinny<2>(a, plan.t, grid, s); break;
      case 3: launch_skinny<3>(a, plan.t, grid, s); break;
      default: launch_skinny<4>(a, plan.t, grid, s); break;
    }
    if (int rc = check_launch("linear_skinny_kernel")) return rc;
  }
  if (!plan.epilogue) return SUFHIP_OK;
  const EpiArgs e{a, act};
  const size_t cus = size_t(device_cus());
  const bool wide = g.act == SUFHIP_ACT_CUBIC && mn >= 2 * cus * EpiCfg<true>::kBlock;
  const size_t block = wide ? EpiCfg<true>::kBlock : EpiCfg<false>::kBlock;
  size_t grid = (mn + block - 1) / block;
  const size_t cap = cus * (wide ? 1 : (g.act == SUFHIP_ACT_NONE ? 4 : 2));
  if (grid > cap) grid = cap;
  const dim3 gd{unsigned(grid)}, bd{unsigned(block)};
  if (g.act == SUFHIP_ACT_RELU)
    hipLaunchKernelGGL((linear_epilogue_kernel<SUFHIP_ACT_RELU, false>), gd, bd, 0, s, e);
  else if (g.act == SUFHIP_ACT_CUBIC && wide)
    hipLaunchKernelGGL((linear_epilogue_kernel<SUFHIP_ACT_CUBIC, true>), gd, bd, 0, s, e);
  else if (g.act == SUFHIP_ACT_CUBIC)
    hipLaunchKernelGGL((linear_epilogue_kernel<SUFHIP_ACT_CUBIC, false>), gd, bd, 0, s, e);
  else
    hipLaunchKernelGGL((linear_epilogue_kernel<SUFHIP_ACT_NONE, false>), gd, bd, 0, s, e);
  return check_launch("linear_epilogue_kernel");
}

}  // extern "C"
