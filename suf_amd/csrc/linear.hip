// Share x public weight for both parties and any number of rows, dense or
// grouped by expert, with the bias, the truncation, an activation and a
// residual in its epilogue (sufhip_linear2), on the int8 matrix cores (gfx950
// v_mfma_i32_16x16x64_i8), exact mod 2^64.
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
#include "walk_device.hpp"

namespace sufhip {
namespace {

typedef int v4acc __attribute__((ext_vector_type(4)));
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
  int tiles, cols, slices;
  // For the epilogue's launch, one of them:
  uint64_t* part;  // both shares [slices][2][rows][N], of several k-slices or without a gate
  uint64_t* zhat;  // the masked opens [rows][N]
  uint64_t mask;
  TruncEpi epi;
  Mat2 res;
  uint64_t* out[2];
  int64_t out_stride;
  int8_t* digits;  // the outputs as digits (the epilogue's launch)
};

// The key-only walks that a launch does beside its own work, in its first
// `groups` workgroups (a multiple of 8, so that the others' order over the XCDs
// stays).
constexpr int kLinWalks = 8;
struct LinWalk {
  WalkJobs<kLinWalks> jobs;
  int groups;
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

constexpr int kTok = 8;  // rows of a row tile

// Row tile number ti: its expert and rows.  Every lane of the
// wave takes part; experts are counted 64 at a time.
struct RowTile {
  int e, begin, end;
};
__device__ __forceinline__ RowTile row_tile(const LinArgs& a, int ti) {
  if (!a.offsets) {
    const int begin = ti * kTok;
    const int end = begin + kTok < a.rows ? begin + kTok : a.rows;
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
    const int n = (hi - lo + kTok - 1) / kTok;
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
      const int begin = flo + (ti - first) * kTok;
      return {e0 + f, begin, begin + kTok < fhi ? begin + kTok : fhi};
    }
    base += __shfl(incl, 63, 64);
  }
  return {-1, 0, 0};
}

// Both shares of output (row, col) as the product leaves them: for the
// epilogue's launch, or with bias, truncation and residual.
__device__ __forceinline__ void put_output(const LinArgs& a, const EpiHdrs& eh, int slice, int e,
                                           int row, int col, uint64_t y0, uint64_t y1) {
  const size_t i = size_t(row) * a.N + col;
  if (a.part) {
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

// The order of the tiles.  Workgroups are dealt round-robin to the 8 XCDs, each
// with an L2 of its own, so an XCD takes a contiguous eighth of the order; and
// the order goes over 1024 columns (kPanel tiles), then the row tiles, then the
// next columns: the sixty workgroups that an XCD runs at once then share some row
// tiles of X and 1024 columns of W, instead of one side alone being read again
// by each (1000 x 2048 x 1024: 288 MB beyond the L2s, 66 us with tiles of 128
// columns row by row; 512 or 2048 columns at a time: within 2 %).
struct TileId {
  int row, col, slice;
};
template <int kPanel>
__device__ __forceinline__ TileId tile_id(const LinArgs& a, int id, int total) {
  const int each = total / 8, more = total % 8, x = id % 8;
  id = x * each + (x < more ? x : more) + id / 8;
  const int cols = a.cols;
  const int plane = a.tiles * cols, slice = id / plane;
  id -= slice * plane;
  const int panel = id / (kPanel * a.tiles), left = cols - kPanel * panel;
  const int wide = left < kPanel ? left : kPanel;
  id -= kPanel * a.tiles * panel;
  return {id / wide, kPanel * panel + id % wide, slice};
}

// A workgroup of four waves takes a row tile (8 tokens of both parties), 64
// kFrags columns, 16 kFrags a wave, and one k-slice.  W goes straight into
// registers; X's digits, which the four waves share, are formed on the way into
// LDS (or come as digits), 64 k at a time, the next chunk's loads in flight
// under this one's products.
//
// Few rows: the stream of W bounds it (logits of one row, 2048 x 32000, 131 MB
// in 27 us).  Many rows: 1000 x 2048 x 1024 takes 56 us from digits, 2.25 POP/s
// of int8, and 60 from shares; with the matrix instructions alone it would be
// 37, and X's way costs 7, W's loads 5, the fragments' reads from LDS 10.  A
// deeper ring, larger tiles (32 tokens x 128 columns, 256 accumulators a wave:
// 72 us) and fragments read a step ahead (57 us) gain nothing.
constexpr int kDepth = 2;  // chunks on their way
template <int kFrags, int J, bool kDigits, bool kWalk>
__global__ void __launch_bounds__(256, 2) linear_product_kernel(LinArgs a, LinWalk wk) {
  if constexpr (kWalk) {
    if (int(blockIdx.x) < wk.groups) {
      hosted_walk_role<kLinWalks, false>(wk.jobs, blockIdx.x * 256 + threadIdx.x);
      return;
    }
  }
  const int groups = kWalk ? wk.groups : 0;
  // [digit][slot] of 16 k.  Row r's sixteen number kk is slot 16 kk + (r + 4 kk)
  // % 16: a wave's dword writes (four rows, four sixteens) and its fragment
  // reads then take every bank once.
  __shared__ __align__(16) int8_t lds[2][8 * 1024];
  const int l = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
  constexpr int kPanel = kFrags > 2 ? 4 : 8;
  const TileId at = tile_id<kPanel>(a, int(blockIdx.x) - groups, int(gridDim.x) - groups);
  const int slice = at.slice, c0 = (at.col * 4 + w) * 16 * kFrags;
  const RowTile rt = row_tile(a, at.row);
  if (rt.e < 0 || rt.begin >= rt.end) return;  // the whole workgroup
  const EpiHdrs eh = epi_hdrs(a.epi);
  // The row that this thread brings to LDS: four words of it from kq on, or
  // (digits) two pieces of 16 bytes.
  const int r = kDigits ? l % 16 : int(threadIdx.x) / 16;
  const int kq = int(threadIdx.x) % 16 * 4;
  const int slot = ((l & 48) + ((l + (l >> 4) * 4) & 15)) * 16;  // of this lane's fragment
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
                     (c0 % kCols) * 32 + (l >> 5) * (J * kTileBytes) + (l & 15) * 32 +
                     ((l >> 4) & 1) * 16;
  const int chunks = a.kb / 2;
  const int q0 = int(int64_t(chunks) * slice / a.slices);
  const int q1 = int(int64_t(chunks) * (slice + 1) / a.slices);
  // W on its way, until its products: kDepth chunks, or (four fragments, whose
  // registers are many) one, a fragment's loads leaving behind its products.
  constexpr int kWays = kFrags > 2 ? 1 : kDepth;
  v4i wr[kWays][kFrags][J];
  auto load_w = [&](int u, int c, int q) {
    if (q >= q1) return;
#pragma unroll
    for (int j = 0; j < J; ++j)
      wr[u][c][j] = load16(wl + size_t(q) * (2 * J * kTileBytes) + j * kTileBytes + c * 512);
  };
  // X on its way, until its place in LDS.
  struct Chunk {
    u64x2u w[kDigits ? 1 : 2];
    v4i d[kDigits ? 2 : 1];
  };
  auto load_x = [&](Chunk& k, int q) {
    if (q >= q1) return;
    if constexpr (kDigits) {
      // Digits w and w + 4 at this lane's place in the fragment.
      const int kb = 2 * q + (l >> 5);
      k.d[0] = k.d[1] = v4i{0, 0, 0, 0};
      if (live && 32 * kb < a.K) {
        const int8_t* at = drow + size_t(kb) * dstep + 16 * ((l >> 4) & 1) + 32 * w;
        k.d[0] = load16(at);
        k.d[1] = load16(at + 128);
      }
    } else {
      const uint64_t* row = xrow + 64 * q;
      const int left = a.K - 64 * q - kq;
      k.w[0] = k.w[1] = u64x2u{0, 0};
      if (live && left >= 4) {
        k.w[0] = *reinterpret_cast<const u64x2u*>(row);
        k.w[1] = *reinterpret_cast<const u64x2u*>(row + 2);
      } else if (live) {
        if (left > 0) k.w[0][0] = row[0];
        if (left > 1) k.w[0][1] = row[1];
        if (left > 2) k.w[1][0] = row[2];
      }
    }
  };
  auto store_x = [&](const Chunk& k, int buf) {
    if constexpr (kDigits) {
      *reinterpret_cast<v4i*>(&lds[buf][w * 1024 + slot]) = k.d[0];
      *reinterpret_cast<v4i*>(&lds[buf][(w + 4) * 1024 + slot]) = k.d[1];
    } else {
      int8_t* at = &lds[buf][(kq & 48) * 16 + ((r + (kq >> 4) * 4) & 15) * 16 + (kq & 15)];
      const uint64_t v[4] = {k.w[0][0], k.w[0][1], k.w[1][0], k.w[1][1]};
      uint32_t d[8];
      digits_of4(v, d);
#pragma unroll
      for (int i = 0; i < 8; ++i) *reinterpret_cast<uint32_t*>(at + 1024 * i) = d[i];
    }
  };
  v4acc acc[kFrags][8];
#pragma unroll
  for (int c = 0; c < kFrags; ++c)
#pragma unroll
    for (int s = 0; s < 8; ++s)
#pragma unroll
      for (int q = 0; q < 4; ++q) acc[c][s][q] = 0;
  // Chunk q, its W in wr[u], its X in LDS; W of chunk q + kWays follows.
  auto products = [&](int u, int buf, int q) {
    v4i d[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) d[i] = *reinterpret_cast<const v4i*>(&lds[buf][i * 1024 + slot]);
#pragma unroll
    for (int c = 0; c < kFrags; ++c) {
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int i = 0; i + j < 8; ++i)
          acc[c][i + j] =
              __builtin_amdgcn_mfma_i32_16x16x64_i8(d[i], wr[u][c][j], acc[c][i + j], 0, 0, 0);
      if (kWays == 1) load_w(u, c, q + 1);
    }
    if (kWays > 1) {
#pragma unroll
      for (int c = 0; c < kFrags; ++c) load_w(u, c, q + kWays);
    }
  };
  // Chunk q's X lies in ring[(q - q0) % kDepth], then in LDS, a step ahead of
  // its products.
  Chunk ring[kDepth];
#pragma unroll
  for (int u = 0; u < kDepth; ++u) {
    if (u < kWays) {
#pragma unroll
      for (int c = 0; c < kFrags; ++c) load_w(u, c, q0 + u);
    }
    load_x(ring[u], q0 + u);
  }
  store_x(ring[0], 0);
  load_x(ring[0], q0 + kDepth);
  __syncthreads();
  for (int q = q0; q < q1; q += kDepth) {
#pragma unroll
    for (int u = 0; u < kDepth; ++u) {
      if (q + u < q1) {
        Chunk& next = ring[(u + 1) % kDepth];
        const int buf = (q + u - q0) & 1;
        products(u % kWays, buf, q + u);
        store_x(next, buf ^ 1);
        load_x(next, q + u + 1 + kDepth);
        __syncthreads();
      }
    }
  }
#pragma unroll
  for (int c = 0; c < kFrags; ++c) {
    const int col = c0 + 16 * c + l % 16;
    if (col >= a.N) continue;
    uint64_t v[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      v[q] = 0;
#pragma unroll
      for (int s = 0; s < 8; ++s) v[q] += uint64_t(int64_t(acc[c][s][q])) << (8 * s);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = rt.begin + 2 * (l / 16) + h;
      if (row < rt.end) put_output(a, eh, slice, rt.e, row, col, v[h], v[2 + h]);
    }
  }
}

// The epilogue's own launch, where k-slices have to be summed, an activation
// follows or the outputs go out as digits.  An activation's keystream binds a
// large one (two AES blocks an element for a cubic): workgroups of 1024 lanes
// with the four-table AES (128 KB of LDS), one a CU.  A small one waits for its
// tables first: 256 lanes and one table of 16 copies (16 KB).
enum { kEpiSmall = 0, kEpiMid = 1, kEpiWide = 2 };
template <int kSize>
struct EpiCfg {  // kEpiMid
  static constexpr int kBlock = 512;
  using Aes = AesLds2<32>;
  static constexpr int kTabWords = Aes::kSpanWords;
  template <class Cs, class Args>
  __device__ __forceinline__ static Aes stage(uint32_t* tab, const Args& A, int W, ChainLds& L) {
    typename Aes::template Filler<kBlock> tf;
    Cs cs;
    tf.load(kTDev.v);
    cs.load(A, W);
    cs.store(A, W, L);
    tf.store(tab);
    return Aes::make(tab);
  }
};
template <>
struct EpiCfg<kEpiWide> {
  static constexpr int kBlock = 1024;
  using Aes = AesLds4;
  static constexpr int kTabWords = Aes::kWords;
  template <class Cs, class Args>
  __device__ __forceinline__ static Aes stage(uint32_t* tab, const Args& A, int W, ChainLds& L) {
    typename Aes::template Filler<kBlock> tf;
    Cs cs;
    tf.load(kTDev.v);
    cs.load(A, W);
    cs.store(A, W, L);
    tf.store(tab);
    return Aes::make(tab);
  }
};
template <>
struct EpiCfg<kEpiSmall> {
  static constexpr int kBlock = 256;
  using Aes = AesLds<16>;
  static constexpr int kTabWords = 256 * 16;
  template <class Cs, class Args>
  __device__ __forceinline__ static Aes stage(uint32_t* tab, const Args& A, int W, ChainLds& L) {
    Cs cs;
    cs.load(A, W);
    fill_ttable<16>(tab, kTDev.v);
    cs.store(A, W, L);
    return Aes{tab, uint32_t(threadIdx.x) % 16};
  }
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

template <int kAct, int kSize>
__global__ void __launch_bounds__(EpiCfg<kSize>::kBlock) linear_epilogue_kernel(EpiArgs A) {
  using Cfg = EpiCfg<kSize>;
  using EpiAes = typename Cfg::Aes;
  constexpr int kEpiBlock = Cfg::kBlock;
  const LinArgs& a = A.a;
  constexpr bool kLut = kAct != SUFHIP_ACT_NONE;
  constexpr int W = kAct == SUFHIP_ACT_CUBIC ? 4 : 2;
  __shared__ __align__(16) uint32_t tab[kLut ? Cfg::kTabWords : 4];
  __shared__ ChainLds L;
  __shared__ TruncHdr th[3][2];
  std::conditional_t<kLut, EpiAes, int> aes;
  if constexpr (kLut) {
    if constexpr (kAct == SUFHIP_ACT_CUBIC) {
      TruncHdrStager<3> hs;
      hs.load(A.act, 0);
      hs.store(th);
    }
    aes = Cfg::template stage<ChainStager<kEpiBlock, 2>>(tab, A.act, W, L);
    __syncthreads();
    chain_compare(A.act, L);
    __syncthreads();
  }
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
    if (a.part) {
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
  bool wide;       // 256 columns a workgroup, else 128
  int tiles;       // row tiles of the grid (an upper bound with experts)
  int col_tiles;
  int slices;
  bool epilogue;   // the epilogue's own launch
  bool walk;       // the walks beside the product
  bool shares;     // the epilogue is handed shares, of each slice, else opens
  size_t words;    // of the workspace, which holds them
};

bool extents_ok(int experts, int K, int N, int digits) {
  return experts >= 1 && experts <= 4096 && K >= 1 && K <= 65536 && N >= 1 && N <= kMaxRows &&
         digits >= 1 && digits <= 4 && size_t(digits) * size_t(K) < (size_t(1) << 17);
}

Plan plan_linear(const sufhip_linear2_args& g) {
  Plan p{};
  // Every expert may end inside a tile, and has one only if it has a row.
  const int experts = g.w.experts < g.rows ? g.w.experts : g.rows;
  // 256 columns a workgroup read X's digits from LDS half as often, where there
  // are workgroups enough: 1000 x 2048 x 1024 (500 of them) 56 us against 67, 400
  // x 2048 x 2048 (400) 52 against 65, 256 x 768 x 2304 (288) 24 against 21; by
  // expert, whose tiles are ragged, 2000 rows x 1024 x 2048 of 16 (2000) 135
  // against 145, 1000 rows (1000) 76 either way, 500 rows 50 against 44.  With
  // three digits of W the sums do not fit the registers.
  const int64_t full = int64_t(g.rows / kTok) * ((g.w.N + 255) / 256);
  p.wide = g.w.digits <= 2 && 2 * full >= (g.d_offsets ? 9 : 3) * int64_t(device_cus());
  p.tiles = g.d_offsets ? g.rows / kTok + experts : (g.rows + kTok - 1) / kTok;
  p.col_tiles = p.wide ? (g.w.N + 255) / 256 : (g.w.N + 127) / 128;
  // k-slices up to two workgroups a CU, of three chunks at least: one row of
  // 768 x 2304 8.4 us with 4, 10.5 with 1; 8 x 4096 x 4096 16.9 with 8, 20.7
  // with 4, 18.4 with 16; 64 x 4096 x 4096 38.8 with 2, 50.2 with 1, 43 with 4.
  const int64_t wgs = int64_t(p.tiles) * p.col_tiles;
  int64_t s = 2 * int64_t(device_cus()) / wgs;
  const int most = (g.w.K + 63) / 64 / 3;
  if (s > most) s = most;
  if (s > 8) s = 8;
  p.slices = s < 1 ? 1 : int(s);
  p.epilogue = p.slices > 1 || g.act != SUFHIP_ACT_NONE || g.out_digits.d_digits;
  // Walks beside the product where its workgroups leave room, one round of the
  // chip, and the epilogue's launch that evaluates the gates follows anyway or
  // has little to do.  (One gate's walks alone take 13 us: logits of one token
  // 42 -> 33 us.  Beside as many workgroups of 256 columns, with a launch for a
  // million outputs of its own, 85 us against 73.)
  const size_t mn = size_t(g.rows) * size_t(g.w.N);
  p.walk = g.walk_count > 0 && g.walk_count <= kLinWalks && !p.wide &&
           wgs * p.slices <= 2 * device_cus() && (p.epilogue || mn <= (size_t(1) << 17));
  p.epilogue = p.epilogue || p.walk;
  // Without a gate nothing is opened: a party's output is its own share.
  p.shares = p.slices > 1 || !g.trunc;
  p.words = !p.epilogue ? 0 : (p.shares ? size_t(p.slices) * 2 * mn : mn);
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

template <int kFrags, int J>
void launch_tiles(const LinArgs& a, const LinWalk& w, unsigned wgs, hipStream_t s) {
  const dim3 grid(wgs + unsigned(w.groups)), block(256);
  if (a.xd && w.groups)
    hipLaunchKernelGGL((linear_product_kernel<kFrags, J, true, true>), grid, block, 0, s, a, w);
  else if (a.xd)
    hipLaunchKernelGGL((linear_product_kernel<kFrags, J, true, false>), grid, block, 0, s, a, w);
  else if (w.groups)
    hipLaunchKernelGGL((linear_product_kernel<kFrags, J, false, true>), grid, block, 0, s, a, w);
  else
    hipLaunchKernelGGL((linear_product_kernel<kFrags, J, false, false>), grid, block, 0, s, a, w);
}

template <int J>
void launch_product(const LinArgs& a, const LinWalk& w, bool wide, unsigned wgs, hipStream_t s) {
  if constexpr (J <= 2) {
    if (wide) return launch_tiles<4, J>(a, w, wgs, s);
  }
  launch_tiles<2, J>(a, w, wgs, s);
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
  if (int rc = mat2_of(*x, out->rows, what, "x", &m)) return rc;
  for (int p = 0; p < 2; ++p)
    if (range_meets(out->d_digits, sufhip_digits2_bytes(out->rows, out->cols),
                    row_set(m, p, out->rows, out->cols)))
      return ff_fail(what, "out meets x");
  const size_t items = size_t(2) * out->rows * ((out->cols + 31) / 32 * 2);
  size_t grid = (items + 255) / 256;
  if (grid > 8192) grid = 8192;
  hipLaunchKernelGGL(split_rows_kernel, dim3(unsigned(grid)), dim3(256), 0, as_stream(stream), m,
                     out->rows, out->cols, out->d_digits);
  return check_launch("split_rows_kernel");
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
  return plan_linear(*args).words * 8;
}

int sufhip_linear2(const sufhip_linear2_args* args, void* stream) {
  const char* what = "sufhip_linear2";
  SUFHIP_REQUIRE(args, "sufhip_linear2: null args");
  const sufhip_linear2_args& g = *args;
  if (int rc = check_extents(g, what)) return rc;
  if (g.walk_count < 0 || (g.walk_count > 0 && (!g.walk_jobs || !g.walk_prg_state)))
    return ff_fail(what, "walk_jobs and walk_prg_state are needed for walk_count jobs");
  if (g.rows == 0)  // the walks may be other operators' gates'
    return g.walk_count > 0
             ? sufhip_trunc_prepare_batch(g.walk_prg_state, g.walk_jobs, g.walk_count, stream)
             : SUFHIP_OK;
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
  } else if (int rc = mat2_of(g.x, g.x_rows, what, "x", &a.x)) {
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
    if (int rc = mat2_of(g.residual, g.rows, what, "residual", &a.res)) return rc;
  if ((g.out[0] == nullptr) != (g.out[1] == nullptr))
    return ff_fail(what, "give both share outputs or neither");
  if (!g.out[0] && !g.out_digits.d_digits) return ff_fail(what, "no output");
  if (g.out_digits.d_digits)
    if (int rc = digits2_of(g.out_digits, g.rows, g.w.N, what, "out_digits")) return rc;
  a.digits = g.out_digits.d_digits;
  a.out_stride = g.out_stride;
  const Plan plan = plan_linear(g);
  const uint64_t tiles = uint64_t(plan.tiles) * plan.slices * plan.col_tiles;
  if (tiles >= (uint64_t(1) << 24) - 4096)  // a launch holds 2^32 lanes
    return ff_fail(what, "more than 2^24 tiles of 8 rows and 128 or 256 columns");
  const size_t need = plan.words * 8;
  if (need && (!g.d_work || (reinterpret_cast<uintptr_t>(g.d_work) & 15) != 0 ||
               g.work_bytes < need))
    return ff_fail(what, "the workspace is null, not 16-byte aligned or too small");
  // Nothing that the call writes meets what it reads, but for out as the
  // residual itself.
  const Range xd{a.xd, a.xd ? sufhip_digits2_bytes(g.x_rows, g.w.K) : 0};
  const Range outd{a.digits, a.digits ? sufhip_digits2_bytes(g.rows, g.w.N) : 0};
  const Range work{g.d_work, need};
  const Range reads[5] = {
      {g.w.d_planes, sufhip_linear_planes_bytes(g.w.experts, g.w.K, g.w.N, g.w.digits)},
      {g.w.d_bias, size_t(g.w.experts) * g.w.N * 8},
      {g.d_rows, size_t(g.rows) * 4},
      {g.d_offsets, (size_t(g.w.experts) + 1) * 4},
      xd};
  RowSet x[2], res[2];
  for (int q = 0; q < 2; ++q) {
    x[q] = row_set(a.x, q, a.xd ? 0 : g.x_rows, g.w.K);
    res[q] = row_set(a.res, q, a.res.p[0] ? g.rows : 0, g.w.N);
  }
  for (const Range& r : reads)
    if (ranges_meet(outd, r) || ranges_meet(work, r))
      return ff_fail(what, "out_digits or the workspace meets an input");
  if (ranges_meet(outd, work)) return ff_fail(what, "out_digits meets the workspace");
  Material keys;
  keys.gate(a.epi);
  if (g.act == SUFHIP_ACT_RELU)
    for (int p = 0; p < 2; ++p) keys.add(g.relu.key[p], g.relu.key_bytes);
  if (g.act == SUFHIP_ACT_CUBIC)
    keys.chain(act, chain_products<SUFHIP_CHAIN_CUBIC>(), g.cubic->lut_key_bytes);
  if (keys.meets(outd) || keys.meets(work))
    return ff_fail(what, "out_digits or the workspace meets a gate, a LUT or a triple");
  for (int q = 0; q < 2; ++q)
    for (const RowSet* in : {&x[q], &res[q]})
      if (range_meets(outd, *in) || range_meets(work, *in))
        return ff_fail(what, "out_digits or the workspace meets an input");
  if (g.out[0]) {
    if (bad_out_stride(g.out_stride, g.rows, g.w.N))
      return ff_fail(what, "output rows overlap, or lie more than 2^35 apart");
    RowSet o[2];
    for (int p = 0; p < 2; ++p) {
      a.out[p] = g.out[p];
      o[p] = {g.out[p], g.out_stride, g.rows, g.w.N};
    }
    if (sets_meet(o[0], o[1])) return ff_fail(what, "the two shares of out meet");
    for (int p = 0; p < 2; ++p) {
      for (int q = 0; q < 2; ++q) {
        if (sets_meet(o[p], x[q])) return ff_fail(what, "out meets x");
        if (sets_meet(o[p], res[q]) && !(p == q && same_set(o[p], res[q])))
          return ff_fail(what, "out meets the residual without being it");
      }
      for (const Range& r : reads)
        if (range_meets(r, o[p])) return ff_fail(what, "out meets an input");
      if (keys.meets(o[p])) return ff_fail(what, "out meets a gate, a LUT or a triple");
      if (range_meets(outd, o[p]) || range_meets(work, o[p]))
        return ff_fail(what, "out meets out_digits or the workspace");
    }
  }
  hipStream_t s = as_stream(stream);
  LinWalk w{};
  if (plan.walk) {  // room for them: a workgroup a CU
    size_t lanes = 0;
    if (int rc = plan_hosted_walk(g.walk_prg_state, g.walk_jobs, g.walk_count,
                                  size_t(device_cus()) * 256, stream, what, w.jobs, &lanes))
      return rc;
    w.groups = int((lanes + 256 * 8 - 1) / (256 * 8)) * 8;
  } else if (g.walk_count > 0) {
    if (int rc = sufhip_trunc_prepare_batch(g.walk_prg_state, g.walk_jobs, g.walk_count, stream))
      return rc;
  }
  uint64_t* words = static_cast<uint64_t*>(g.d_work);
  a.tiles = plan.tiles;
  a.cols = plan.col_tiles;
  a.slices = plan.slices;
  if (plan.epilogue) (plan.shares ? a.part : a.zhat) = words;
  const unsigned wgs = unsigned(tiles);
  switch (g.w.digits) {
    case 1: launch_product<1>(a, w, plan.wide, wgs, s); break;
    case 2: launch_product<2>(a, w, plan.wide, wgs, s); break;
    case 3: launch_product<3>(a, w, plan.wide, wgs, s); break;
    default: launch_product<4>(a, w, plan.wide, wgs, s); break;
  }
  if (int rc = check_launch("linear_product_kernel")) return rc;
  if (!plan.epilogue) return SUFHIP_OK;
  const EpiArgs e{a, act};
  const size_t cus = size_t(device_cus());
  // Wide from two full passes of the chip on, as the chains' own launch; small
  // below one of the mid form's.
  const int size = g.act == SUFHIP_ACT_CUBIC && mn >= 2 * cus * 1024 ? kEpiWide
                   : g.act != SUFHIP_ACT_NONE && mn < cus * 1024     ? kEpiSmall
                                                                     : kEpiMid;
  const size_t block = size == kEpiWide ? 1024 : (size == kEpiMid ? 512 : 256);
  size_t grid = (mn + block - 1) / block;
  const size_t cap = cus * (size == kEpiWide ? 1 : (g.act == SUFHIP_ACT_NONE ? 4 : 2));
  if (grid > cap && size != kEpiSmall) grid = cap;
  const dim3 gd{unsigned(grid)}, bd{unsigned(block)};
  if (g.act == SUFHIP_ACT_NONE)
    hipLaunchKernelGGL((linear_epilogue_kernel<SUFHIP_ACT_NONE, kEpiMid>), gd, bd, 0, s, e);
  else if (g.act == SUFHIP_ACT_RELU && size == kEpiSmall)
    hipLaunchKernelGGL((linear_epilogue_kernel<SUFHIP_ACT_RELU, kEpiSmall>), gd, bd, 0, s, e);
  else if (g.act == SUFHIP_ACT_RELU)
    hipLaunchKernelGGL((linear_epilogue_kernel<SUFHIP_ACT_RELU, kEpiMid>), gd, bd, 0, s, e);
  else if (size == kEpiSmall)
    hipLaunchKernelGGL((linear_epilogue_kernel<SUFHIP_ACT_CUBIC, kEpiSmall>), gd, bd, 0, s, e);
  else if (size == kEpiMid)
    hipLaunchKernelGGL((linear_epilogue_kernel<SUFHIP_ACT_CUBIC, kEpiMid>), gd, bd, 0, s, e);
  else
    hipLaunchKernelGGL((linear_epilogue_kernel<SUFHIP_ACT_CUBIC, kEpiWide>), gd, bd, 0, s, e);
  return check_launch("linear_epilogue_kernel");
}

}  // extern "C"
