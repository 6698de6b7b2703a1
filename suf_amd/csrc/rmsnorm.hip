// Root-mean-square norm with the residual's addition (sufhip_rmsnorm2), both
// parties, a workgroup a row.
//
//   s = x + residual,  S = sum s s,  v = S / cols + eps,  o = s / sqrt(v)
//
// Both products have s on one side, and what is opened is s minus a mask: with
// one mask a for both, D = s - a is opened once, and the row needs
//   S_p = a2_p + sum (2 D a_p + [p = 0] D D)           a2 = sum a a, a word a row
//   (s y)_p = ab_p + D b_p + a_p E + [p = 0] D E       E = y - b, b a word a row
// so an element costs its mask's two shares and ab's two, where two triples
// of its own (a square's and a row product's) would be ten words.  The sum
// over a row is linear, so it is taken before any truncation, on words mod
// 2^64: it loses nothing.
#include <hip/hip_runtime.h>

#include "chain_device.hpp"
#include "feedforward_device.hpp"
#include "reduce_device.hpp"

namespace sufhip {
namespace {

constexpr int kRmsCopies = 4;  // the T table serves one wave a workgroup
using RmsAes = AesLds<kRmsCopies>;

enum { kMs0 = 0, kMs1 = 1, kMs2 = 2, kNorm = 3, kWeight = 4, kGates = 5 };

struct RmsArgs {
  Mat2 x, r;  // r.p NULL: no residual
  int rows, cols;
  uint64_t inv_len, eps;
  const uint64_t* a[2];
  const uint64_t* a2[2];
  const uint64_t* b[2];
  const uint64_t* ab[2];
  TruncEpi tr[kGates];
  uint64_t mask[kGates];
  ChainArgs rs;
  const int64_t* w;
  uint64_t* total[2];
  int64_t total_stride;
  uint64_t* out[2];
  int64_t out_stride;
  int8_t* digits;
};
static_assert(sizeof(RmsArgs) <= 4096, "kernel argument blocks must fit in 4 KB");

// The kernel's argument read afresh from the kernarg segment, an opaque copy of
// its address per phase of a row: a phase's pointers are scalar loads where
// they are used.  All of them held over the kernel exceed the scalar registers
// and were moved to vector lanes and back (215 of them).
__device__ __forceinline__ const RmsArgs& rms_args() {
  typedef const __attribute__((address_space(4))) RmsArgs* Ptr;
  Ptr p = (Ptr)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const RmsArgs*)p;
}

// A row's values in registers from its sum to its output: s less its mask, and
// the mask's shares.
template <int kPer>
struct RmsRow {
  uint64_t D[kPer], a0[kPer], a1[kPer];
};

// Columns c0 + thread + k kBlock of row r.  again: for the output of a row that
// was summed before (and whose total, if any, is written).
template <int kPer, int kBlock>
__device__ __forceinline__ void rms_load(RmsRow<kPer>& v, int r, int c0, bool again) {
  const RmsArgs& A = rms_args();
  const int cols = A.cols;
  const size_t base = size_t(r) * size_t(cols);
  uint64_t s[kPer][2];
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int c = c0 + int(threadIdx.x) + k * kBlock;
    s[k][0] = s[k][1] = v.a0[k] = v.a1[k] = 0;
    if (c < cols) {
      if (again && A.total[0]) {
        s[k][0] = A.total[0][int64_t(r) * A.total_stride + c];
        s[k][1] = A.total[1][int64_t(r) * A.total_stride + c];
      } else {
        s[k][0] = A.x.p[0][int64_t(r) * A.x.stride + c];
        s[k][1] = A.x.p[1][int64_t(r) * A.x.stride + c];
        if (A.r.p[0]) {
          s[k][0] += A.r.p[0][int64_t(r) * A.r.stride + c];
          s[k][1] += A.r.p[1][int64_t(r) * A.r.stride + c];
        }
      }
      v.a0[k] = A.a[0][base + c];
      v.a1[k] = A.a[1][base + c];
    }
    v.D[k] = (s[k][0] - v.a0[k]) + (s[k][1] - v.a1[k]);
  }
  if (!again && A.total[0]) {
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int c = c0 + int(threadIdx.x) + k * kBlock;
      if (c < cols) {
        A.total[0][int64_t(r) * A.total_stride + c] = s[k][0];
        A.total[1][int64_t(r) * A.total_stride + c] = s[k][1];
      }
    }
  }
}

// The outputs at those columns: b the shares of the row's mask, E the open of
// its factor.
template <int kPer, int kBlock>
__device__ __forceinline__ void rms_put(const RmsRow<kPer>& v, int r, int c0, uint64_t b0,
                                        uint64_t b1, uint64_t E) {
  const RmsArgs& A = rms_args();
  const int cols = A.cols;
  const size_t base = size_t(r) * size_t(cols);
  const EpiHdrs hn = epi_hdrs(A.tr[kNorm]), hw = epi_hdrs(A.tr[kWeight]);
  uint64_t open[kPer], y[kPer][2];
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int c = c0 + int(threadIdx.x) + k * kBlock;
    uint64_t z0 = v.D[k] * b0 + v.a0[k] * E + v.D[k] * E, z1 = v.D[k] * b1 + v.a1[k] * E;
    if (c < cols) {
      z0 += A.ab[0][base + c];
      z1 += A.ab[1][base + c];
    }
    open[k] = z0 + z1 + A.mask[kNorm];
  }
#pragma unroll
  for (int k = 0; k < kPer; ++k) gate2(A.tr[kNorm], hn, open[k], y[k]);
  if (A.w) {
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int c = c0 + int(threadIdx.x) + k * kBlock;
      const uint64_t w = c < cols ? uint64_t(A.w[c]) : 0;
      gate2(A.tr[kWeight], hw, y[k][0] * w + y[k][1] * w + A.mask[kWeight], y[k]);
    }
  }
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int c = c0 + int(threadIdx.x) + k * kBlock;
    if (c >= cols) continue;
    if (A.out[0]) {
      A.out[0][int64_t(r) * A.out_stride + c] = y[k][0];
      A.out[1][int64_t(r) * A.out_stride + c] = y[k][1];
    }
    if (A.digits) {
      put_digits(A.digits, size_t(A.rows), size_t(r), c, 0, y[k][0]);
      put_digits(A.digits, size_t(A.rows), size_t(r), c, 1, y[k][1]);
    }
  }
}

// A row of up to kPer * kBlock values stays in registers from the sum to the
// output; with kLong a longer one is read again for the output.
template <int kPer, int kBlock, bool kLong>
__global__ void __launch_bounds__(kBlock, 1024 / kBlock) rmsnorm2_kernel(RmsArgs) {
  constexpr int kWaves = kBlock / 64;
  constexpr int kSpan = kPer * kBlock;
  constexpr int kProds = chain_products<SUFHIP_CHAIN_RSQRT>();
  __shared__ __align__(16) uint32_t tab[256 * kRmsCopies];
  __shared__ ChainLds L;
  __shared__ TruncHdr th[kNorm][2];  // the row's gates
  __shared__ TruncHdr rth[kProds][2];
  __shared__ uint64_t red[2][kWaves];
  __shared__ uint64_t bc[4];
  __shared__ ChainPre pre;
  {
    const RmsArgs& A = rms_args();
    fill_ttable<kRmsCopies>(tab, kTDev.v);
    chain_stage(A.rs, 2, L);
    if (int(threadIdx.x) < 2 * kNorm)
      th[threadIdx.x >> 1][threadIdx.x & 1] =
          read_trunc_hdr(A.tr[threadIdx.x >> 1].key[threadIdx.x & 1]);
    TruncHdrStager<kProds> hs;
    hs.load(A.rs, 64);
    hs.store(rth);
    __syncthreads();
    chain_compare(A.rs, L);
    __syncthreads();
  }
  const int rows = rms_args().rows, cols = rms_args().cols;
  for (int r = blockIdx.x; r < rows; r += int(gridDim.x)) {
    if (threadIdx.x < 24)
      pre.word(threadIdx.x) = chain_triple_word(rms_args().rs, threadIdx.x, size_t(r));
    RmsRow<kPer> v;
    uint64_t q0 = 0, q1 = 0;
    for (int c0 = 0; c0 < (kLong ? cols : 1); c0 += kSpan) {
      rms_load<kPer, kBlock>(v, r, c0, false);
#pragma unroll
      for (int k = 0; k < kPer; ++k) {
        q0 += 2 * v.D[k] * v.a0[k] + v.D[k] * v.D[k];
        q1 += 2 * v.D[k] * v.a1[k];
      }
    }
    block_sum2_u64<kWaves>(q0, q1, red);
    if (threadIdx.x < 64) {
      const RmsArgs& A = rms_args();
      const RmsAes aes{tab, threadIdx.x % kRmsCopies};
      const ChainKeyInfo K = chain_key_info(A.rs, L);
      auto gate = [&](int j, uint64_t x) {
        return Two{{trunc_table_eval_h(th[j][0], A.tr[j].table[0], A.tr[j].f, x),
                    trunc_table_eval_h(th[j][1], A.tr[j].table[1], A.tr[j].f, x)}};
      };
      const uint64_t b0 = A.b[0][r], b1 = A.b[1][r];
      Two m = gate(kMs0, (q0 + A.a2[0][r]) + (q1 + A.a2[1][r]) + A.mask[kMs0]);
      m = gate(kMs1, m.v[0] * A.inv_len + m.v[1] * A.inv_len + A.mask[kMs1]);
      m = gate(kMs2, m.v[0] + m.v[1] + A.mask[kMs2]);
      const Two ms{{m.v[0] + A.eps, m.v[1]}};
      const Two y =
          chain_eval_quad<SUFHIP_CHAIN_RSQRT, RmsAes>(A.rs, L, K, aes, size_t(r), ms, pre, rth);
      if (threadIdx.x == 0) {
        bc[0] = b0;
        bc[1] = b1;
        bc[2] = (y.v[0] - b0) + (y.v[1] - b1);
      }
    }
    __syncthreads();
    const uint64_t b0 = bc[0], b1 = bc[1], E = bc[2];
    for (int c0 = 0; c0 < (kLong ? cols : 1); c0 += kSpan) {
      if (kLong) rms_load<kPer, kBlock>(v, r, c0, true);
      rms_put<kPer, kBlock>(v, r, c0, b0, b1, E);
    }
    const RmsArgs& A = rms_args();
    if (A.digits) {  // up to the next multiple of 32
      const int end = (cols + 31) / 32 * 32, c = cols + int(threadIdx.x);
      if (c < end) {
        put_digits(A.digits, size_t(rows), size_t(r), c, 0, 0);
        put_digits(A.digits, size_t(rows), size_t(r), c, 1, 0);
      }
    }
    __syncthreads();  // bc and pre are rewritten for the next row
  }
}

template <int kPer, int kBlock, bool kLong>
int launch_rms(const RmsArgs& A, hipStream_t s) {
  int dev = 0, cus = 256;
  if (hipGetDevice(&dev) == hipSuccess)
    (void)hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev);
  const int cap = cus * (2048 / kBlock > 8 ? 8 : 2048 / kBlock);
  const int grid = A.rows < cap ? A.rows : cap;
  hipLaunchKernelGGL((rmsnorm2_kernel<kPer, kBlock, kLong>), dim3(unsigned(grid)), dim3(kBlock), 0,
                     s, A);
  return check_launch("rmsnorm2_kernel");
}

}  // namespace
}  // namespace sufhip

using namespace sufhip;

extern "C" {

int sufhip_rmsnorm2(const sufhip_rmsnorm2_args* args, void* stream) {
  const char* what = "sufhip_rmsnorm2";
  SUFHIP_REQUIRE(args, "sufhip_rmsnorm2: null args");
  const sufhip_rmsnorm2_args& g = *args;
  if (g.rows < 0 || g.cols < 0 || g.rows > kMaxRows || g.cols > (1 << 20))
    return ff_fail(what, "rows in [0, 2^24] and cols in [0, 2^20]");
  if (g.rows == 0 || g.cols == 0) return SUFHIP_OK;
  const size_t n = size_t(g.rows) * size_t(g.cols);
  RmsArgs A{};
  A.rows = g.rows;
  A.cols = g.cols;
  A.inv_len = g.inv_len;
  A.eps = g.eps;
  if (int rc = mat2_of(g.x, g.rows, g.cols, what, "x", &A.x)) return rc;
  if ((g.residual.p[0] == nullptr) != (g.residual.p[1] == nullptr))
    return ff_fail(what, "one share of the residual is missing");
  if (g.residual.p[0])
    if (int rc = mat2_of(g.residual, g.rows, g.cols, what, "residual", &A.r)) return rc;
  for (int p = 0; p < 2; ++p) {
    if (!g.a[p] || !g.a2[p] || !g.b[p] || !g.ab[p])
      return ff_fail(what, "a, a2, b and ab are needed for both parties");
    A.a[p] = g.a[p];
    A.a2[p] = g.a2[p];
    A.b[p] = g.b[p];
    A.ab[p] = g.ab[p];
    A.total[p] = g.total[p];
    A.out[p] = g.out[p];
  }
  for (int q = 0; q < 3; ++q) {
    if (int rc = gate_of(g.tr_ms[q], size_t(g.rows), what, &A.tr[kMs0 + q])) return rc;
    A.mask[kMs0 + q] = g.ms_mask[q];
  }
  if (int rc = gate_of(g.tr_norm, n, what, &A.tr[kNorm])) return rc;
  A.mask[kNorm] = g.norm_mask;
  A.w = g.d_weight;
  if (A.w) {
    if (int rc = gate_of(g.tr_weight, n, what, &A.tr[kWeight])) return rc;
    A.mask[kWeight] = g.weight_mask;
  }
  if (g.rsqrt.kind != SUFHIP_CHAIN_RSQRT || g.rsqrt.n != size_t(g.rows))
    return ff_fail(what, "rsqrt must be a SUFHIP_CHAIN_RSQRT chain with n = rows");
  if (int rc = make_chain_args(g.rsqrt, false, what, &A.rs)) return rc;
  if ((g.total[0] == nullptr) != (g.total[1] == nullptr) ||
      (g.out[0] == nullptr) != (g.out[1] == nullptr))
    return ff_fail(what, "give both share outputs or neither");
  if (!g.out[0] && !g.out_digits.d_digits && !g.total[0]) return ff_fail(what, "no output");
  if (g.out_digits.d_digits)
    if (int rc = digits2_of(g.out_digits, g.rows, g.cols, what, "out_digits")) return rc;
  A.total_stride = g.total_stride;
  A.out_stride = g.out_stride;
  A.digits = g.out_digits.d_digits;
  // Outputs: rows of their own; where they meet x or the residual they are them.
  RowSet outs[5];
  int count = 0;
  for (int p = 0; p < 2; ++p) {
    if (g.total[0]) outs[count++] = {g.total[p], g.total_stride, g.rows, g.cols};
    if (g.out[0]) outs[count++] = {g.out[p], g.out_stride, g.rows, g.cols};
  }
  for (int i = 0; i < count; ++i) {
    if (outs[i].stride < 0 || rows_overlap(outs[i].stride, g.rows, g.cols))
      return ff_fail(what, "output rows overlap");
    const int p = g.total[0] && g.out[0] ? i / 2 : i;
    for (int q = 0; q < 2; ++q) {
      const RowSet in[2] = {row_set(A.x, q, g.rows, g.cols), row_set(A.r, q, g.rows, g.cols)};
      for (int k = 0; k < (A.r.p[0] ? 2 : 1); ++k)
        if (sets_meet(outs[i], in[k]) && !(p == q && same_set(outs[i], in[k])))
          return ff_fail(what, "an output meets x or the residual without being it");
      const RowSet mat[4] = {{g.a[q], 0, 1, 0}, {g.ab[q], 0, 1, 0}, {g.a2[q], 0, 1, g.rows},
                             {g.b[q], 0, 1, g.rows}};
      for (int k = 0; k < 4; ++k) {
        RowSet m = mat[k];
        if (k < 2) m = {m.p, g.cols, g.rows, g.cols};
        if (sets_meet(outs[i], m)) return ff_fail(what, "an output meets the dealer's material");
      }
    }
    for (int j = 0; j < i; ++j)
      if (sets_meet(outs[i], outs[j])) return ff_fail(what, "two outputs meet");
  }
  if (A.digits) {
    const size_t bytes = sufhip_digits2_bytes(g.rows, g.cols);
    for (int q = 0; q < 2; ++q) {
      const RowSet in[4] = {row_set(A.x, q, g.rows, g.cols),
                            row_set(A.r, q, A.r.p[0] ? g.rows : 0, g.cols),
                            {g.a[q], g.cols, g.rows, g.cols},
                            {g.ab[q], g.cols, g.rows, g.cols}};
      for (const RowSet& s : in)
        if (range_meets(A.digits, bytes, s)) return ff_fail(what, "out_digits meets an input");
    }
    for (int i = 0; i < count; ++i)
      if (range_meets(A.digits, bytes, outs[i])) return ff_fail(what, "out_digits meets an output");
  }
  hipStream_t s = as_stream(stream);
  if (g.cols <= 1024) return launch_rms<4, 256, false>(A, s);
  if (g.cols <= 2048) return launch_rms<4, 512, false>(A, s);
  if (g.cols <= 4096) return launch_rms<8, 512, false>(A, s);
  return launch_rms<4, 1024, true>(A, s);
}

}  // extern "C"
