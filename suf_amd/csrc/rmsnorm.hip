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

// The lane's number afresh, for the same reason: addresses formed from it are
// not held over the kernel.
__device__ __forceinline__ int rms_lane() {
  int t = int(threadIdx.x);
  asm volatile("" : "+v"(t));
  return t;
}

typedef uint64_t u64x2u __attribute__((ext_vector_type(2), aligned(8)));

// Four neighbours from column c on; zeros past the row's end.
__device__ __forceinline__ void load4(const uint64_t* row, int c, int cols, uint64_t (&v)[4]) {
  if (c + 4 <= cols) {
    const u64x2u a = *reinterpret_cast<const u64x2u*>(row + c);
    const u64x2u b = *reinterpret_cast<const u64x2u*>(row + c + 2);
    v[0] = a[0];
    v[1] = a[1];
    v[2] = b[0];
    v[3] = b[1];
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = c + q < cols ? row[c + q] : 0;
  }
}

__device__ __forceinline__ void store4(uint64_t* row, int c, int cols, const uint64_t (&v)[4]) {
  if (c + 4 <= cols) {
    *reinterpret_cast<u64x2u*>(row + c) = u64x2u{v[0], v[1]};
    *reinterpret_cast<u64x2u*>(row + c + 2) = u64x2u{v[2], v[3]};
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (c + q < cols) row[c + q] = v[q];
  }
}

// One lane's four values of a row from its sum to its output: s less its mask,
// and the mask's shares.
struct RmsQuad {
  uint64_t D[4], a0[4], a1[4];
};

// Columns c .. c + 3 of row r.  again: for the output of a row that was summed
// before (and whose total, if any, is written).
__device__ __forceinline__ void rms_load(RmsQuad& v, int r, int c, bool again) {
  const RmsArgs& A = rms_args();
  const int cols = A.cols;
  const size_t base = size_t(r) * size_t(cols);
  uint64_t s[2][4];
  if (again && A.total[0]) {
#pragma unroll
    for (int p = 0; p < 2; ++p) load4(A.total[p] + int64_t(r) * A.total_stride, c, cols, s[p]);
    load4(A.a[0] + base, c, cols, v.a0);
    load4(A.a[1] + base, c, cols, v.a1);
  } else {
    uint64_t x[2][4];
#pragma unroll
    for (int p = 0; p < 2; ++p) load4(A.x.p[p] + int64_t(r) * A.x.stride, c, cols, s[p]);
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int q = 0; q < 4; ++q) x[p][q] = 0;
    if (A.r.p[0]) {
#pragma unroll
      for (int p = 0; p < 2; ++p) load4(A.r.p[p] + int64_t(r) * A.r.stride, c, cols, x[p]);
    }
    load4(A.a[0] + base, c, cols, v.a0);
    load4(A.a[1] + base, c, cols, v.a1);
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int q = 0; q < 4; ++q) s[p][q] += x[p][q];
    if (!again && A.total[0]) {
#pragma unroll
      for (int p = 0; p < 2; ++p) store4(A.total[p] + int64_t(r) * A.total_stride, c, cols, s[p]);
    }
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) v.D[q] = (s[0][q] - v.a0[q]) + (s[1][q] - v.a1[q]);
}

// The outputs at those columns: b0, b1 the shares of the row's mask, E the open
// of its factor.
__device__ __forceinline__ void rms_put(const RmsQuad& v, int r, int c, uint64_t b0,
                                        uint64_t b1, uint64_t E) {
  const RmsArgs& A = rms_args();
  const int cols = A.cols;
  const size_t base = size_t(r) * size_t(cols);
  const EpiHdrs hn = epi_hdrs(A.tr[kNorm]), hw = epi_hdrs(A.tr[kWeight]);
  uint64_t z[2][4], y[2][4];
#pragma unroll
  for (int p = 0; p < 2; ++p) load4(A.ab[p] + base, c, cols, z[p]);
  uint64_t w[4] = {0, 0, 0, 0};
  if (A.w) load4(reinterpret_cast<const uint64_t*>(A.w), c, cols, w);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    z[0][q] += v.D[q] * b0 + v.a0[q] * E + v.D[q] * E;
    z[1][q] += v.D[q] * b1 + v.a1[q] * E;
    uint64_t o[2];
    gate2(A.tr[kNorm], hn, z[0][q] + z[1][q] + A.mask[kNorm], o);
    y[0][q] = o[0];
    y[1][q] = o[1];
  }
  if (A.w) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint64_t o[2];
      gate2(A.tr[kWeight], hw, y[0][q] * w[q] + y[1][q] * w[q] + A.mask[kWeight], o);
      y[0][q] = o[0];
      y[1][q] = o[1];
    }
  }
  if (A.out[0]) {
#pragma unroll
    for (int p = 0; p < 2; ++p) store4(A.out[p] + int64_t(r) * A.out_stride, c, cols, y[p]);
  }
  if (A.digits) {  // zeros past the row's end, up to the next multiple of 32
#pragma unroll
    for (int p = 0; p < 2; ++p) {
#pragma unroll
      for (int q = 0; q < 4; ++q) y[p][q] = c + q < cols ? y[p][q] : 0;
      uint32_t d[8];
      digits_of4(y[p], d);
      int8_t* at = A.digits + digit_off(size_t(p) * A.rows + r, c, size_t(A.rows));
#pragma unroll
      for (int i = 0; i < 8; ++i) *reinterpret_cast<uint32_t*>(at + 32 * i) = d[i];
    }
  }
}

// A row of up to 4 kQuads kBlock values stays on the CU from the sum to the
// output; with kLong a longer one is read again for the output.
template <int kQuads, int kBlock, bool kLong>
__global__ void __launch_bounds__(kBlock, 1024 / kBlock) rmsnorm2_kernel(RmsArgs) {
  constexpr int kWaves = kBlock / 64;
  constexpr int kSpan = 4 * kQuads * kBlock;
  constexpr int kProds = chain_products<SUFHIP_CHAIN_RSQRT>();
  __shared__ __align__(16) uint32_t tab[256 * kRmsCopies];
  __shared__ ChainLds L;
  __shared__ TruncHdr th[kNorm][2];  // the row's gates
  __shared__ TruncHdr rth[kProds][2];
  __shared__ uint64_t red[2][kWaves];
  __shared__ uint64_t bc[4];
  __shared__ ChainPre pre;
  // Wave 0's values of the row while it runs the row's chain, which needs their
  // registers.
  __shared__ uint64_t held[kLong ? 1 : 12 * kQuads][64];
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
  // Lanes whose columns end before this write nothing, not even digits.
  const int end = (cols + 31) / 32 * 32;
  for (int r = blockIdx.x; r < rows; r += int(gridDim.x)) {
    if (const int t = rms_lane(); t < 24)
      pre.word(t) = chain_triple_word(rms_args().rs, t, size_t(r));
    RmsQuad v[kQuads];
    uint64_t q0 = 0, q1 = 0;
    for (int c0 = 0; c0 < (kLong ? cols : 1); c0 += kSpan) {
#pragma unroll
      for (int k = 0; k < kQuads; ++k) {
        const int c = c0 + 4 * (rms_lane() + k * kBlock);
        rms_load(v[k], r, c, false);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          q0 += 2 * v[k].D[q] * v[k].a0[q] + v[k].D[q] * v[k].D[q];
          q1 += 2 * v[k].D[q] * v[k].a1[q];
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    block_sum2_u64<kWaves>(q0, q1, red);
    if (threadIdx.x < 64) {
      if constexpr (!kLong) {
        const int t = rms_lane();
#pragma unroll
        for (int k = 0; k < kQuads; ++k)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            held[12 * k + q][t] = v[k].D[q];
            held[12 * k + 4 + q][t] = v[k].a0[q];
            held[12 * k + 8 + q][t] = v[k].a1[q];
          }
        asm volatile("" ::: "memory");  // and nothing of them stays in registers
      }
      const RmsArgs& A = rms_args();
      const RmsAes aes{tab, uint32_t(rms_lane()) % kRmsCopies};
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
      const Two y = chain_eval_quad<SUFHIP_CHAIN_RSQRT, RmsAes>(rms_args().rs, L, K, aes,
                                                                size_t(r), ms, pre, rth);
      if (threadIdx.x == 0) {
        bc[0] = b0;
        bc[1] = b1;
        bc[2] = (y.v[0] - b0) + (y.v[1] - b1);
      }
      if constexpr (!kLong) {
        asm volatile("" ::: "memory");
        const int t = rms_lane();
#pragma unroll
        for (int k = 0; k < kQuads; ++k)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            v[k].D[q] = held[12 * k + q][t];
            v[k].a0[q] = held[12 * k + 4 + q][t];
            v[k].a1[q] = held[12 * k + 8 + q][t];
          }
      }
    }
    __syncthreads();
    const uint64_t b0 = bc[0], b1 = bc[1], E = bc[2];
    for (int c0 = 0; c0 < (kLong ? cols : 1); c0 += kSpan) {
#pragma unroll
      for (int k = 0; k < kQuads; ++k) {
        const int c = c0 + 4 * (rms_lane() + k * kBlock);
        if (kLong) rms_load(v[k], r, c, true);
        if (c < end) rms_put(v[k], r, c, b0, b1, E);
        __builtin_amdgcn_sched_barrier(0);  // one quad's registers at a time
      }
    }
    __syncthreads();  // bc and pre are rewritten for the next row
  }
}

template <int kQuads, int kBlock, bool kLong>
int launch_rms(const RmsArgs& A, hipStream_t s) {
  int dev = 0, cus = 256;
  if (hipGetDevice(&dev) == hipSuccess)
    (void)hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev);
  const int cap = cus * (2048 / kBlock > 8 ? 8 : 2048 / kBlock);
  const int grid = A.rows < cap ? A.rows : cap;
  hipLaunchKernelGGL((rmsnorm2_kernel<kQuads, kBlock, kLong>), dim3(unsigned(grid)), dim3(kBlock), 0,
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
  if (g.cols <= 1024) return launch_rms<1, 256, false>(A, s);
  if (g.cols <= 2048) return launch_rms<2, 256, false>(A, s);
  if (g.cols <= 4096) return launch_rms<2, 512, false>(A, s);
  return launch_rms<1, 1024, true>(A, s);
}

}  // extern "C"
