// Root-mean-square norm with the residual's addition (sufhip_rmsnorm2), both
// parties: a workgroup a row, or three launches for a large one.
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
#include "walk_device.hpp"

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
  uint64_t* sums;   // the launches of a large norm: [2][rows] sums of s s
  uint64_t* opens;  // [rows] opens of the rows' factors
};

// Key-only walks beside a large norm's sums: its own nine gates of both parties.
constexpr int kRmsWalks = 18;
struct RmsWalk {
  WalkJobs<kRmsWalks> jobs;
  int groups;  // workgroups of them, the launch's first
};
static_assert(sizeof(RmsArgs) + sizeof(RmsWalk) <= 4096,
              "kernel argument blocks must fit in 4 KB");

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
// of its factor; lds: the elements' gates' tables (the norm's, the weight's), or
// none, to read them in memory.
template <bool kLds = false>
__device__ __forceinline__ void rms_put(const RmsQuad& v, int r, int c, uint64_t b0,
                                        uint64_t b1, uint64_t E, const LdsGate* lds = nullptr) {
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
    const uint64_t open = z[0][q] + z[1][q] + A.mask[kNorm];
    if constexpr (kLds)
      gate2(A.tr[kNorm], hn, lds[0], open, o);
    else
      gate2(A.tr[kNorm], hn, open, o);
    y[0][q] = o[0];
    y[1][q] = o[1];
  }
  if (A.w) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint64_t o[2];
      const uint64_t open = y[0][q] * w[q] + y[1][q] * w[q] + A.mask[kWeight];
      if constexpr (kLds)
        gate2(A.tr[kWeight], hw, lds[1], open, o);
      else
        gate2(A.tr[kWeight], hw, open, o);
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

// The row's factor from its sums: the gates of the mean square and the chain,
// on one wave, every lane with the same values.  The caller staged the chain's
// LUT, triples and headers.  Returns the shares.
__device__ __forceinline__ Two rms_factor(const uint32_t* tab, const ChainLds& L,
                                          const TruncHdr (*th)[2], const TruncHdr (*rth)[2],
                                          const ChainPre& pre, int r, uint64_t s0, uint64_t s1) {
  const RmsArgs& A = rms_args();
  const RmsAes aes{tab, uint32_t(rms_lane()) % kRmsCopies};
  const ChainKeyInfo K = chain_key_info(A.rs, L);
  auto gate = [&](int j, uint64_t x) {
    return Two{{trunc_table_eval_h(th[j][0], A.tr[j].table[0], A.tr[j].f, x),
                trunc_table_eval_h(th[j][1], A.tr[j].table[1], A.tr[j].f, x)}};
  };
  Two m = gate(kMs0, (s0 + A.a2[0][r]) + (s1 + A.a2[1][r]) + A.mask[kMs0]);
  m = gate(kMs1, m.v[0] * A.inv_len + m.v[1] * A.inv_len + A.mask[kMs1]);
  m = gate(kMs2, m.v[0] + m.v[1] + A.mask[kMs2]);
  const Two ms{{m.v[0] + A.eps, m.v[1]}};
  return chain_eval_quad<SUFHIP_CHAIN_RSQRT, RmsAes>(rms_args().rs, L, K, aes, size_t(r), ms, pre,
                                                     rth);
}

// What rms_factor needs in LDS; ends with a barrier.
__device__ __forceinline__ void rms_stage(uint32_t* tab, ChainLds& L, TruncHdr (*th)[2],
                                          TruncHdr (*rth)[2]) {
  const RmsArgs& A = rms_args();
  fill_ttable<kRmsCopies>(tab, kTDev.v);
  chain_stage(A.rs, 2, L);
  if (int(threadIdx.x) < 2 * kNorm)
    th[threadIdx.x >> 1][threadIdx.x & 1] =
        read_trunc_hdr(A.tr[threadIdx.x >> 1].key[threadIdx.x & 1]);
  TruncHdrStager<chain_products<SUFHIP_CHAIN_RSQRT>()> hs;
  hs.load(A.rs, 64);
  hs.store(rth);
  __syncthreads();
  chain_compare(A.rs, L);
  __syncthreads();
}

// A row of up to 4 kQuads kBlock values stays on the CU from the sum to the
// output; with kLong a longer one is read again for the output.  One row is
// bound by latency, seven gates and a LUT one after the other: 14 us for 768
// values in a captured graph, 18 after other work.  Many stream their 12 words a
// value: 1000 x 2048 with its total 55 us, 3.6 TB/s (with a weight too 67), the
// workgroups' chains between their loads.
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
  rms_stage(tab, L, th, rth);
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
      const Two y = rms_factor(tab, L, th, rth, pre, r, q0, q1);
      const uint64_t b0 = rms_args().b[0][r], b1 = rms_args().b[1][r];
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

// A large norm in three launches, each at the memory's pace: the rows' sums (and
// total), with the gates' walks beside them; the rows' factors, a wave a row;
// the outputs.  Row by row in one launch, the workgroups all wait for their
// chains at the same time, and behind each other's loads: 1999 x 2048 with
// total and weight 134 us after 22 of walks.  In three: 57 us of sums and walks
// (262 MB, 4.6 TB/s), 17 of factors, 54 of outputs (262 MB, 4.8 TB/s: as a
// copy).  Factors in the outputs' launch: 72 us for the two.
//
// kWaveRow: a wave a row (rows of up to 1024 values), else a workgroup a row.
template <bool kWaveRow, bool kWalk>
__global__ void __launch_bounds__(256) rms_sum_kernel(RmsArgs, RmsWalk wk) {
  if constexpr (kWalk) {
    if (int(blockIdx.x) < wk.groups) {
      hosted_walk_role<kRmsWalks, false>(wk.jobs, blockIdx.x * 256 + threadIdx.x);
      return;
    }
  }
  __shared__ uint64_t red[2][4];
  const int first = int(blockIdx.x) - (kWalk ? wk.groups : 0);
  const int step = int(gridDim.x) - (kWalk ? wk.groups : 0);
  const int rows = rms_args().rows, cols = rms_args().cols;
  const int wave = int(threadIdx.x) >> 6;
  const int lane = kWaveRow ? int(threadIdx.x) & 63 : int(threadIdx.x);
  constexpr int kPerGroup = kWaveRow ? 4 : 1, kSpan = kWaveRow ? 256 : 1024;
  for (int r = first * kPerGroup + (kWaveRow ? wave : 0); r < rows; r += step * kPerGroup) {
    uint64_t q0 = 0, q1 = 0;
    for (int c = 4 * lane; c < cols; c += kSpan) {
      RmsQuad v;
      rms_load(v, r, c, false);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        q0 += 2 * v.D[q] * v.a0[q] + v.D[q] * v.D[q];
        q1 += 2 * v.D[q] * v.a1[q];
      }
    }
    if constexpr (kWaveRow) {
      q0 = wave_sum_u64(q0);
      q1 = wave_sum_u64(q1);
    } else {
      block_sum2_u64<4>(q0, q1, red);
    }
    if (lane == 0) {
      rms_args().sums[r] = q0;
      rms_args().sums[size_t(rows) + r] = q1;
    }
  }
}

__global__ void __launch_bounds__(256) rms_factor_kernel(RmsArgs) {
  __shared__ __align__(16) uint32_t tab[256 * kRmsCopies];
  __shared__ ChainLds L;
  __shared__ TruncHdr th[kNorm][2];
  __shared__ TruncHdr rth[chain_products<SUFHIP_CHAIN_RSQRT>()][2];
  __shared__ ChainPre pre[4];
  rms_stage(tab, L, th, rth);
  const int rows = rms_args().rows;
  const int wave = int(threadIdx.x) >> 6, lane = int(threadIdx.x) & 63;
  // Every wave of a workgroup makes the same number of rounds (the barriers).
  for (int r0 = int(blockIdx.x) * 4; r0 < rows; r0 += int(gridDim.x) * 4) {
    const int r = r0 + wave < rows ? r0 + wave : rows - 1;
    if (lane < 24) pre[wave].word(lane) = chain_triple_word(rms_args().rs, lane, size_t(r));
    __syncthreads();
    const RmsArgs& A = rms_args();
    const Two y =
        rms_factor(tab, L, th, rth, pre[wave], r, A.sums[r], A.sums[size_t(rows) + r]);
    if (lane == 0 && r0 + wave < rows)
      rms_args().opens[r] =
          (y.v[0] - rms_args().b[0][r]) + (y.v[1] - rms_args().b[1][r]);
    __syncthreads();  // pre is rewritten for the next row
  }
}

// kGates: of the elements' gates, the norm's and the weight's, how many have
// their tables in LDS (all or none).
template <int kGates>
__global__ void __launch_bounds__(kGates ? 1024 : 256) rms_out_kernel(RmsArgs) {
  __shared__ __align__(16) LdsGate lds[kGates ? kGates : 1];
  if constexpr (kGates > 0) {
    stage_gate(rms_args().tr[kNorm], lds[0]);
    if constexpr (kGates > 1) stage_gate(rms_args().tr[kWeight], lds[1]);
    __syncthreads();
  }
  const int rows = rms_args().rows, cols = rms_args().cols;
  const uint32_t quads = uint32_t((cols + 31) / 32) * 8;  // with the digits' padding
  const size_t n = size_t(rows) * quads;
  for (size_t i = size_t(blockIdx.x) * blockDim.x + threadIdx.x; i < n;
       i += size_t(gridDim.x) * blockDim.x) {
    const int r = int(i / quads), c = 4 * int(i % quads);
    RmsQuad v;
    rms_load(v, r, c, true);
    const RmsArgs& A = rms_args();
    rms_put<(kGates > 0)>(v, r, c, A.b[0][r], A.b[1][r], A.opens[r], lds);
  }
}

int device_cus() {
  int dev = 0, cus = 256;
  if (hipGetDevice(&dev) == hipSuccess)
    (void)hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev);
  return cus;
}

// Whether a norm takes the three launches.  One launch / three, in us, the nine
// gates' walks included, with residual and total: 512 x 1024 47 / 57, 512 x 2048
// 54 / 65, 1000 x 2048 76 / 82, 1999 x 2048 with a weight 156 / 130.  The shape
// counts too, which the rule leaves out: 488 x 4096 87 / 82, and with rows of
// more than 4096 values, read twice either way, 64 x 16384 87 / 61; with many
// short ones, a chain each, 20000 x 96 327 / 117.
bool rms_large(int rows, int cols) { return size_t(rows) * size_t(cols) >= (size_t(1) << 21); }

int launch_large(const RmsArgs& A, const RmsWalk& w, hipStream_t s) {
  const int cus = device_cus();
  const bool wave = A.cols <= 1024;
  int groups = wave ? (A.rows + 3) / 4 : A.rows;
  if (groups > 8 * cus) groups = 8 * cus;
  const dim3 g(unsigned(groups + w.groups)), b(256);
  if (wave && w.groups)
    hipLaunchKernelGGL((rms_sum_kernel<true, true>), g, b, 0, s, A, w);
  else if (wave)
    hipLaunchKernelGGL((rms_sum_kernel<true, false>), g, b, 0, s, A, w);
  else if (w.groups)
    hipLaunchKernelGGL((rms_sum_kernel<false, true>), g, b, 0, s, A, w);
  else
    hipLaunchKernelGGL((rms_sum_kernel<false, false>), g, b, 0, s, A, w);
  if (int rc = check_launch("rms_sum_kernel")) return rc;
  groups = (A.rows + 3) / 4;
  if (groups > 4 * cus) groups = 4 * cus;
  hipLaunchKernelGGL(rms_factor_kernel, dim3(unsigned(groups)), b, 0, s, A);
  if (int rc = check_launch("rms_factor_kernel")) return rc;
  if (!A.out[0] && !A.digits) return SUFHIP_OK;
  const size_t n = size_t(A.rows) * size_t((A.cols + 31) / 32) * 8;
  if (A.tr[kNorm].f <= kLdsGateBits && (!A.w || A.tr[kWeight].f <= kLdsGateBits)) {
    const dim3 lg{unsigned(cus)}, lb{1024};
    if (A.w)
      hipLaunchKernelGGL(rms_out_kernel<2>, lg, lb, 0, s, A);
    else
      hipLaunchKernelGGL(rms_out_kernel<1>, lg, lb, 0, s, A);
  } else {
    size_t out = (n + 255) / 256;
    if (out > size_t(32) * cus) out = size_t(32) * cus;
    hipLaunchKernelGGL(rms_out_kernel<0>, dim3(unsigned(out)), b, 0, s, A);
  }
  return check_launch("rms_out_kernel");
}

template <int kQuads, int kBlock, bool kLong>
int launch_rms(const RmsArgs& A, hipStream_t s) {
  const int cap = device_cus() * (2048 / kBlock > 8 ? 8 : 2048 / kBlock);
  const int grid = A.rows < cap ? A.rows : cap;
  hipLaunchKernelGGL((rmsnorm2_kernel<kQuads, kBlock, kLong>), dim3(unsigned(grid)),
                     dim3(kBlock), 0, s, A);
  return check_launch("rmsnorm2_kernel");
}

}  // namespace
}  // namespace sufhip

using namespace sufhip;

extern "C" {

size_t sufhip_rmsnorm2_work_bytes(int rows, int cols) {
  if (rows < 1 || cols < 1 || rows > kMaxRows || cols > (1 << 20)) return 0;
  return rms_large(rows, cols) ? (size_t(rows) * 24 + 15) / 16 * 16 : 0;
}

int sufhip_rmsnorm2(const sufhip_rmsnorm2_args* args, void* stream) {
  const char* what = "sufhip_rmsnorm2";
  SUFHIP_REQUIRE(args, "sufhip_rmsnorm2: null args");
  const sufhip_rmsnorm2_args& g = *args;
  if (g.rows < 0 || g.cols < 0 || g.rows > kMaxRows || g.cols > (1 << 20))
    return ff_fail(what, "rows in [0, 2^24] and cols in [0, 2^20]");
  if (g.walk_count < 0 || (g.walk_count > 0 && (!g.walk_jobs || !g.walk_prg_state)))
    return ff_fail(what, "walk_jobs and walk_prg_state are needed for walk_count jobs");
  if (g.rows == 0 || g.cols == 0)  // the walks may be other operators' gates'
    return g.walk_count > 0
             ? sufhip_trunc_prepare_batch(g.walk_prg_state, g.walk_jobs, g.walk_count, stream)
             : SUFHIP_OK;
  const size_t n = size_t(g.rows) * size_t(g.cols);
  RmsArgs A{};
  A.rows = g.rows;
  A.cols = g.cols;
  A.inv_len = g.inv_len;
  A.eps = g.eps;
  if (int rc = mat2_of(g.x, g.rows, what, "x", &A.x)) return rc;
  if ((g.residual.p[0] == nullptr) != (g.residual.p[1] == nullptr))
    return ff_fail(what, "one share of the residual is missing");
  if (g.residual.p[0])
    if (int rc = mat2_of(g.residual, g.rows, what, "residual", &A.r)) return rc;
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
    if (bad_out_stride(outs[i].stride, g.rows, g.cols))
      return ff_fail(what, "output rows overlap, or lie more than 2^35 apart");
    const int p = g.total[0] && g.out[0] ? i / 2 : i;
    for (int q = 0; q < 2; ++q) {
      const RowSet in[2] = {row_set(A.x, q, g.rows, g.cols), row_set(A.r, q, g.rows, g.cols)};
      for (int k = 0; k < (A.r.p[0] ? 2 : 1); ++k)
        if (sets_meet(outs[i], in[k]) && !(p == q && same_set(outs[i], in[k])))
          return ff_fail(what, "an output meets x or the residual without being it");
    }
    for (int j = 0; j < i; ++j)
      if (sets_meet(outs[i], outs[j])) return ff_fail(what, "two outputs meet");
  }
  const size_t need = sufhip_rmsnorm2_work_bytes(g.rows, g.cols);
  if (need && (!g.d_work || (reinterpret_cast<uintptr_t>(g.d_work) & 15) != 0 ||
               g.work_bytes < need))
    return ff_fail(what, "the workspace is null, not 16-byte aligned or too small");
  const Range outd{A.digits, A.digits ? sufhip_digits2_bytes(g.rows, g.cols) : 0};
  const Range work{g.d_work, need};
  if (ranges_meet(outd, work)) return ff_fail(what, "out_digits meets the workspace");
  for (int i = 0; i < count; ++i)
    if (range_meets(outd, outs[i]) || range_meets(work, outs[i]))
      return ff_fail(what, "an output meets out_digits or the workspace");
  for (int q = 0; q < 2; ++q) {
    for (const RowSet& in : {row_set(A.x, q, g.rows, g.cols),
                             row_set(A.r, q, A.r.p[0] ? g.rows : 0, g.cols)})
      if (range_meets(outd, in) || range_meets(work, in))
        return ff_fail(what, "out_digits or the workspace meets an input");
    for (const Range& m : {Range{g.a[q], n * 8}, Range{g.ab[q], n * 8},
                           Range{g.a2[q], size_t(g.rows) * 8}, Range{g.b[q], size_t(g.rows) * 8},
                           Range{g.d_weight, size_t(g.cols) * 8}}) {
      bool bad = ranges_meet(outd, m) || ranges_meet(work, m);
      for (int i = 0; i < count; ++i) bad = bad || range_meets(m, outs[i]);
      if (bad) return ff_fail(what, "an output or the workspace meets the dealer's material");
    }
  }
  Material keys;
  for (int k = 0; k < kGates; ++k) keys.gate(A.tr[k]);
  keys.chain(A.rs, chain_products<SUFHIP_CHAIN_RSQRT>(), g.rsqrt.lut_key_bytes);
  bool bad = keys.meets(outd) || keys.meets(work);
  for (int i = 0; i < count; ++i) bad = bad || keys.meets(outs[i]);
  if (bad) return ff_fail(what, "an output or the workspace meets a gate, a LUT or a triple");
  hipStream_t s = as_stream(stream);
  if (need) {
    A.sums = static_cast<uint64_t*>(g.d_work);
    A.opens = A.sums + 2 * size_t(g.rows);
    RmsWalk w{};
    if (g.walk_count > 0) {
      size_t lanes = 0;  // room for a workgroup a CU
      if (int rc = plan_hosted_walk(g.walk_prg_state, g.walk_jobs, g.walk_count,
                                    size_t(device_cus()) * 256, stream, what, w.jobs, &lanes))
        return rc;
      w.groups = int((lanes + 255) / 256);
    }
    return launch_large(A, w, s);
  }
  if (g.walk_count > 0)
    if (int rc = sufhip_trunc_prepare_batch(g.walk_prg_state, g.walk_jobs, g.walk_count, stream))
      return rc;
  if (g.cols <= 1024) return launch_rms<1, 256, false>(A, s);
  // A row's latency counts where a CU has two at most (1 x 2048: 16.8 us, 19.4
  // with half the lanes), their number where it has more (1000 x 2048: 53 us, 61
  // with twice the lanes).
  if (g.cols <= 2048 && g.rows > 2 * device_cus()) return launch_rms<2, 256, false>(A, s);
  if (g.cols <= 2048) return launch_rms<1, 512, false>(A, s);
  if (g.cols <= 4096) return launch_rms<1, 1024, false>(A, s);
  return launch_rms<1, 1024, true>(A, s);
}

}  // extern "C"
