// The weighted sum of rows (sufhip_expert_mix2), both parties:
//   out[t] = trunc(sum_k weights[t][k] z[slots[t][k]]) + residual[t]
//
// A lane takes two neighbouring columns of a token; the row numbers and
// weights are the same for the whole wave's token mostly and come from the
// caches.  Memory bounds it.
#include <hip/hip_runtime.h>

#include "feedforward_device.hpp"

namespace sufhip {
namespace {

struct MixArgs {
  Mat2 z, res;
  int z_rows, tokens, each, cols;
  const int32_t* slots;
  const int64_t* weights;
  TruncEpi epi;
  uint64_t mask;
  uint64_t* out[2];
  int64_t out_stride;
};

typedef uint64_t u64x2u __attribute__((ext_vector_type(2), aligned(8)));

// Two neighbours from column c on, the second one if it is there.
__device__ __forceinline__ u64x2u load2(const uint64_t* p, bool two) {
  if (two) return *reinterpret_cast<const u64x2u*>(p);
  return u64x2u{p[0], 0};
}

// kLds: the gate's tables in LDS, for many outputs.
template <bool kLds>
__global__ void __launch_bounds__(kLds ? 1024 : 256, kLds ? 8 : 4) expert_mix2_kernel(MixArgs a) {
  __shared__ __align__(16) uint64_t tables[kLds ? sizeof(LdsGate) / 8 : 1];
  LdsGate& lds = reinterpret_cast<LdsGate&>(tables);
  if constexpr (kLds) {
    stage_gate(a.epi, lds);
    __syncthreads();
  }
  const EpiHdrs eh = epi_hdrs(a.epi);
  const uint32_t half = uint32_t(a.cols + 1) / 2;
  const size_t n = size_t(a.tokens) * half;
  for (size_t i = size_t(blockIdx.x) * blockDim.x + threadIdx.x; i < n;
       i += size_t(gridDim.x) * blockDim.x) {
    const int t = int(uint32_t(i) / half), c = 2 * int(uint32_t(i) % half);
    const bool two = c + 1 < a.cols;
    const int32_t* slots = a.slots + size_t(t) * a.each;
    const int64_t* weights = a.weights + size_t(t) * a.each;
    uint64_t y[2][2] = {};
    // Two rows at a time, their loads together; a row that is not there has
    // weight 0 and reads row 0.
    for (int k = 0; k < a.each; k += 2) {
      const int k1 = k + 1 < a.each ? k + 1 : k;
      int r0 = slots[k], r1 = slots[k1];
      uint64_t w0 = uint64_t(weights[k]), w1 = k1 > k ? uint64_t(weights[k1]) : 0;
      if (r0 < 0 || r0 >= a.z_rows) r0 = 0, w0 = 0;
      if (r1 < 0 || r1 >= a.z_rows) r1 = 0, w1 = 0;
      u64x2u v[2][2];
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        v[p][0] = load2(a.z.p[p] + int64_t(r0) * a.z.stride + c, two);
        v[p][1] = load2(a.z.p[p] + int64_t(r1) * a.z.stride + c, two);
      }
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int h = 0; h < 2; ++h) y[h][p] += w0 * v[p][0][h] + w1 * v[p][1][h];
    }
    u64x2u res[2] = {u64x2u{0, 0}, u64x2u{0, 0}};
    if (a.res.p[0]) {
#pragma unroll
      for (int p = 0; p < 2; ++p) res[p] = load2(a.res.p[p] + int64_t(t) * a.res.stride + c, two);
    }
    if (a.epi.on) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint64_t open = y[h][0] + y[h][1] + a.mask;
        if constexpr (kLds)
          gate2(a.epi, eh, lds, open, y[h]);
        else
          gate2(a.epi, eh, open, y[h]);
      }
    }
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      uint64_t* o = a.out[p] + int64_t(t) * a.out_stride + c;
      if (two) {
        *reinterpret_cast<u64x2u*>(o) = u64x2u{y[0][p] + res[p][0], y[1][p] + res[p][1]};
      } else {
        o[0] = y[0][p] + res[p][0];
      }
    }
  }
}

}  // namespace
}  // namespace sufhip

using namespace sufhip;

extern "C" int sufhip_expert_mix2(const sufhip_expert_mix2_args* args, void* stream) {
  const char* what = "sufhip_expert_mix2";
  SUFHIP_REQUIRE(args, "sufhip_expert_mix2: null args");
  const sufhip_expert_mix2_args& g = *args;
  if (g.tokens < 0 || g.cols < 0 || g.each < 0 || g.z_rows < 0 || g.tokens > kMaxRows ||
      g.z_rows > kMaxRows || g.each > 1024 ||
      uint64_t(g.tokens) * uint64_t(g.cols) >= (uint64_t(1) << 31))
    return ff_fail(what, "tokens and z_rows in [0, 2^24], each in [0, 1024], tokens cols < 2^31");
  if (g.tokens == 0 || g.cols == 0) return SUFHIP_OK;
  MixArgs a{};
  a.z_rows = g.z_rows;
  a.tokens = g.tokens;
  a.each = g.z_rows > 0 ? g.each : 0;  // without rows nothing is added
  a.cols = g.cols;
  a.slots = g.d_slots;
  a.weights = g.d_weights;
  if (g.each > 0 && (!g.d_slots || !g.d_weights)) return ff_fail(what, "null d_slots or d_weights");
  if (g.each > 0 && g.z_rows > 0)
    if (int rc = mat2_of(g.z, g.z_rows, what, "z", &a.z)) return rc;
  if (g.trunc)
    if (int rc = gate_of(*g.trunc, size_t(g.tokens) * g.cols, what, &a.epi)) return rc;
  a.mask = g.mask;
  if ((g.residual.p[0] == nullptr) != (g.residual.p[1] == nullptr))
    return ff_fail(what, "one share of the residual is missing");
  if (g.residual.p[0])
    if (int rc = mat2_of(g.residual, g.tokens, what, "residual", &a.res)) return rc;
  if (!g.out[0] || !g.out[1]) return ff_fail(what, "out is null");
  if (bad_out_stride(g.out_stride, g.tokens, g.cols))
    return ff_fail(what, "output rows overlap, or lie more than 2^35 apart");
  RowSet o[2];
  for (int p = 0; p < 2; ++p) {
    a.out[p] = g.out[p];
    o[p] = {g.out[p], g.out_stride, g.tokens, g.cols};
  }
  a.out_stride = g.out_stride;
  if (sets_meet(o[0], o[1])) return ff_fail(what, "the two shares of out meet");
  const size_t listed = size_t(g.tokens) * g.each;
  Material keys;
  keys.gate(a.epi);
  for (int p = 0; p < 2; ++p) {
    if (range_meets(Range{g.d_slots, listed * 4}, o[p]) ||
        range_meets(Range{g.d_weights, listed * 8}, o[p]))
      return ff_fail(what, "out meets the slots or the weights");
    if (keys.meets(o[p])) return ff_fail(what, "out meets the gate");
    for (int q = 0; q < 2; ++q) {
      if (a.z.p[0] && sets_meet(o[p], row_set(a.z, q, g.z_rows, g.cols)))
        return ff_fail(what, "out meets z");
      if (a.res.p[0]) {
        const RowSet r = row_set(a.res, q, g.tokens, g.cols);
        if (sets_meet(o[p], r) && !(p == q && same_set(o[p], r)))
          return ff_fail(what, "out meets the residual without being it");
      }
    }
  }
  const size_t n = size_t(g.tokens) * size_t((g.cols + 1) / 2);
  hipStream_t s = as_stream(stream);
  if (a.epi.on && a.epi.f <= kLdsGateBits && n >= (size_t(1) << 19)) {
    int dev = 0, cus = 256;
    if (hipGetDevice(&dev) == hipSuccess)
      (void)hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev);
    hipLaunchKernelGGL(expert_mix2_kernel<true>, dim3(unsigned(2 * cus)), dim3(1024), 0, s, a);
  } else {
    size_t grid = (n + 255) / 256;
    if (grid > 16384) grid = 16384;
    hipLaunchKernelGGL(expert_mix2_kernel<false>, dim3(unsigned(grid)), dim3(256), 0, s, a);
  }
  return check_launch("expert_mix2_kernel");
}
