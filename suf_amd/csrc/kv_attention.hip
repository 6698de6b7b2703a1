// The two products of attention over a paged cache, both parties, exact mod
// 2^64 (sufhip_kv_scores2, sufhip_kv_values2).
//
// With D = (x_0 - a_0) + (x_1 - a_1) a party's share of a product is
//   Z_p = C_p + D B_p + L_p E,   L_0 = A_0 + D,  L_1 = A_1,
// E and B_p read from the cache's pages.
#include <hip/hip_runtime.h>

#include "kv_device.hpp"
#include "suf_hip.h"
#include "sufhip_internal.hpp"
#include "trunc_device.hpp"

namespace sufhip {
namespace {

constexpr int kBlock = 256;

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
  int64_t first;
  int len;
};
__device__ __forceinline__ Span span_of(const ProductArgs& a, int h, int t, int kv) {
  const int64_t r = int64_t(h) * a.b.tokens + t;
  const int64_t f = a.offsets[r], l = int64_t(a.offsets[r + 1]) - f;
  if (f < 0 || l <= 0 || f + l > a.n) return {0, 0};
  return {f, int(l < kv ? l : kv)};
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

__global__ void __launch_bounds__(kBlock) kv_scores2_kernel(ProductArgs a) {
  const EpiHdrs eh = epi_hdrs(a.epi);
  const int dim = a.pool.dim;
  for (int64_t row = blockIdx.y; row < int64_t(a.heads) * a.b.tokens; row += gridDim.y) {
    const int h = int(row / a.b.tokens), t = int(row - int64_t(h) * a.b.tokens);
    const int s = seq_of(a.b, t);
    if (s < 0) continue;
    const Span w = span_of(a, h, t, a.b.lens[s]);
    const uint64_t* x0 = a.x[0] + t * a.xts + h * a.xhs;
    const uint64_t* x1 = a.x[1] + t * a.xts + h * a.xhs;
    const int64_t q = (int64_t(t) * a.heads + h) * dim;
    for (int j = blockIdx.x * kBlock + threadIdx.x; j < w.len; j += gridDim.x * kBlock) {
      const int64_t i = w.first + j;
      uint64_t z0 = a.c[0][i], z1 = a.c[1][i];
      const int64_t k = kv_place(a.b, a.pool, s, h / a.group, j);
      if (k >= 0) {
        for (int d = 0; d < dim; ++d) {
          const uint64_t a0 = a.a[0][q + d], a1 = a.a[1][q + d];
          const uint64_t D = x0[d] - a0 + x1[d] - a1, E = a.pool.e[k + d];
          z0 += D * a.pool.b[0][k + d] + (a0 + D) * E;
          z1 += D * a.pool.b[1][k + d] + a1 * E;
        }
      }
      put2(a, eh, i, z0, z1);
    }
  }
}

__global__ void __launch_bounds__(kBlock) kv_values2_kernel(ProductArgs a) {
  const EpiHdrs eh = epi_hdrs(a.epi);
  const int dim = a.pool.dim;
  for (int64_t row = blockIdx.x; row < int64_t(a.heads) * a.b.tokens; row += gridDim.x) {
    const int h = int(row / a.b.tokens), t = int(row - int64_t(h) * a.b.tokens);
    const int s = seq_of(a.b, t);
    if (s < 0) continue;
    const Span w = span_of(a, h, t, a.b.lens[s]);
    const int64_t o = (int64_t(t) * a.heads + h) * dim;
    const int d = threadIdx.x;
    if (d >= dim) continue;
    uint64_t z0 = a.c[0][o + d], z1 = a.c[1][o + d];
    for (int j = 0; j < w.len; ++j) {
      const int64_t i = w.first + j;
      const int64_t k = kv_place(a.b, a.pool, s, h / a.group, j);
      if (k < 0) continue;
      const uint64_t a0 = a.a[0][i], a1 = a.a[1][i];
      const uint64_t D = a.x[0][i] - a0 + a.x[1][i] - a1, E = a.pool.e[k + d];
      z0 += D * a.pool.b[0][k + d] + (a0 + D) * E;
      z1 += D * a.pool.b[1][k + d] + a1 * E;
    }
    put2(a, eh, o + d, z0, z1);
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
  if (rows > 0x7fffffffu) return kv_fail(what, "at most 2^31 - 1 rows");
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

extern "C" {

int sufhip_kv_scores2(const sufhip_kv_product2_args* args, void* stream) {
  ProductArgs a{};
  bool empty = false;
  if (int rc = product_args(args, false, "sufhip_kv_scores2", &a, &empty)) return rc;
  if (empty) return SUFHIP_OK;
  const int64_t rows = int64_t(a.heads) * a.b.tokens;
  const int mk = args->batch.max_keys;
  const dim3 grid(unsigned(mk > kBlock ? (mk + kBlock - 1) / kBlock : 1),
                  unsigned(rows < 65535 ? rows : 65535));
  hipLaunchKernelGGL(kv_scores2_kernel, grid, dim3(kBlock), 0, as_stream(stream), a);
  return check_launch("kv_scores2_kernel");
}

size_t sufhip_kv_values2_work_bytes(const sufhip_kv_batch* batch, const sufhip_kv_pool* pool,
                                    int heads) {
  (void)batch;
  (void)pool;
  (void)heads;
  return 0;
}

int sufhip_kv_values2(const sufhip_kv_product2_args* args, void* stream) {
  ProductArgs a{};
  bool empty = false;
  if (int rc = product_args(args, true, "sufhip_kv_values2", &a, &empty)) return rc;
  if (empty) return SUFHIP_OK;
  const int64_t rows = int64_t(a.heads) * a.b.tokens;
  const dim3 grid(unsigned(rows < (1 << 20) ? rows : (1 << 20)));
  hipLaunchKernelGGL(kv_values2_kernel, grid, dim3(kBlock), 0, as_stream(stream), a);
  return check_launch("kv_values2_kernel");
}

}  // extern "C"
