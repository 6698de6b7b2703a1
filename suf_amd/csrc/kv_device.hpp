// The packed batch and the paged pools of attention over a cache
// (sufhip_kv_batch, sufhip_kv_pool in suf_hip.h): device-side lookups and
// host-side argument checks, shared by the append (kv_cache.hip) and the
// products (kv_attention.hip).
//
// What stands in device memory (sequence starts, lengths, page numbers, row
// offsets) is not checked by the host.  Every lookup here is bounded by the
// arrays' host-side extents instead, so wrong contents give wrong values but
// no access outside the arrays.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <string>

#include "suf_hip.h"
#include "sufhip_internal.hpp"

namespace sufhip {

struct KvBatch {
  int seqs, tokens, max_pages;
  const int32_t* cu;
  const int32_t* lens;
  const int32_t* table;
};

struct KvPool {
  uint64_t* e;
  uint64_t* b[2];
  int pages, shift, heads, dim;  // page_tokens = 1 << shift
};

// Division of n < 2^31 by a launch-time constant d >= 1: n m / 2^(31 + s)
// with s = ceil(log2 d), m = floor(2^(31 + s) / d) + 1, exact for such n
// (the error n / 2^(31 + s) is below 1 / d).
struct FastDiv {
  uint32_t d, m, s;
};
inline FastDiv fast_div(uint32_t d) {
  uint32_t s = 0;
  while ((uint64_t(1) << s) < d) ++s;
  return {d, uint32_t((uint64_t(1) << (31 + s)) / d + 1), s};
}
__device__ __forceinline__ uint32_t div_by(const FastDiv& f, uint32_t n) {
  return uint32_t((uint64_t(n) * f.m) >> (31 + f.s));
}

// The sequence of packed token t, or -1 for a padding row.
__device__ __forceinline__ int seq_of(const KvBatch& b, int t) {
  int lo = 0, hi = b.seqs;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (b.cu[mid] <= t)
      lo = mid;
    else
      hi = mid;
  }
  return b.seqs > 0 && b.cu[lo] <= t && t < b.cu[lo + 1] ? lo : -1;
}

// First word of key j's head in a pool, or -1 when no page holds it.
__device__ __forceinline__ int64_t kv_place(const KvBatch& b, const KvPool& p, int s, int head,
                                            int64_t j) {
  const int64_t at = j >> p.shift;
  if (j < 0 || at >= b.max_pages) return -1;
  const int page = b.table[int64_t(s) * b.max_pages + at];
  if (page < 0 || page >= p.pages) return -1;
  const int64_t row = ((int64_t(page) * p.heads + head) << p.shift) + (j & ((1 << p.shift) - 1));
  return row * p.dim;
}

inline int kv_fail(const char* what, const char* msg) {
  set_error(std::string(what) + ": " + msg);
  return SUFHIP_ERR_INVALID;
}

inline int kv_batch_of(const sufhip_kv_batch& g, const char* what, KvBatch* out) {
  if (g.seqs < 0 || g.tokens < 0 || g.max_pages < 0 || g.max_new < 0 || g.max_keys < 0)
    return kv_fail(what, "seqs, tokens, max_pages, max_new and max_keys must be >= 0");
  if (g.seqs > 0 && g.tokens > 0 &&
      (!g.d_cu_tokens || !g.d_kv_lens || (g.max_pages > 0 && !g.d_pages)))
    return kv_fail(what, "null d_cu_tokens, d_kv_lens or d_pages");
  *out = {g.seqs, g.tokens, g.max_pages, g.d_cu_tokens, g.d_kv_lens, g.d_pages};
  return SUFHIP_OK;
}

inline int kv_pool_of(const sufhip_kv_pool& g, const char* what, KvPool* out) {
  if (!g.e || !g.b[0] || !g.b[1]) return kv_fail(what, "null pool array");
  if (g.pages < 0 || g.kv_heads < 1 || g.page_tokens < 1 ||
      (g.page_tokens & (g.page_tokens - 1)) || g.dim < 1 || g.dim > SUFHIP_KV_MAX_DIM)
    return kv_fail(what, "a pool needs pages >= 0, kv_heads >= 1, page_tokens a power of two and "
                         "1 <= dim <= 256");
  int shift = 0;
  while ((1 << shift) < g.page_tokens) ++shift;
  *out = {g.e, {g.b[0], g.b[1]}, g.pages, shift, g.kv_heads, g.dim};
  return SUFHIP_OK;
}

}  // namespace sufhip
