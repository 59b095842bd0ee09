// kv4.cuh — the paged 4-bit key/value cache: what kv4_append.cu and kv4_attention.cu share.
//
// k and v are int4 [pages, kv_heads, page, dim], two per byte, low nibble first (the format of the int4 weights), and
// k_scale and v_scale f16 [pages, kv_heads, page, dim / group]: a cached value is nibble * scale. The tokens that a
// head keeps on a page are contiguous, so a page of one head is one run of page * dim / 2 bytes.
#pragma once

#include "common.cuh"

namespace up {
namespace kv4 {

constexpr int64_t kMaxPage = 4096;
constexpr int64_t kMaxDim = 256;

// What every entry asks of a cache: dims and groups in whole 32-dimension chunks (16 bytes), pages a power of two of at
// least 8 tokens (so that 8 tokens' scales are 16-byte runs too), 16-byte aligned arrays.
inline int check_cache(const up_kv4_cache* c) {
  UP_CHECK_ARG(c != nullptr && c->pages >= 0 && c->kv_heads > 0);
  if (c->dim <= 0 || c->dim % 32 != 0 || c->dim > kMaxDim) return UP_ERR_UNSUPPORTED;
  if (c->group <= 0 || c->group % 32 != 0 || c->dim % c->group != 0) return UP_ERR_UNSUPPORTED;
  if (c->page < 8 || c->page > kMaxPage || (c->page & (c->page - 1)) != 0) return UP_ERR_UNSUPPORTED;
  if (c->kv_heads > 0xffff || c->pages > 0x7fffffff) return UP_ERR_UNSUPPORTED;
  if (c->pages == 0) return UP_OK;
  UP_CHECK_ARG(c->k != nullptr && c->v != nullptr && c->k_scale != nullptr && c->v_scale != nullptr);
  UP_CHECK_ARG(aligned(c->k, 16) && aligned(c->v, 16) && aligned(c->k_scale, 16) && aligned(c->v_scale, 16));
  return UP_OK;
}

inline int log2_of(int64_t pow2) {
  int n = 0;
  while (((int64_t)1 << n) < pow2) ++n;
  return n;
}

}  // namespace kv4
}  // namespace up
