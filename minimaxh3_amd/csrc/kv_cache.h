// Pages of an e4m3 cache of keys and values, as the kernels that write, read and attend to it address them.
#pragma once

#include "common.h"

namespace mxf8 {

// Exponents that a page's scale takes when it is written.  Their span, 95, is what lets the attention keep its
// probabilities scaled by the values' powers of two within fp32.
constexpr int KV_E_MIN = -32, KV_E_MAX = 63;

struct KvPages {
  const uint8_t *k, *v;    // codes [pages, H, page, D]
  const uint8_t *ks, *vs;  // exponent + 127, [pages, H]
  const int32_t* table;    // [B, width] page numbers
  int64_t table_stride, pages;
  int H, width, shift;  // page = 1 << shift tokens
};

// Entry i of sequence b, for an i that is the same for the whole wave: read through the scalar cache.
__device__ __forceinline__ int kv_entry(const KvPages& c, int b, int i) {
  typedef const __attribute__((address_space(4))) int32_t* consts;
  return ((consts)(uintptr_t)c.table)[b * c.table_stride + __builtin_amdgcn_readfirstlane(i)];
}
__device__ __forceinline__ bool kv_valid(const KvPages& c, int p) { return (uint32_t)p < (uint64_t)c.pages; }

// Page `i` of sequence b, or -1 where there is none (an entry that names no page of the pool counts as none).
__device__ __forceinline__ int kv_page(const KvPages& c, int b, int i) {
  const int p = c.table[b * c.table_stride + i];
  return kv_valid(c, p) ? p : -1;
}

// Tokens of sequence b that can be there: lengths beyond the table's pages, and negative ones, are cut.
__device__ __forceinline__ int kv_length(const KvPages& c, int64_t n) {
  const int64_t cap = (int64_t)c.width << c.shift;
  return (int)(n < 0 ? 0 : n < cap ? n : cap);
}

// 2^(e) of a scale byte
__device__ __forceinline__ float kv_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

int kv_check_pages(const char* what, const void* k, const void* v, const void* ks, const void* vs, int64_t pages,
                   int64_t H, int64_t page, int64_t D, const int32_t* table, int64_t table_stride, int64_t width,
                   int64_t B, KvPages* c);

}  // namespace mxf8
