// gr_paged_host.h -- host-side checks shared by the entry points over a paged
// cache, of 16-bit rows or quantised.
#pragma once
#include <cstdint>

#include "gr_host.h"
#include "gr_overlap.h"
#include "grammar_rt.h"

namespace gr {

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

inline int page_shift(int size) { return __builtin_ctz((unsigned)size); }

// The cache and the batch of a call: pointers, sizes and alignment. What the
// device arrays hold (page ids, lengths, starts) is bounded by the kernels.
inline int check_paged(const gr_paged_cache* c, const gr_paged_batch* b, const char* who) {
  if (!c || !b || !c->k || !c->v || !b->table || !b->lens) return fail(GR_E_ARG, "%s: null argument", who);
  if (c->dtype != GR_F16 && c->dtype != GR_BF16)
    return fail(GR_E_ARG, "%s: dtype %d unsupported (GR_F16 or GR_BF16)", who, c->dtype);
  if (c->head_dim != 64 && c->head_dim != 128)
    return fail(GR_E_ARG, "%s: head dim %d unsupported (64 or 128)", who, c->head_dim);
  if (c->pages <= 0 || c->heads <= 0) return fail(GR_E_ARG, "%s: the cache needs pages and heads", who);
  if (c->page_size < 16 || c->page_size > (1 << 20) || (c->page_size & (c->page_size - 1)))
    return fail(GR_E_ARG, "%s: page size %d unsupported (a power of two from 16 to 2^20)", who, c->page_size);
  if (!aligned16(c->k) || !aligned16(c->v)) return fail(GR_E_ARG, "%s: base pointers must be 16-byte aligned (cache)", who);
  for (int i = 0; i < 3; ++i)
    if (c->k_strides[i] < 0 || c->k_strides[i] % 8 || c->v_strides[i] < 0 || c->v_strides[i] % 8)
      return fail(GR_E_ARG, "%s: strides must be non-negative multiples of 8 elements (cache)", who);
  // a kernel reaches the slots of 16 rows and their elements with a 32-bit byte offset
  if (c->k_strides[2] >= (1LL << 26) || c->v_strides[2] >= (1LL << 26))
    return fail(GR_E_ARG, "%s: slot strides must be below 2^26 elements", who);
  if (b->B <= 0 || b->rows < 0 || b->width <= 0 || b->table_stride < 0)
    return fail(GR_E_ARG, "%s: B and the page table's width must be positive", who);
  const long long tokens = b->starts ? (long long)b->rows : (long long)b->B * b->rows;
  if (tokens > 0x7fffffffLL) return fail(GR_E_ARG, "%s: %lld tokens are too many for one call", who, tokens);
  if ((long long)b->width * c->page_size > (1LL << 30))
    return fail(GR_E_ARG, "%s: a page table of %d pages of %d holds more than 2^30 keys", who, b->width, c->page_size);
  return GR_OK;
}

// The scales of a quantised cache, whose rows are bytes.
inline int check_scales(const gr_paged_cache* c, const gr_paged_scales* s, const char* who) {
  if (!s->scales) return fail(GR_E_ARG, "%s: null argument (scales)", who);
  if (!aligned16(s->scales)) return fail(GR_E_ARG, "%s: base pointers must be 16-byte aligned (scales)", who);
  for (int i = 0; i < 3; ++i) {
    if (s->strides[i] < 0 || s->strides[i] % 16)
      return fail(GR_E_ARG, "%s: strides must be non-negative multiples of 16 (scales)", who);
    if (c->k_strides[i] % 16 || c->v_strides[i] % 16)
      return fail(GR_E_ARG, "%s: strides must be multiples of 16 elements (quantised cache)", who);
  }
  return GR_OK;
}

// The same memory in single bytes, and a quantised cache's scales.
inline strided bytes_of(strided a, int size) {
  for (int i = 0; i < 3; ++i) a.s[i] *= size;
  a.n[3] *= size;
  return a;
}
inline strided scales_of(const gr_paged_cache* c, const gr_paged_scales* s) {
  return {s->scales, {c->pages, c->heads, 2, c->page_size}, {s->strides[0], s->strides[1], s->strides[2], 1}};
}

}  // namespace gr
