// gr_rotary_host.h -- what the entry points that rotate heads (gr_rotary, gr_norm_rotary,
// the appends) share on the host: checks of arguments, and the launch of
// gr_rope_body's instances, which each translation unit makes for itself.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "gr_host.h"
#include "gr_overlap.h"
#include "gr_paged_host.h"
#include "gr_rotary.h"
#include "grammar_rt.h"

namespace {

// Lanes of a row that is reduced (gr_row_lanes).
inline int row_lanes(int D) {
  int n = 1;
  while (16 * n < D) n *= 2;
  return n;
}

template <class T, bool APPEND, bool INTER, int ITER, bool PAST, bool NORM, bool Q8>
__global__ __launch_bounds__(256) void gr_rope_kernel(gr_rope_args a, int inverse) {
  gr_rope_body<T, APPEND, INTER, ITER, PAST, NORM, Q8>(a, inverse != 0);
}

// ITER passes to a wave.
template <class T, bool APPEND, bool INTER, bool PAST, bool NORM, bool Q8, int ITER>
int launch_iter(const gr_rope_args& a, int passes, int inverse, const char* who, hipStream_t st) {
  const long long waves = (long long)a.tokens * ((passes + ITER - 1) / ITER);
  if (waves > 0x7fffffffLL / 64)
    return gr::fail(GR_E_ARG, "%s: %d tokens of %d head rows are too many for one call", who, a.tokens, a.q.heads + a.k.heads + a.v.heads);
  hipLaunchKernelGGL((gr_rope_kernel<T, APPEND, INTER, ITER, PAST, NORM, Q8>), dim3((unsigned)((waves + 3) / 4)), dim3(256), 0, st, a, inverse);
  return gr::hip_check(hipGetLastError(), GR_E_LAUNCH, who);
}

template <class T, bool APPEND, bool INTER, bool PAST, bool NORM, bool Q8>
int launch(const gr_rope_args& a, int inverse, const char* who, hipStream_t st) {
  const int rows = a.q.heads + a.k.heads + a.v.heads;
  const int rpp = 64 / (NORM || Q8 ? row_lanes(a.D) : a.D / 16), passes = (rows + rpp - 1) / rpp;
  // Passes to a wave. One while two would leave a CU fewer than 4 waves (128 tokens
  // of 64 heads of 128 3.8 us, two 4.0; 1,024 tokens of 48 7.8 and 6.8). Else four,
  // or two of 16-bit rows of 128 and more (two / four, 8,192 tokens: 64 heads of 96
  // 42.5 / 33.8 us, 48 of 64 22.3 / 19.2, 32 of 128 in fp32 46.6 / 43.9; 64 of 128
  // 43.3 / 49.0, 48 of 128 33.2 / 32.7).
  const long long full = (long long)a.tokens * passes;
  const int cus = gr::cu_count() > 0 ? gr::cu_count() : 256;
  int iter = passes < 2 || full < 8LL * cus ? 1 : passes == 2 || (sizeof(T) == 2 && a.D >= 128) ? 2 : 4;
  if constexpr (NORM || Q8) {
    // Rows that are normed or quantised have more to compute for a token and a pass: up to
    // five, shared out evenly. Norm of 2 x 4,096 tokens of 32 + 8 heads of 128 (10 passes) in
    // twos 37.5 us, up to three 34.3, fives 30.8; 9,668 tokens of 48 heads of 128 (6) into a
    // quantised cache in twos 56.6, threes 47.7.
    const int groups = (passes + 4) / 5;
    iter = full < 8LL * cus ? 1 : (passes + groups - 1) / groups;
    if (iter == 5) return launch_iter<T, APPEND, INTER, PAST, NORM, Q8, 5>(a, passes, inverse, who, st);
    if (iter == 4) return launch_iter<T, APPEND, INTER, PAST, NORM, Q8, 4>(a, passes, inverse, who, st);
    if (iter == 3) return launch_iter<T, APPEND, INTER, PAST, NORM, Q8, 3>(a, passes, inverse, who, st);
  } else if constexpr (!PAST) {
    if (iter == 4) return launch_iter<T, APPEND, INTER, false, false, false, 4>(a, passes, inverse, who, st);
  }
  if (iter == 2) return launch_iter<T, APPEND, INTER, PAST, NORM, Q8, 2>(a, passes, inverse, who, st);
  return launch_iter<T, APPEND, INTER, PAST, NORM, Q8, 1>(a, passes, inverse, who, st);
}

// Whether every row of a destination begins on a 128-byte line (16-bit elements).
inline bool on_lines(const gr_rope_rows& k) {
  return k.heads == 0 || (((uintptr_t)k.dst & 127) == 0 && ((k.db | k.dt | k.dh) & 63) == 0);
}

template <class T, bool APPEND, bool NORM = false, bool Q8 = false>
int launch_inter(const gr_rope_args& a, bool inter, int inverse, const char* who, hipStream_t st) {
  if (inter) return launch<T, APPEND, true, false, NORM, Q8>(a, inverse, who, st);
  if constexpr (sizeof(T) == 2) {
    // whole lines: 8 lanes of 16 bytes side by side, in the rotated part and behind it,
    // of rows that begin on a line (2 x 4,096 tokens of 32 + 32 heads of 128: 43.7 us, rows
    // 16 bytes off a line 50.5 and past the caches 93.5, 64 off 45.5 and 47.8)
    if (2 * a.pairs % 128 == 0 && a.D % 128 == 0 && on_lines(a.q) &&
        (Q8 || (on_lines(a.k) && on_lines(a.v))))
      return launch<T, APPEND, false, true, NORM, Q8>(a, inverse, who, st);
  }
  return launch<T, APPEND, false, false, NORM, Q8>(a, inverse, who, st);
}

// An output may be its own input, and shares no other memory with the call's
// arrays: the waves of a token read and write its heads in no order.
inline int check_apart(const gr::strided& out, const gr::strided& own, const gr::strided* others, int n, int size, const char* name,
                const char* who) {
  bool bad = !gr::same_array(out, own) && gr::overlap(out, own, size);
  for (int i = 0; i < n; ++i) bad |= gr::overlap(out, others[i], size);
  return bad ? gr::fail(GR_E_ARG, "%s: %s shares memory with another array (it may be its own input, by the same strides)", who, name)
             : GR_OK;
}

// The rotation's own arguments: head_dim a multiple of 16 up to 256, at most 8 axes.
inline int take_rotary(gr_rope_args& a, const gr_rotary_spec* r, const char* who) {
  if (!r->turns || ((uintptr_t)r->turns & 7)) return gr::fail(GR_E_ARG, "%s: the rotation's turns must be an 8-byte aligned buffer", who);
  if (r->head_dim < 16 || r->head_dim > 256 || r->head_dim % 16)
    return gr::fail(GR_E_ARG, "%s: head dim %d unsupported (a multiple of 16 up to 256)", who, r->head_dim);
  if (r->pairs < 8 || r->pairs % 8 || 2 * r->pairs > r->head_dim)
    return gr::fail(GR_E_ARG, "%s: %d rotated pairs unsupported (a multiple of 8, at most half the head dim)", who, r->pairs);
  if (r->naxes < 1 || r->naxes > 8) return gr::fail(GR_E_ARG, "%s: %d position axes unsupported (1 to 8)", who, r->naxes);
  if (r->naxes > 1 && (!r->axes || ((uintptr_t)r->axes & 7)))
    return gr::fail(GR_E_ARG, "%s: the pairs' axes must be an 8-byte aligned buffer", who);
  a.D = r->head_dim;
  a.pairs = r->pairs;
  a.naxes = r->naxes;
  a.turns = reinterpret_cast<const unsigned long long*>(r->turns);
  a.axes = r->axes;
  return GR_OK;
}

inline int take_rows(gr_rope_rows& k, const void* src, void* dst, int heads, const long long* ss, const long long* ds,
              const char* name, const char* who) {
  if (!src || !dst || !ss || !ds) return gr::fail(GR_E_ARG, "%s: null argument (%s)", who, name);
  if (heads <= 0) return gr::fail(GR_E_ARG, "%s: %s needs at least one head", who, name);
  if (!gr::aligned16(src) || !gr::aligned16(dst)) return gr::fail(GR_E_ARG, "%s: base pointers must be 16-byte aligned (%s)", who, name);
  for (int i = 0; i < 3; ++i)
    if (ss[i] < 0 || ss[i] % 8 || ds[i] < 0 || ds[i] % 8)
      return gr::fail(GR_E_ARG, "%s: strides must be non-negative multiples of 8 elements (%s)", who, name);
  k = {src, dst, ss[0], ss[1], ss[2], ds[0], ds[1], ds[2], heads};
  return GR_OK;
}

// The arguments of a rotation of dense heads, checked.
inline int take_heads(gr_rope_args& a, const gr_rotary_spec* rotary, const void* q, void* q_out, int Hq,
                      const long long* q_strides, const long long* q_out_strides, const void* k, void* k_out, int Hk,
                      const long long* k_strides, const long long* k_out_strides, int dtype, int B, int N,
                      const int* positions, const long long* position_strides, const char* who) {
  if (!rotary || !positions || !position_strides) return gr::fail(GR_E_ARG, "%s: null argument", who);
  if (B <= 0 || N <= 0 || (long long)B * N > 0x7fffffffLL) return gr::fail(GR_E_ARG, "%s: B and N must be positive, B N below 2^31", who);
  if (dtype != GR_F16 && dtype != GR_BF16 && dtype != GR_F32)
    return gr::fail(GR_E_ARG, "%s: dtype %d unsupported (GR_F16, GR_BF16 or GR_F32)", who, dtype);
  int rc = take_rotary(a, rotary, who);
  if (rc) return rc;
  if ((rc = take_rows(a.q, q, q_out, Hq, q_strides, q_out_strides, "q", who))) return rc;
  if (k && (rc = take_rows(a.k, k, k_out, Hk, k_strides, k_out_strides, "k", who))) return rc;
  const int D = rotary->head_dim, size = dtype == GR_F32 ? 4 : 2;
  const gr::strided qi = gr::heads_of(q, B, N, Hq, D, q_strides), qo = gr::heads_of(q_out, B, N, Hq, D, q_out_strides);
  if (!k) {
    if ((rc = check_apart(qo, qi, nullptr, 0, size, "q_out", who))) return rc;
  } else {
    const gr::strided ki = gr::heads_of(k, B, N, Hk, D, k_strides), ko = gr::heads_of(k_out, B, N, Hk, D, k_out_strides);
    const gr::strided not_q[2] = {ki, ko};
    if ((rc = check_apart(qo, qi, not_q, 2, size, "q_out", who)) || (rc = check_apart(ko, ki, &qi, 1, size, "k_out", who))) return rc;
  }
  a.tokens = B * N;
  a.per_seq = N;
  a.pos = positions;
  for (int i = 0; i < 3; ++i) a.ps[i] = position_strides[i];
  return GR_OK;
}

// Whether a vector of weights shares memory with heads.
inline bool meets(const void* w, int D, int wsize, const gr::strided& heads, int size) {
  return w && gr::overlap({w, {1, 1, 1, (long long)D * wsize}, {0, 0, 0, 1}}, gr::bytes_of(heads, size), 1);
}

// Heads that a call writes are none of its norm's weights.
inline int check_weights(const gr_head_norm* n, int D, const gr::strided& out, int size, const char* name, const char* who) {
  const int wsize = n->dtype == GR_F32 ? 4 : 2;
  return meets(n->q_weight, D, wsize, out, size) || meets(n->k_weight, D, wsize, out, size)
             ? gr::fail(GR_E_ARG, "%s: %s shares memory with the norm's weights", who, name)
             : GR_OK;
}

// A norm's weights, in fp32 or in the rows' type.
inline int take_norm(gr_rope_args& a, const gr_head_norm* n, int dtype, const char* who) {
  if (!gr::aligned16(n->q_weight) || !gr::aligned16(n->k_weight))
    return gr::fail(GR_E_ARG, "%s: the norm's weights must be 16-byte aligned", who);
  if (n->dtype != GR_F32 && n->dtype != dtype)
    return gr::fail(GR_E_ARG, "%s: the norm's weights must be GR_F32 or of the rows' type, not %d", who, n->dtype);
  if (!(n->eps >= 0.f) || !(n->eps < 1e30f)) return gr::fail(GR_E_ARG, "%s: the norm's eps must not be negative", who);
  a.wq = n->q_weight;
  a.wk = n->k_weight;
  a.w32 = n->dtype == GR_F32;
  a.eps = n->eps;
  return GR_OK;
}

// An append's arguments, checked; scales and norm NULL where there are none.
inline int take_append(gr_rope_args& a, const gr_paged_cache* cache, const gr_paged_scales* scales, const gr_paged_batch* batch,
                       const gr_rotary_spec* rotary, const gr_head_norm* norm, const void* q, void* q_out, int Hq,
                       const long long* q_strides, const long long* q_out_strides, const void* k, const void* v,
                       const long long* k_strides, const long long* v_strides, const int* positions,
                       const long long* position_strides, const char* who) {
  int rc = gr::check_paged(cache, batch, who);
  if (rc || (scales && (rc = gr::check_scales(cache, scales, who)))) return rc;
  if (batch->rows == 0) return GR_OK;
  if (!k || !v || (positions && !position_strides)) return gr::fail(GR_E_ARG, "%s: null argument", who);
  const gr_rotary_spec none = {nullptr, nullptr, 0, 1, cache->head_dim, 0};
  const gr_rotary_spec* r = rotary ? rotary : &none;
  if (rotary && (rc = take_rotary(a, rotary, who))) return rc;
  if (norm && (rc = take_norm(a, norm, cache->dtype, who))) return rc;
  if (r->head_dim != cache->head_dim)
    return gr::fail(GR_E_ARG, "%s: the rotation's head dim %d is not the cache's %d", who, r->head_dim, cache->head_dim);
  a.D = cache->head_dim;
  a.naxes = r->naxes;
  if (q && (rc = take_rows(a.q, q, q_out, Hq, q_strides, q_out_strides, "q", who))) return rc;
  // a cache's strides are {page, head, slot}
  const long long kd[3] = {cache->k_strides[0], cache->k_strides[2], cache->k_strides[1]};
  const long long vd[3] = {cache->v_strides[0], cache->v_strides[2], cache->v_strides[1]};
  if ((rc = take_rows(a.k, k, cache->k, cache->heads, k_strides, kd, "k", who))) return rc;
  if ((rc = take_rows(a.v, v, cache->v, cache->heads, v_strides, vd, "v", who))) return rc;
  if (q) {
    const int B = batch->starts ? 1 : batch->B, N = batch->rows, D = cache->head_dim;
    const gr::strided others[4] = {
        gr::heads_of(k, B, N, cache->heads, D, k_strides), gr::heads_of(v, B, N, cache->heads, D, v_strides),
        gr::heads_of(cache->k, cache->pages, cache->page_size, cache->heads, D, kd),
        gr::heads_of(cache->v, cache->pages, cache->page_size, cache->heads, D, vd)};
    const gr::strided qo = gr::heads_of(q_out, B, N, Hq, D, q_out_strides), qi = gr::heads_of(q, B, N, Hq, D, q_strides);
    if ((rc = check_apart(qo, qi, others, scales ? 2 : 4, 2, "q_out", who))) return rc;
    if (scales) {
      const gr::strided bytes = gr::bytes_of(qo, 2);
      if (gr::overlap(bytes, others[2], 1) || gr::overlap(bytes, others[3], 1) || gr::overlap(bytes, gr::scales_of(cache, scales), 1))
        return gr::fail(GR_E_ARG, "%s: q_out shares memory with the cache", who);
    }
    if (norm && (rc = check_weights(norm, D, qo, 2, "q_out", who))) return rc;
  }
  a.tokens = batch->starts ? batch->rows : batch->B * batch->rows;
  a.per_seq = batch->starts ? 1 : batch->rows;
  a.pos = positions;
  if (positions)
    for (int i = 0; i < 3; ++i) a.ps[i] = position_strides[i];
  a.table = batch->table;
  a.table_stride = batch->table_stride;
  a.width = batch->width;
  a.pages = cache->pages;
  a.page_shift = gr::page_shift(cache->page_size);
  a.B = batch->B;
  a.lens = batch->lens;
  a.starts = batch->starts;
  if (scales) {
    a.scales = static_cast<unsigned char*>(scales->scales);
    a.sp = scales->strides[0];
    a.sh = scales->strides[1];
    a.skind = scales->strides[2];
  }
  return GR_OK;
}

}  // namespace
