// gr_rotary.hip -- prebuilt instances of the position rotation (gr_rotary.h)
// behind gr_rotary() and gr_paged_append().
#include <hip/hip_runtime.h>

#include <cstdint>

#include "gr_host.h"
#include "gr_overlap.h"
#include "gr_paged_host.h"
#include "gr_rotary.h"
#include "grammar_rt.h"

namespace {

template <class T, bool APPEND, bool INTER, int ITER, bool PAST>
__global__ __launch_bounds__(256) void gr_rope_kernel(gr_rope_args a, int inverse) {
  gr_rope_body<T, APPEND, INTER, ITER, PAST>(a, inverse != 0);
}

template <class T, bool APPEND, bool INTER, bool PAST>
int launch(const gr_rope_args& a, int inverse, const char* who, hipStream_t st) {
  const int rows = a.q.heads + a.k.heads + a.v.heads;
  const int rpp = 64 / (a.D / 16), passes = (rows + rpp - 1) / rpp;
  // Passes to a wave. One while two would leave a CU fewer than 4 waves (128 tokens
  // of 64 heads of 128 3.8 us, two 4.0; 1,024 tokens of 48 7.8 and 6.8). Else four,
  // or two of 16-bit rows of 128 and more (two / four, 8,192 tokens: 64 heads of 96
  // 42.5 / 33.8 us, 48 of 64 22.3 / 19.2, 32 of 128 in fp32 46.6 / 43.9; 64 of 128
  // 43.3 / 49.0, 48 of 128 33.2 / 32.7).
  const long long full = (long long)a.tokens * passes;
  const int cus = gr::cu_count() > 0 ? gr::cu_count() : 256;
  const int iter = passes < 2 || full < 8LL * cus ? 1 : passes == 2 || (sizeof(T) == 2 && a.D >= 128) ? 2 : 4;
  const long long waves = (long long)a.tokens * ((passes + iter - 1) / iter);
  if (waves > 0x7fffffffLL / 64) return gr::fail(GR_E_ARG, "%s: %d tokens of %d head rows are too many for one call", who, a.tokens, rows);
  const dim3 grid((unsigned)((waves + 3) / 4));
  if constexpr (!PAST) {
    if (iter == 4) {
      hipLaunchKernelGGL((gr_rope_kernel<T, APPEND, INTER, 4, false>), grid, dim3(256), 0, st, a, inverse);
      return gr::hip_check(hipGetLastError(), GR_E_LAUNCH, who);
    }
  }
  if (iter == 2) hipLaunchKernelGGL((gr_rope_kernel<T, APPEND, INTER, 2, PAST>), grid, dim3(256), 0, st, a, inverse);
  else hipLaunchKernelGGL((gr_rope_kernel<T, APPEND, INTER, 1, PAST>), grid, dim3(256), 0, st, a, inverse);
  return gr::hip_check(hipGetLastError(), GR_E_LAUNCH, who);
}

// Whether every row of a destination begins on a 128-byte line (16-bit elements).
bool on_lines(const gr_rope_rows& k) {
  return k.heads == 0 || (((uintptr_t)k.dst & 127) == 0 && ((k.db | k.dt | k.dh) & 63) == 0);
}

template <class T, bool APPEND>
int launch_inter(const gr_rope_args& a, bool inter, int inverse, const char* who, hipStream_t st) {
  if (inter) return launch<T, APPEND, true, false>(a, inverse, who, st);
  if constexpr (sizeof(T) == 2) {
    // whole lines: 8 lanes of 16 bytes side by side, in the rotated part and behind it,
    // of rows that begin on a line (2 x 4,096 tokens of 32 + 32 heads of 128: 43.7 us, rows
    // 16 bytes off a line 50.5 and past the caches 93.5, 64 off 45.5 and 47.8)
    if (2 * a.pairs % 128 == 0 && a.D % 128 == 0 && on_lines(a.q) && on_lines(a.k) && on_lines(a.v))
      return launch<T, APPEND, false, true>(a, inverse, who, st);
  }
  return launch<T, APPEND, false, false>(a, inverse, who, st);
}

// An output may be its own input, and shares no other memory with the call's
// arrays: the waves of a token read and write its heads in no order.
int check_apart(const gr::strided& out, const gr::strided& own, const gr::strided* others, int n, int size, const char* name,
                const char* who) {
  bool bad = !gr::same_array(out, own) && gr::overlap(out, own, size);
  for (int i = 0; i < n; ++i) bad |= gr::overlap(out, others[i], size);
  return bad ? gr::fail(GR_E_ARG, "%s: %s shares memory with another array (it may be its own input, by the same strides)", who, name)
             : GR_OK;
}

// The rotation's own arguments: head_dim a multiple of 16 up to 256, at most 8 axes.
int take_rotary(gr_rope_args& a, const gr_rotary_spec* r, const char* who) {
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

int take_rows(gr_rope_rows& k, const void* src, void* dst, int heads, const long long* ss, const long long* ds,
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

}  // namespace

extern "C" int gr_rotary(const gr_rotary_spec* rotary, const void* q, void* q_out, int Hq, const long long* q_strides,
                         const long long* q_out_strides, const void* k, void* k_out, int Hk, const long long* k_strides,
                         const long long* k_out_strides, int dtype, int B, int N, const int* positions,
                         const long long* position_strides, int inverse, void* stream) {
  const char* const who = "gr_rotary";
  if (!rotary || !positions || !position_strides) return gr::fail(GR_E_ARG, "gr_rotary: null argument");
  if (B <= 0 || N <= 0 || (long long)B * N > 0x7fffffffLL) return gr::fail(GR_E_ARG, "gr_rotary: B and N must be positive, B N below 2^31");
  gr_rope_args a = {};
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
  hipStream_t st = (hipStream_t)stream;
  const bool inter = rotary->interleaved != 0;
  if (dtype == GR_F16) return launch_inter<_Float16, false>(a, inter, inverse, who, st);
  if (dtype == GR_BF16) return launch_inter<__bf16, false>(a, inter, inverse, who, st);
  if (dtype == GR_F32) return launch_inter<float, false>(a, inter, inverse, who, st);
  return gr::fail(GR_E_ARG, "gr_rotary: dtype %d unsupported (GR_F16, GR_BF16 or GR_F32)", dtype);
}

extern "C" int gr_paged_append(const gr_paged_cache* cache, const gr_paged_batch* batch, const gr_rotary_spec* rotary,
                               const void* q, void* q_out, int Hq, const long long* q_strides,
                               const long long* q_out_strides, const void* k, const void* v,
                               const long long* k_strides, const long long* v_strides, const int* positions,
                               const long long* position_strides, void* stream) {
  const char* const who = "gr_paged_append";
  gr_rope_args a = {};
  int rc = gr::check_paged(cache, batch, who);
  if (rc) return rc;
  if (batch->rows == 0) return GR_OK;
  if (!k || !v || (positions && !position_strides)) return gr::fail(GR_E_ARG, "gr_paged_append: null argument");
  const gr_rotary_spec none = {nullptr, nullptr, 0, 1, cache->head_dim, 0};
  const gr_rotary_spec* r = rotary ? rotary : &none;
  if (rotary && (rc = take_rotary(a, rotary, who))) return rc;
  if (r->head_dim != cache->head_dim)
    return gr::fail(GR_E_ARG, "gr_paged_append: the rotation's head dim %d is not the cache's %d", r->head_dim, cache->head_dim);
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
    if ((rc = check_apart(gr::heads_of(q_out, B, N, Hq, D, q_out_strides), gr::heads_of(q, B, N, Hq, D, q_strides), others, 4, 2,
                          "q_out", who)))
      return rc;
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
  hipStream_t st = (hipStream_t)stream;
  const bool inter = r->interleaved != 0;
  if (cache->dtype == GR_F16) return launch_inter<_Float16, true>(a, inter, 0, who, st);
  return launch_inter<__bf16, true>(a, inter, 0, who, st);
}

extern "C" int gr_selftest_overlap(const void* a, const long long* a_sizes, const long long* a_strides, const void* b,
                                   const long long* b_sizes, const long long* b_strides, int size) {
  gr::strided x = {a, {}, {}}, y = {b, {}, {}};
  for (int i = 0; i < 4; ++i) {
    x.n[i] = a_sizes[i]; x.s[i] = a_strides[i];
    y.n[i] = b_sizes[i]; y.s[i] = b_strides[i];
  }
  return gr::overlap(x, y, size);
}
