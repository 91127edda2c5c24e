// gr_rotary.hip -- prebuilt instances of the position rotation (gr_rotary.h)
// behind gr_rotary() and gr_paged_append().
#include <hip/hip_runtime.h>

#include "gr_rotary_host.h"

extern "C" int gr_rotary(const gr_rotary_spec* rotary, const void* q, void* q_out, int Hq, const long long* q_strides,
                         const long long* q_out_strides, const void* k, void* k_out, int Hk, const long long* k_strides,
                         const long long* k_out_strides, int dtype, int B, int N, const int* positions,
                         const long long* position_strides, int inverse, void* stream) {
  const char* const who = "gr_rotary";
  gr_rope_args a = {};
  const int rc = take_heads(a, rotary, q, q_out, Hq, q_strides, q_out_strides, k, k_out, Hk, k_strides, k_out_strides, dtype, B, N,
                            positions, position_strides, who);
  if (rc) return rc;
  hipStream_t st = (hipStream_t)stream;
  const bool inter = rotary->interleaved != 0;
  if (dtype == GR_F16) return launch_inter<_Float16, false>(a, inter, inverse, who, st);
  if (dtype == GR_BF16) return launch_inter<__bf16, false>(a, inter, inverse, who, st);
  return launch_inter<float, false>(a, inter, inverse, who, st);
}

extern "C" int gr_paged_append(const gr_paged_cache* cache, const gr_paged_batch* batch, const gr_rotary_spec* rotary,
                               const void* q, void* q_out, int Hq, const long long* q_strides,
                               const long long* q_out_strides, const void* k, const void* v,
                               const long long* k_strides, const long long* v_strides, const int* positions,
                               const long long* position_strides, void* stream) {
  const char* const who = "gr_paged_append";
  gr_rope_args a = {};
  const int rc = take_append(a, cache, nullptr, batch, rotary, nullptr, q, q_out, Hq, q_strides, q_out_strides, k, v, k_strides,
                             v_strides, positions, position_strides, who);
  if (rc || a.tokens == 0) return rc;
  hipStream_t st = (hipStream_t)stream;
  const bool inter = rotary && rotary->interleaved != 0;
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
