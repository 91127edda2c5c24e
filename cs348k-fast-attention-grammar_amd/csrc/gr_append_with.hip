// gr_append_with.hip -- prebuilt instances of gr_rope_body that append normed rows,
// quantised rows or both, behind gr_paged_append_with().
#include <hip/hip_runtime.h>

#include "gr_rotary_host.h"

namespace {

template <class T>
int dispatch(const gr_rope_args& a, bool norm, bool q8, bool inter, const char* who, hipStream_t st) {
  if (q8) return norm ? launch_inter<T, true, true, true>(a, inter, 0, who, st) : launch_inter<T, true, false, true>(a, inter, 0, who, st);
  return launch_inter<T, true, true>(a, inter, 0, who, st);
}

}  // namespace

extern "C" int gr_paged_append_with(const gr_paged_cache* cache, const gr_paged_scales* scales, const gr_paged_batch* batch,
                                    const gr_rotary_spec* rotary, const gr_head_norm* norm, const void* q, void* q_out, int Hq,
                                    const long long* q_strides, const long long* q_out_strides, const void* k, const void* v,
                                    const long long* k_strides, const long long* v_strides, const int* positions,
                                    const long long* position_strides, void* stream) {
  if (!scales && !norm)
    return gr_paged_append(cache, batch, rotary, q, q_out, Hq, q_strides, q_out_strides, k, v, k_strides, v_strides, positions,
                           position_strides, stream);
  const char* const who = "gr_paged_append_with";
  gr_rope_args a = {};
  const int rc = take_append(a, cache, scales, batch, rotary, norm, q, q_out, Hq, q_strides, q_out_strides, k, v, k_strides,
                             v_strides, positions, position_strides, who);
  if (rc || a.tokens == 0) return rc;
  hipStream_t st = (hipStream_t)stream;
  const bool inter = rotary && rotary->interleaved != 0;
  if (cache->dtype == GR_F16) return dispatch<_Float16>(a, norm, scales, inter, who, st);
  return dispatch<__bf16>(a, norm, scales, inter, who, st);
}
