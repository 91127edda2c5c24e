// gr_paged8.hip -- prebuilt instances of attention over a quantised paged cache
// (gr_paged.h) behind gr_paged_attn_scaled().
#include <hip/hip_runtime.h>

#include "gr_paged_launch.h"

extern "C" size_t gr_paged_attn_scaled_workspace(const gr_paged_cache* cache, const gr_paged_scales* scales,
                                                 const gr_paged_batch* batch, int Hq) {
  if (!scales) return 0;
  return attn_workspace<true>(cache, scales, batch, Hq, "gr_paged_attn_scaled_workspace");
}

extern "C" int gr_paged_attn_scaled(const gr_paged_cache* cache, const gr_paged_scales* scales, const gr_paged_batch* batch,
                                    const void* q, void* o, float* lse, int Hq, const long long* q_strides,
                                    const long long* o_strides, int causal, float scale, void* workspace, size_t workspace_bytes,
                                    void* stream) {
  if (!scales) return gr::fail(GR_E_ARG, "gr_paged_attn_scaled: null argument");
  return attn<true>(cache, scales, batch, q, o, lse, Hq, q_strides, o_strides, causal, scale, workspace, workspace_bytes, stream,
                    "gr_paged_attn_scaled");
}
