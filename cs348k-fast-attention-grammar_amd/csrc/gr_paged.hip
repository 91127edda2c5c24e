// gr_paged.hip -- prebuilt instances of attention over a paged cache
// (gr_paged.h) behind gr_paged_attn().
#include <hip/hip_runtime.h>

#include "gr_paged_launch.h"

extern "C" size_t gr_paged_attn_workspace(const gr_paged_cache* cache, const gr_paged_batch* batch, int Hq) {
  return attn_workspace<false>(cache, nullptr, batch, Hq, "gr_paged_attn_workspace");
}

extern "C" int gr_paged_attn(const gr_paged_cache* cache, const gr_paged_batch* batch, const void* q, void* o, float* lse,
                             int Hq, const long long* q_strides, const long long* o_strides, int causal, float scale,
                             void* workspace, size_t workspace_bytes, void* stream) {
  return attn<false>(cache, nullptr, batch, q, o, lse, Hq, q_strides, o_strides, causal, scale, workspace, workspace_bytes, stream,
                     "gr_paged_attn");
}
