// gr_norm.hip -- prebuilt instances of normed and rotated heads (gr_rotary.h) and their
// gradient (gr_norm.h) behind gr_norm_rotary() and gr_norm_rotary_bwd().
#include <hip/hip_runtime.h>

#include "gr_norm.h"
#include "gr_rotary_host.h"

namespace {

template <class T, bool INTER>
__global__ __launch_bounds__(64 * GR_NORM_WAVES) void gr_norm_bwd_kernel(gr_norm_bwd_args a) {
  extern __shared__ float gr_norm_lds[];
  gr_norm_bwd_body<T, INTER>(a, gr_norm_lds);
}

template <class W>
__global__ __launch_bounds__(1024) void gr_norm_dw_kernel(const float* part, int n, int D, W* dwq, W* dwk) {
  gr_norm_dw_body<W>(part, n, D, dwq, dwk);
}

struct BwdPlan {
  int per, blocks;                // passes of a token that a wave takes, workgroups
};

BwdPlan bwd_plan(int rows, int D, long long tokens) {
  const int rpp = 64 / row_lanes(D), passes = (rows + rpp - 1) / rpp;
  const int cus = gr::cu_count() > 0 ? gr::cu_count() : 256;
  BwdPlan p;
  // all of a token's where that leaves every wave of the GPU two tokens, else fewer
  const long long waves = 2LL * cus * GR_NORM_WAVES, full = tokens * passes / (2 * waves);
  p.per = full < 1 ? 1 : full < passes ? (int)full : passes;
  const long long tasks = tokens * ((passes + p.per - 1) / p.per), all = (tasks + GR_NORM_WAVES - 1) / GR_NORM_WAVES;
  p.blocks = (int)(all < 2LL * cus ? all : 2LL * cus);
  return p;
}

template <class T, bool INTER>
int launch_bwd(const gr_norm_bwd_args& a, const BwdPlan& p, hipStream_t st) {
  const size_t lds = (size_t)GR_NORM_WAVES * 2 * a.D * sizeof(float);
  hipLaunchKernelGGL((gr_norm_bwd_kernel<T, INTER>), dim3(p.blocks), dim3(64 * GR_NORM_WAVES), lds, st, a);
  return gr::hip_check(hipGetLastError(), GR_E_LAUNCH, "gr_norm_rotary_bwd launch");
}

template <class W>
int launch_dw(const gr_norm_bwd_args& a, int n, void* dwq, void* dwk, hipStream_t st) {
  hipLaunchKernelGGL((gr_norm_dw_kernel<W>), dim3(2 * a.D / 16), dim3(1024), 0, st, a.part, n, a.D, (W*)dwq, (W*)dwk);
  return gr::hip_check(hipGetLastError(), GR_E_LAUNCH, "gr_norm_rotary_bwd weights launch");
}

}  // namespace

extern "C" int gr_norm_rotary(const gr_rotary_spec* rotary, const gr_head_norm* norm, const void* q, void* q_out, int Hq,
                              const long long* q_strides, const long long* q_out_strides, const void* k, void* k_out,
                              int Hk, const long long* k_strides, const long long* k_out_strides, int dtype, int B, int N,
                              const int* positions, const long long* position_strides, void* stream) {
  const char* const who = "gr_norm_rotary";
  gr_rope_args a = {};
  if (!norm) return gr::fail(GR_E_ARG, "gr_norm_rotary: null argument");
  int rc = take_heads(a, rotary, q, q_out, Hq, q_strides, q_out_strides, k, k_out, Hk, k_strides, k_out_strides, dtype, B, N,
                      positions, position_strides, who);
  if (rc || (rc = take_norm(a, norm, dtype, who))) return rc;
  const int D = rotary->head_dim, size = dtype == GR_F32 ? 4 : 2;
  if ((rc = check_weights(norm, D, gr::heads_of(q_out, B, N, Hq, D, q_out_strides), size, "q_out", who))) return rc;
  if (k && (rc = check_weights(norm, D, gr::heads_of(k_out, B, N, Hk, D, k_out_strides), size, "k_out", who))) return rc;
  hipStream_t st = (hipStream_t)stream;
  const bool inter = rotary->interleaved != 0;
  if (dtype == GR_F16) return launch_inter<_Float16, false, true>(a, inter, 0, who, st);
  if (dtype == GR_BF16) return launch_inter<__bf16, false, true>(a, inter, 0, who, st);
  return launch_inter<float, false, true>(a, inter, 0, who, st);
}

extern "C" size_t gr_norm_rotary_bwd_workspace(int Hq, int Hk, int head_dim, int B, int N) {
  if (Hq <= 0 || Hk < 0 || head_dim < 16 || head_dim > 256 || head_dim % 16 || B <= 0 || N <= 0) return 0;
  return (size_t)bwd_plan(Hq + Hk, head_dim, (long long)B * N).blocks * 2 * head_dim * sizeof(float);
}

extern "C" int gr_norm_rotary_bwd(const gr_rotary_spec* rotary, const gr_head_norm* norm, const void* q, const void* dq_out,
                                  void* dq, int Hq, const long long* q_strides, const long long* dq_out_strides,
                                  const long long* dq_strides, const void* k, const void* dk_out, void* dk, int Hk,
                                  const long long* k_strides, const long long* dk_out_strides, const long long* dk_strides,
                                  int dtype, int B, int N, const int* positions, const long long* position_strides,
                                  void* dq_weight, void* dk_weight, void* workspace, size_t workspace_bytes, void* stream) {
  const char* const who = "gr_norm_rotary_bwd";
  if (!norm) return gr::fail(GR_E_ARG, "gr_norm_rotary_bwd: null argument");
  gr_rope_args r = {}, g = {};
  // x to dx, and dy to dx: each pair is checked as a forward call's would be
  int rc = take_heads(r, rotary, q, dq, Hq, q_strides, dq_strides, k, dk, Hk, k_strides, dk_strides, dtype, B, N, positions,
                      position_strides, who);
  if (rc || (rc = take_norm(r, norm, dtype, who))) return rc;
  if ((rc = take_heads(g, rotary, dq_out, dq, Hq, dq_out_strides, dq_strides, k ? dk_out : nullptr, dk, Hk, dk_out_strides,
                       dk_strides, dtype, B, N, positions, position_strides, who)))
    return rc;
  if (k && !dk_out) return gr::fail(GR_E_ARG, "gr_norm_rotary_bwd: null argument (dk_out)");
  const int D = rotary->head_dim, size = dtype == GR_F32 ? 4 : 2, wsize = norm->dtype == GR_F32 ? 4 : 2;
  if (((uintptr_t)dq_weight & 3) || ((uintptr_t)dk_weight & 3))
    return gr::fail(GR_E_ARG, "gr_norm_rotary_bwd: the weights' gradients must be 4-byte aligned");
  const gr::strided to[2] = {gr::heads_of(dq, B, N, Hq, D, dq_strides), k ? gr::heads_of(dk, B, N, Hk, D, dk_strides) : gr::strided{}};
  for (int i = 0; i < (k ? 2 : 1); ++i) {
    if ((rc = check_weights(norm, D, to[i], size, i ? "dk" : "dq", who))) return rc;
    if (meets(dq_weight, D, wsize, to[i], size) || meets(dk_weight, D, wsize, to[i], size))
      return gr::fail(GR_E_ARG, "gr_norm_rotary_bwd: a weights' gradient shares memory with another output");
  }
  if (dk_weight && meets(dq_weight, D, wsize, {dk_weight, {1, 1, 1, D}, {0, 0, 0, 1}}, wsize))
    return gr::fail(GR_E_ARG, "gr_norm_rotary_bwd: a weights' gradient shares memory with another output");
  const BwdPlan p = bwd_plan(Hq + (k ? Hk : 0), D, (long long)B * N);
  gr_norm_bwd_args a = {};
  a.q = r.q;
  a.k = r.k;
  a.gq = g.q;
  a.gk = g.k;
  a.tokens = r.tokens;
  a.per_seq = r.per_seq;
  a.D = D;
  a.pairs = r.pairs;
  a.naxes = r.naxes;
  a.turns = r.turns;
  a.axes = r.axes;
  a.pos = r.pos;
  for (int i = 0; i < 3; ++i) a.ps[i] = r.ps[i];
  a.wq = r.wq;
  a.wk = r.wk;
  a.w32 = r.w32;
  a.eps = r.eps;
  a.per = p.per;
  const bool weights = dq_weight || dk_weight;
  if (weights) {
    if (!workspace || !gr::aligned16(workspace) || workspace_bytes < (size_t)p.blocks * 2 * D * sizeof(float))
      return gr::fail(GR_E_ARG, "gr_norm_rotary_bwd: the weights' gradients need a 16-byte aligned workspace of %zu bytes, not %zu",
                      (size_t)p.blocks * 2 * D * sizeof(float), workspace ? workspace_bytes : 0);
    a.part = static_cast<float*>(workspace);
  }
  hipStream_t st = (hipStream_t)stream;
  const bool inter = rotary->interleaved != 0;
  if (dtype == GR_F16) rc = inter ? launch_bwd<_Float16, true>(a, p, st) : launch_bwd<_Float16, false>(a, p, st);
  else if (dtype == GR_BF16) rc = inter ? launch_bwd<__bf16, true>(a, p, st) : launch_bwd<__bf16, false>(a, p, st);
  else rc = inter ? launch_bwd<float, true>(a, p, st) : launch_bwd<float, false>(a, p, st);
  if (rc || !weights) return rc;
  if (norm->dtype == GR_F32) return launch_dw<float>(a, p.blocks, dq_weight, dk_weight, st);
  if (dtype == GR_F16) return launch_dw<_Float16>(a, p.blocks, dq_weight, dk_weight, st);
  return launch_dw<__bf16>(a, p.blocks, dq_weight, dk_weight, st);
}
