// gr_paged_read.hip -- prebuilt instances of reading a paged cache back
// (gr_paged_read.h) behind gr_paged_read().
#include <hip/hip_runtime.h>

#include "gr_host.h"
#include "gr_overlap.h"
#include "gr_paged_host.h"
#include "gr_paged_read.h"
#include "grammar_rt.h"

namespace {

template <class T, int D, bool Q8>
__global__ __launch_bounds__(256) void gr_paged_read_kernel(gr_read_args a) {
  gr_paged_read_body<T, D, Q8>(a);
}

template <class T, int D, bool Q8>
int launch(gr_read_args& a, hipStream_t st) {
  constexpr int RPW = gr_read_rows(D);
  a.chunks = (a.rows + RPW - 1) / RPW;
  const long long places = a.starts ? a.chunks : (long long)a.B * a.chunks;
  const int cus = gr::cu_count() > 0 ? gr::cu_count() : 256;
  const long long run = places * a.heads / (16LL * cus);
  a.per_wave = run < 1 ? 1 : run > a.heads ? a.heads : (int)run;
  const long long waves = places * ((a.heads + a.per_wave - 1) / a.per_wave);
  if (waves > 0x7fffffffLL / 64) return gr::fail(GR_E_ARG, "gr_paged_read: %lld rows are too many for one call", places * RPW);
  hipLaunchKernelGGL((gr_paged_read_kernel<T, D, Q8>), dim3((unsigned)((waves + 3) / 4)), dim3(256), 0, st, a);
  return gr::hip_check(hipGetLastError(), GR_E_LAUNCH, "gr_paged_read launch");
}

template <class T, bool Q8>
int launch_dim(gr_read_args& a, int D, hipStream_t st) {
  return D == 64 ? launch<T, 64, Q8>(a, st) : launch<T, 128, Q8>(a, st);
}

}  // namespace

extern "C" int gr_paged_read(const gr_paged_cache* cache, const gr_paged_scales* scales, const gr_paged_batch* batch, void* k_out,
                             void* v_out, const long long* k_strides, const long long* v_strides, void* stream) {
  const char* const who = "gr_paged_read";
  int rc = gr::check_paged(cache, batch, who);
  if (rc || (scales && (rc = gr::check_scales(cache, scales, who)))) return rc;
  if (batch->rows == 0) return GR_OK;
  if (!k_out || !v_out || !k_strides || !v_strides) return gr::fail(GR_E_ARG, "gr_paged_read: null argument");
  if (!gr::aligned16(k_out) || !gr::aligned16(v_out)) return gr::fail(GR_E_ARG, "gr_paged_read: base pointers must be 16-byte aligned");
  for (int i = 0; i < 3; ++i)
    if (k_strides[i] < 0 || k_strides[i] % 8 || v_strides[i] < 0 || v_strides[i] % 8)
      return gr::fail(GR_E_ARG, "gr_paged_read: strides must be non-negative multiples of 8 elements");
  {
    const int B = batch->starts ? 1 : batch->B, N = batch->rows, D = cache->head_dim, H = cache->heads;
    const long long ks[3] = {cache->k_strides[0], cache->k_strides[2], cache->k_strides[1]};
    const long long vs[3] = {cache->v_strides[0], cache->v_strides[2], cache->v_strides[1]};
    const gr::strided ko = gr::heads_of(k_out, B, N, H, D, k_strides), vo = gr::heads_of(v_out, B, N, H, D, v_strides);
    const gr::strided kc = gr::heads_of(cache->k, cache->pages, cache->page_size, H, D, ks);
    const gr::strided vc = gr::heads_of(cache->v, cache->pages, cache->page_size, H, D, vs);
    const int size = scales ? 1 : 2;
    bool bad = gr::overlap(ko, vo, 2);
    for (const gr::strided& o : {gr::bytes_of(ko, 2), gr::bytes_of(vo, 2)})
      bad |= gr::overlap(o, gr::bytes_of(kc, size), 1) || gr::overlap(o, gr::bytes_of(vc, size), 1) ||
             (scales && gr::overlap(o, gr::scales_of(cache, scales), 1));
    if (bad) return gr::fail(GR_E_ARG, "gr_paged_read: k_out and v_out share memory with each other or the cache");
  }
  gr_read_args a = {};
  a.k = cache->k;
  a.v = cache->v;
  a.ksp = cache->k_strides[0]; a.ksh = cache->k_strides[1]; a.kss = cache->k_strides[2];
  a.vsp = cache->v_strides[0]; a.vsh = cache->v_strides[1]; a.vss = cache->v_strides[2];
  if (scales) {
    a.scales = static_cast<const unsigned char*>(scales->scales);
    a.sp = scales->strides[0]; a.sh = scales->strides[1]; a.skind = scales->strides[2];
  }
  a.ko = k_out;
  a.vo = v_out;
  a.kb = k_strides[0]; a.kt = k_strides[1]; a.kh = k_strides[2];
  a.vb = v_strides[0]; a.vt = v_strides[1]; a.vh = v_strides[2];
  a.table = batch->table;
  a.table_stride = batch->table_stride;
  a.lens = batch->lens;
  a.starts = batch->starts;
  a.B = batch->B;
  a.rows = batch->rows;
  a.width = batch->width;
  a.pages = cache->pages;
  a.page_shift = gr::page_shift(cache->page_size);
  a.heads = cache->heads;
  hipStream_t st = (hipStream_t)stream;
  const int D = cache->head_dim;
  if (!scales) return launch_dim<_Float16, false>(a, D, st);      // (copied bit by bit, whichever type)
  return cache->dtype == GR_F16 ? launch_dim<_Float16, true>(a, D, st) : launch_dim<__bf16, true>(a, D, st);
}
