// gr_paged.hip -- prebuilt instances of attention over a paged cache
// (gr_paged.h) behind gr_paged_attn().
#include <hip/hip_runtime.h>

#include <cstdint>

#include "gr_host.h"
#include "gr_overlap.h"
#include "gr_paged.h"
#include "gr_paged_host.h"
#include "grammar_rt.h"

namespace {

constexpr int imax(int a, int b) { return a > b ? a : b; }

template <int D, int BN, int NW, int KG, int NS, int KGS>
struct Lds {
  static constexpr int BYTES = imax(gr_paged_lds<D, BN, NW, KG, NS>::BYTES, KGS ? gr_paged_lds<D, 32, 1, KGS ? KGS : 1, 2>::BYTES : 0);
};

// One workgroup of four waves a CU where its LDS allows no two, else (and with
// eight waves) two waves a SIMD.
template <class T, int D, int BN, int NW, int KG, int NS, int KGS, bool SHARED>
__global__ __launch_bounds__(64 * NW * KG)
__attribute__((amdgpu_waves_per_eu(NW* KG == 4 && Lds<D, BN, NW, KG, NS, KGS>::BYTES > 80 * 1024 ? 1 : 2)))
void gr_paged_kernel(gr_paged_args a) {
  extern __shared__ __attribute__((aligned(16))) char gr_lds[];
  gr_paged_body<T, D, BN, NW, KG, NS, KGS, SHARED>(a, gr_lds);
}

template <class T, int D, int BM, bool SMALL>
__global__ __launch_bounds__(256) void gr_paged_merge_kernel(gr_paged_args a) {
  gr_paged_merge_body<T, D, BM, SMALL>(a);
}

// How a call is cut into workgroups.
struct Plan {
  int nw;                        // waves of 32 rows
  long long tiles;               // row tiles of a key head
  int groups;                    // key groups of a tile of 128 rows
  int shares;                    // 0: a workgroup a tile
};

Plan plan_of(const gr_paged_cache& c, const gr_paged_batch& b, int Hq) {
  Plan p;
  const int G = Hq / c.heads, D = c.head_dim;
  const long long most = b.starts && b.max_new > 0 && b.max_new < b.rows ? b.max_new : b.rows;
  const int cus = gr::cu_count() > 0 ? gr::cu_count() : 256;
  const long long cap = (long long)b.width * c.page_size;
  const long long len = b.max_len > 0 && b.max_len < cap ? b.max_len : cap;
  p.nw = most * G <= 32 ? 1 : most * G <= 64 ? 2 : 4;
  // Chunks whose tiles of 128 rows would leave most CUs idle take tiles of 64
  // with four key groups: 16 or 64 tiles (one chunk of 512, 4 key heads, G 1 or 4)
  // at 512 keys 13.0 us to 9.4 and 13.0 to 9.8 (D 64), 18.1 to 13.4 and 18.5 to
  // 14.1 (D 128). Over longer contexts, where keys are shared out anyway, only at D
  // 128 (16 tiles, 2,048 keys 30 to 22 us, 64 tiles, 8,192 keys 62 to 71).
  const long long rows128 = (b.starts ? (long long)b.rows : (long long)b.B * b.rows) * G / 128 * c.heads;
  if (p.nw == 4 && (len <= 1000 ? 4 * rows128 <= cus : D == 128 && 4 * rows128 < cus)) p.nw = 2;
  const int BM = 32 * p.nw;
  // packed rows: every sequence may have a part-filled tile
  p.tiles = b.starts ? (long long)b.rows * G / BM + b.B : (long long)b.B * (((long long)b.rows * G + BM - 1) / BM);
  const int resident = cus * (D == 128 && p.nw < 4 ? 1 : 2);      // workgroups (their LDS)
  // Tiles of 128 rows that leave a CU at most one of them halve the chain of their
  // key steps, with two key groups of four waves: 175 or 176 tiles, 1,500 keys 27.0
  // us to 23.0 (D 64), 44.5 to 36.0 (D 128); 256 tiles, 2,048 keys 33.8 to 28.8 and 57.0
  // to 46.2; 1,024 tiles 83.6 to 93.6 and 145 to 170. Single tokens beside them take a
  // workgroup each too: up to 7/4 of the CUs in all (400, D 64, 49.5 to 45.7; 528 24.0
  // to 27.0).
  const long long wgs = p.tiles * c.heads;
  p.groups = p.nw == 4 && rows128 <= cus && 4 * wgs <= 7LL * cus ? 2 : 1;
  // Work is shared out from a length on that grows with the workgroups that one a
  // tile would make: in brackets shared / a workgroup a tile, lengths spread by a
  // half around the mean. One token, D 128: 64 tiles, mean 600 keys 13.8 / 15.5 us,
  // 400 13.7 / 12.8; 256 tiles, 2,400 52.0 / 55.4, 1,200 32.5 / 31.2. D 64: 64
  // tiles, 1,200 12.7 / 16.3, 600 12.3 / 10.6; 512 tiles, 4,800 115.7 / 114.7. Tiles
  // of 128 rows in two groups: D 64, 16 tiles, 1,600 keys 18.8 / 21.7, 1,100 20.1 /
  // 18.1; 128 tiles, 4,500 44.4 / 49.4, 2,400 34.3 / 30.7; D 128, 96 tiles, 2,400 42.6 /
  // 49.5, 1,100 35.2 / 28.7; from three quarters of the CUs on not at all (176 tiles,
  // 8,000 87.8 / 82.7 and 162 / 144). In one group: 528 tiles, 16,384 keys 612 / 578.
  const double fill = wgs < resident ? (double)wgs / resident : 1.0;
  double least = D == 64 ? 1200 : 900, slope = D == 64 ? 7000 : 3000;
  bool can = true;
  if (p.nw == 4) {
    least = 1300;
    slope = p.groups == 1 ? 6500 : D == 64 ? 12500 : 8000;
    can = p.groups == 1 ? wgs < resident : 4 * wgs < 3LL * cus;
  }
  const double from = slope * fill > least ? slope * fill : least;
  const bool shared = can && (double)len > from && wgs * (cap / 64 + 1 + GR_PAGED_COST) <= 0x7fffffffLL;
  p.shares = !shared ? 0 : resident < GR_PAGED_MAX_SHARES ? resident : GR_PAGED_MAX_SHARES;
  return p;
}

size_t share_bytes(const Plan& p, int D) { return (size_t)2 * 32 * p.nw * (D + 2) * sizeof(float); }

// A workgroup a tile.
template <class T, int D, int BN, int NW, int KG, int NS, int KGS>
int launch_alone(const gr_paged_args& a, hipStream_t st) {
  constexpr int LDS = Lds<D, BN, NW, KG, NS, KGS>::BYTES;
  hipLaunchKernelGGL((gr_paged_kernel<T, D, BN, NW, KG, NS, KGS, false>), dim3((unsigned)((long long)a.tiles * a.Hkv)),
                     dim3(64 * NW * KG), LDS, st, a);
  return gr::hip_check(hipGetLastError(), GR_E_LAUNCH, "gr_paged_attn launch");
}

template <class T, int D, int BN, int NW, int KG, int NS, int KGS>
int launch_shared(const gr_paged_args& a, hipStream_t st) {
  constexpr int BM = 32 * NW, LDS = Lds<D, BN, NW, KG, NS, KGS>::BYTES;
  hipLaunchKernelGGL((gr_paged_kernel<T, D, BN, NW, KG, NS, KGS, true>), dim3((unsigned)a.shares), dim3(64 * NW * KG), LDS, st, a);
  const int rc = gr::hip_check(hipGetLastError(), GR_E_LAUNCH, "gr_paged_attn launch");
  if (rc) return rc;
  const long long wgs = (long long)a.tiles * a.Hkv;
  const int rows = a.starts ? BM : (a.rows * a.G < BM ? a.rows * a.G : BM);      // of a tile, at most
  // workgroups of a tile: one pass over its rows where it has few parts, and a
  // row each where few tiles of many parts would leave CUs idle
  const int few = (rows * D + 1023) / 1024, spare = (int)(1024 / wgs);
  const int y = few > spare ? few : spare < rows ? spare : rows;
  hipLaunchKernelGGL((gr_paged_merge_kernel<T, D, BM, (KGS > 0)>), dim3((unsigned)wgs, y), dim3(256), 0, st, a);
  return gr::hip_check(hipGetLastError(), GR_E_LAUNCH, "gr_paged_attn merge launch");
}

template <class T, int D>
int launch(const gr_paged_args& a, const Plan& p, hipStream_t st) {
  if (p.nw == 1) return a.shares ? launch_shared<T, D, 32, 1, 4, 2, 0>(a, st) : launch_alone<T, D, 32, 1, 4, 2, 0>(a, st);
  if (p.nw == 2) return a.shares ? launch_shared<T, D, 32, 2, 4, 2, 0>(a, st) : launch_alone<T, D, 32, 2, 4, 2, 0>(a, st);
  // (keys 32 a step in two groups at D 128: two rings of 64 would take a CU's LDS)
  if (a.shares) return launch_shared<T, D, 64, 4, 1, 2, D == 64 ? 4 : 2>(a, st);
  if (p.groups == 2) return launch_alone<T, D, D == 64 ? 64 : 32, 4, 2, 2, 4>(a, st);
  return launch_alone<T, D, 64, 4, 1, 2, D == 64 ? 4 : 2>(a, st);
}

int check_heads(const gr_paged_cache* c, const gr_paged_batch* b, int Hq) {
  if (Hq <= 0 || Hq % c->heads)
    return gr::fail(GR_E_ARG, "gr_paged_attn: %d query heads are not a multiple of the cache's %d", Hq, c->heads);
  const long long tokens = b->starts ? (long long)b->rows : (long long)b->B * b->rows;
  if (tokens * Hq >= (1LL << 30)) return gr::fail(GR_E_ARG, "gr_paged_attn: %lld tokens of %d heads are too many for one call", tokens, Hq);
  return GR_OK;
}

}  // namespace

extern "C" size_t gr_paged_attn_workspace(const gr_paged_cache* cache, const gr_paged_batch* batch, int Hq) {
  if (gr::check_paged(cache, batch, "gr_paged_attn_workspace") || check_heads(cache, batch, Hq) || batch->rows == 0) return 0;
  const Plan p = plan_of(*cache, *batch, Hq);
  return p.shares * share_bytes(p, cache->head_dim);
}

extern "C" int gr_paged_attn(const gr_paged_cache* cache, const gr_paged_batch* batch, const void* q, void* o, float* lse,
                             int Hq, const long long* q_strides, const long long* o_strides, int causal, float scale,
                             void* workspace, size_t workspace_bytes, void* stream) {
  int rc = gr::check_paged(cache, batch, "gr_paged_attn");
  if (rc || (rc = check_heads(cache, batch, Hq))) return rc;
  if (batch->rows == 0) return GR_OK;
  if (!q || !o || !q_strides || !o_strides) return gr::fail(GR_E_ARG, "gr_paged_attn: null argument");
  if (!gr::aligned16(q) || !gr::aligned16(o) || !gr::aligned16(workspace))
    return gr::fail(GR_E_ARG, "gr_paged_attn: base pointers must be 16-byte aligned");
  if ((uintptr_t)lse & 3) return gr::fail(GR_E_ARG, "gr_paged_attn: lse must be 4-byte aligned");
  for (int i = 0; i < 3; ++i)
    if (q_strides[i] < 0 || q_strides[i] % 8 || o_strides[i] < 0 || o_strides[i] % 8)
      return gr::fail(GR_E_ARG, "gr_paged_attn: strides must be non-negative multiples of 8 elements");
  if (!(scale > 0.f)) return gr::fail(GR_E_ARG, "gr_paged_attn: scale must be positive");
  {
    // o may be q (a tile's rows are read before its result is written) and nothing else
    const int B = batch->starts ? 1 : batch->B, N = batch->rows, D = cache->head_dim;
    const gr::strided qi = gr::heads_of(q, B, N, Hq, D, q_strides), oo = gr::heads_of(o, B, N, Hq, D, o_strides);
    const long long ks[3] = {cache->k_strides[0], cache->k_strides[2], cache->k_strides[1]};
    const long long vs[3] = {cache->v_strides[0], cache->v_strides[2], cache->v_strides[1]};
    if ((!gr::same_array(oo, qi) && gr::overlap(oo, qi, 2)) ||
        gr::overlap(oo, gr::heads_of(cache->k, cache->pages, cache->page_size, cache->heads, D, ks), 2) ||
        gr::overlap(oo, gr::heads_of(cache->v, cache->pages, cache->page_size, cache->heads, D, vs), 2))
      return gr::fail(GR_E_ARG, "gr_paged_attn: o shares memory with the cache or with q (it may be q, by the same strides)");
  }
  Plan p = plan_of(*cache, *batch, Hq);
  // as many shares as the workspace holds
  const size_t fit = workspace ? workspace_bytes / share_bytes(p, cache->head_dim) : 0;
  if ((size_t)p.shares > fit) p.shares = fit < 2 ? 0 : (int)fit;
  if (p.tiles * cache->heads > 0x7fffffffLL / 512) return gr::fail(GR_E_ARG, "gr_paged_attn: grid out of range");
  gr_paged_args a = {};
  a.q = q;
  a.o = o;
  a.lse = lse;
  a.q_sb = q_strides[0]; a.q_st = q_strides[1]; a.q_sh = q_strides[2];
  a.o_sb = o_strides[0]; a.o_st = o_strides[1]; a.o_sh = o_strides[2];
  a.k = cache->k;
  a.v = cache->v;
  a.k_sp = cache->k_strides[0]; a.k_sh = cache->k_strides[1]; a.k_ss = cache->k_strides[2];
  a.v_sp = cache->v_strides[0]; a.v_sh = cache->v_strides[1]; a.v_ss = cache->v_strides[2];
  a.table = batch->table;
  a.table_stride = batch->table_stride;
  a.lens = batch->lens;
  a.starts = batch->starts;
  a.B = batch->B;
  a.rows = batch->rows;
  a.width = batch->width;
  a.pages = cache->pages;
  a.page_shift = gr::page_shift(cache->page_size);
  a.Hq = Hq;
  a.Hkv = cache->heads;
  a.G = Hq / cache->heads;
  a.causal = causal;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.tiles = (int)p.tiles;
  a.shares = p.shares;
  if (p.shares) {
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = a.part_o + (size_t)p.shares * 2 * 32 * p.nw * cache->head_dim;
  }
  hipStream_t st = (hipStream_t)stream;
  if (cache->dtype == GR_F16)
    return cache->head_dim == 64 ? launch<_Float16, 64>(a, p, st) : launch<_Float16, 128>(a, p, st);
  return cache->head_dim == 64 ? launch<__bf16, 64>(a, p, st) : launch<__bf16, 128>(a, p, st);
}
