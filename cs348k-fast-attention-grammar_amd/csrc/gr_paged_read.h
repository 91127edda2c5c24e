// gr_paged_read.h -- a paged cache's sequences as dense keys and values.
//
// Row j of a sequence comes from slot j % S of page table[j / S], a quantised one as
// its e4m3 numbers times its power of two, which v_cvt_scalef32_pk gives exactly where T holds
// them and rounded to nearest below T's normal range.
//
// Layout: D / 8 lanes have a row, 8 elements each, so that a store instruction writes
// whole lines. A wave takes the 512 / D rows of one place for a run of heads, keys and
// values of UN heads asked for at once; page ids and lengths are read once for all. Bound by
// memory: six contexts of 3,000 to 21,000 keys, 8 heads of 128, quantised (429 MB, two thirds
// of it written past the caches) take 86 us, 5.0 TB/s; three of 100 to 500 keys, 8 heads of
// 64, 3.6, a launch and three dependent trips (length, page id, rows).
#pragma once
#include "gr_common.h"
#include "gr_e4m3.h"

struct gr_read_args {
  const void *k, *v;
  long long ksp, ksh, kss, vsp, vsh, vss;   // page, head, slot (elements)
  const unsigned char* scales;
  long long sp, sh, skind;
  void *ko, *vo;
  long long kb, kt, kh, vb, vt, vh;         // batch, token, head
  const int* table;
  long long table_stride;
  const int* lens;
  const int* starts;
  int B, rows, width, pages, page_shift;
  int heads, per_wave;                      // heads of the cache, and of a wave
  int chunks;                               // places: of a sequence (uniform batches), or of all rows
};

// Rows of a place.
constexpr int gr_read_rows(int D) { return 512 / D; }

template <class T, int D, bool Q8>
__device__ __forceinline__ void gr_paged_read_body(const gr_read_args& a) {
  constexpr int LPR = D / 8, RPW = gr_read_rows(D), UN = Q8 ? 4 : 2;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)((blockIdx.x * blockDim.x + threadIdx.x) >> 6));
  const int runs = (a.heads + a.per_wave - 1) / a.per_wave;
  const int place = wave / runs, h0 = (wave - place * runs) * a.per_wave;
  const int h1 = gr_imin(h0 + a.per_wave, a.heads);
  const int c = lane % LPR;
  // this lane's row: its sequence, its key, and where it goes
  int b, j, row;
  if (a.starts) {
    const int first = place * RPW;
    if (first >= a.rows) return;
    row = first + lane / LPR;
    int ends = 0;                                // sequences that end at or before the place's first row
    for (int b0 = 0; b0 < a.B; b0 += 64)
      ends += __builtin_popcountll(__builtin_amdgcn_ballot_w64(b0 + lane < a.B && a.starts[gr_imin(b0 + lane, a.B - 1) + 1] <= first));
    b = ends;
    while (b < a.B && a.starts[b + 1] <= row) ++b;
    if (row >= a.rows || b >= a.B) return;
    const int s0 = a.starts[b], s1 = a.starts[b + 1];
    if (row < s0 || s0 < 0 || s1 > a.rows) return;
    j = row - s0;
  } else {
    b = place / a.chunks;
    if (b >= a.B) return;
    row = j = (place - b * a.chunks) * RPW + lane / LPR;
    if (row >= a.rows) return;
  }
  long long page = -1;
  const int pi = j >> a.page_shift, slot = j & ((1 << a.page_shift) - 1);
  if (j < a.lens[b] && pi < a.width) {
    const int id = a.table[b * a.table_stride + pi];
    if (id >= 0 && id < a.pages) page = id;
  }
  const long long at = page < 0 ? 0 : page;
  const int bo = a.starts ? 0 : b;
  typedef typename gr_bytes<Q8>::type E;         // element of the cache: a byte, or 16 bits
  const E* const ks = static_cast<const E*>(a.k) + at * a.ksp + slot * a.kss + 8 * c;
  const E* const vs = static_cast<const E*>(a.v) + at * a.vsp + slot * a.vss + 8 * c;
  const unsigned char* const ss = Q8 ? a.scales + at * a.sp + slot : nullptr;
  T* const kd = static_cast<T*>(a.ko) + bo * a.kb + row * a.kt + 8 * c;
  T* const vd = static_cast<T*>(a.vo) + bo * a.vb + row * a.vt + 8 * c;
#pragma unroll 1
  for (int h = h0; h < h1; h += UN) {
    gr_u32x4 x[2 * UN];
    unsigned sb[2 * UN];
#pragma unroll
    for (int i = 0; i < 2 * UN; ++i) {
      x[i] = (gr_u32x4){0, 0, 0, 0};
      sb[i] = 0;
      if (page >= 0 && h + i / 2 < h1) {
        const E* const s = i & 1 ? vs + (h + i / 2) * a.vsh : ks + (h + i / 2) * a.ksh;
        if constexpr (Q8) {
          const gr_u32x2 w = *reinterpret_cast<const gr_u32x2*>(s);
          x[i][0] = w[0];
          x[i][1] = w[1];
          sb[i] = ss[(h + i / 2) * a.sh + (i & 1 ? a.skind : 0)];
        } else {
          x[i] = gr_ld16(s);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 2 * UN; ++i) {
      if (h + i / 2 >= h1) break;
      gr_u32x4 w = x[i];
      if constexpr (Q8) {
        const float scale = gr_e8m0(sb[i]);
        w = (gr_u32x4){gr_from_e4m3<T, false>(x[i][0], scale), gr_from_e4m3<T, true>(x[i][0], scale),
                       gr_from_e4m3<T, false>(x[i][1], scale), gr_from_e4m3<T, true>(x[i][1], scale)};
      }
      __builtin_nontemporal_store(w, reinterpret_cast<gr_u32x4*>(i & 1 ? vd + (h + i / 2) * a.vh : kd + (h + i / 2) * a.kh));
    }
  }
}
