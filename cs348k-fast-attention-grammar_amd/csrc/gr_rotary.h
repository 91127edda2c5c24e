// gr_rotary.h -- rotation of query and key heads by position, alone or on the
// way into a paged key/value cache.
//
// Pair j of a head, (x1, x2), becomes (x1 cos t - x2 sin t, x1 sin t + x2 cos t)
// with t = pos f_j, f_j an angle per position; the gradient is the rotation by
// -t. Nothing is tabulated: f_j comes as a whole number of 2^-64 turns, so that
// pos f_j modulo a turn is one wrapping integer product, off by what f_j was rounded
// to that whole number (pos 2^-65 turns: 2^-34 of a turn at position 2^31), of which
// the upper 32 bits are used (less than 2^-32 of a turn, 1.5e-9 radians, at any
// position). In fp32 the angle of position 200,000 would be off by 2^-7. A table of sines
// would be read once a token, as this is computed once a token, but holds a
// fixed number of positions per axis.
//
// Layout: a wave takes one token and ITER passes over its head rows. A head is
// D / 16 units of 8 + 8 elements (two 16-byte accesses in fp16 / bf16): 8 pairs,
// or 8 elements of each half of what is behind the rotated part. Lane l has unit
// l % (D / 16) of row l / (D / 16) of every pass, so its 8 sines and cosines serve
// all of its rows. The rows of all passes are requested before the angles are
// computed.
//
// Bound by memory once there are tokens enough: 2 x 4,096 tokens of 32 + 32 heads
// of 128 (268 MB, bf16) take 43-52 us, 5.2-6.2 TB/s, where a large copy reaches
// 5.15; 320 tokens of 4 + 4 heads of 64 take 4.0 us, a launch and two trips to
// memory.
//
// Stores that write whole lines go past the caches, where the attention that
// reads the rows runs on other XCDs: 8,193 tokens of 32 + 8 + 8 heads of 128 into
// pages 45.5 us to 41.3, 1,024 tokens 7.6 to 6.6, and the attention behind takes as
// long. Stores of parts of lines stay in them: 2 x 4,096 tokens of 32 + 32 heads of
// 32 take 15.0 us, past the caches 30; of 128 with neighbours as pairs 45.5 and 76, in
// rows that begin 16 bytes off a line 50.5 and 93.5.
#pragma once
#include "gr_common.h"

// One kind of head rows: strides in elements, {batch, token, head} of the source
// and {batch or (into a cache) page, token or slot, head} of the destination.
struct gr_rope_rows {
  const void* src;
  void* dst;
  long long sb, st, sh, db, dt, dh;
  int heads;
};

struct gr_rope_args {
  gr_rope_rows q, k, v;          // v: append only (heads 0 else)
  int tokens, per_seq;           // all tokens; tokens of a sequence (uniform batches)
  int D, pairs, naxes;
  const unsigned long long* turns;
  const unsigned char* axes;
  const int* pos;                // strides {axis, batch, token}; nullptr (append): the token's place in its sequence
  long long ps[3];
  // append
  const int* table;
  long long table_stride;
  int width, pages, page_shift, B;
  const int* lens;
  const int* starts;             // nullptr: uniform batch
};

// sin and cos of 2 pi h 2^-32: the nearest quarter turn off exactly in
// integers, the rest (at most pi / 4) by the Taylor sums to x^9 and x^10, whose
// next terms are 1.8e-9 and 1.2e-10; the argument's rounding is 2^-23 of it.
__device__ __forceinline__ void gr_turn_sincos(unsigned h, float& s, float& c) {
  const unsigned q = (h + 0x20000000u) >> 30;
  const float x = (float)(int)(h - (q << 30)) * 1.4629180792671596e-9f;   // 2 pi 2^-32
  const float y = x * x;
  const float sn = fmaf(x * y, fmaf(y, fmaf(y, fmaf(y, 2.7557319224e-6f, -1.9841269841e-4f), 8.3333333333e-3f),
                                    -1.6666666667e-1f), x);
  const float cs = fmaf(y, fmaf(y, fmaf(y, fmaf(y, fmaf(y, -2.7557319224e-7f, 2.4801587302e-5f), -1.3888888889e-3f),
                                        4.1666666667e-2f), -0.5f), 1.0f);
  const float a = (q & 1) ? cs : sn, b = (q & 1) ? sn : cs;
  s = (q & 2) ? -a : a;
  c = ((q + 1) & 2) ? -b : b;
}

// 8 elements as they are in memory.
template <class T>
struct gr_rope8 {
  static constexpr int W = sizeof(T) / 2;    // 16-byte words
  gr_u32x4 w[W];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] = gr_ld16(reinterpret_cast<const char*>(p) + 16 * i);
  }
  template <bool PAST>
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      char* const at = reinterpret_cast<char*>(p) + 16 * i;
      if constexpr (PAST) __builtin_nontemporal_store(w[i], reinterpret_cast<gr_u32x4*>(at));
      else gr_st16(at, w[i]);
    }
  }
  __device__ __forceinline__ float get(int e) const {
    if constexpr (W == 2) {
      const unsigned u = w[e >> 2][e & 3];   // (a bit cast of the element itself reads element 0)
      return __builtin_bit_cast(float, u);
    } else {
      const unsigned u = w[0][e >> 1];
      return (float)__builtin_bit_cast(T, (unsigned short)((e & 1) ? u >> 16 : u & 0xffffu));
    }
  }
  // elements e and e + 1 (e even), rounded to T once
  __device__ __forceinline__ void put2(int e, float a, float b) {
    if constexpr (W == 2) {
      w[e >> 2][e & 3] = __builtin_bit_cast(unsigned, a);
      w[(e + 1) >> 2][(e + 1) & 3] = __builtin_bit_cast(unsigned, b);
    } else {
      w[0][e >> 1] = gr_pack2f<T>(a, b);
    }
  }
};

// PAST: stores go past the caches (of whole 128-byte lines only)
template <class T, bool APPEND, bool INTER, int ITER, bool PAST>
__device__ __forceinline__ void gr_rope_body(const gr_rope_args& a, bool inverse) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)((blockIdx.x * blockDim.x + threadIdx.x) >> 6));
  const int units = a.D >> 4;                    // of a head row
  const int rpp = 64 / units;                    // rows a pass
  const int h0 = a.q.heads, h1 = h0 + a.k.heads, rows = h1 + (APPEND ? a.v.heads : 0);
  const int passes = (rows + rpp - 1) / rpp, groups = (passes + ITER - 1) / ITER;
  const int tok = wave / groups;
  if (tok >= a.tokens) return;
  const int row0 = (wave - tok * groups) * ITER * rpp + lane / units, u = lane % units;
  const int ru = a.pairs >> 3;                   // rotated units
  const bool lane_live = lane < rpp * units;
  const int lo = u < ru ? (INTER ? 16 * u : 8 * u) : 2 * a.pairs + 8 * (u - ru);
  const int hi = u < ru ? (INTER ? 16 * u + 8 : a.pairs + 8 * u) : lo + 8 * (units - ru);

  // the token's sequence and index in it
  int b, i, at = 0;
  if (APPEND && a.starts) {
    int ends = 0;                                // sequences that end at or before this token
    for (int b0 = 0; b0 < a.B; b0 += 64)
      ends += __builtin_popcountll(__builtin_amdgcn_ballot_w64(b0 + lane < a.B && a.starts[gr_imin(b0 + lane, a.B - 1) + 1] <= tok));
    if (ends >= a.B) return;                     // behind the last sequence
    b = ends;
    const int s0 = a.starts[b], s1 = a.starts[b + 1];
    if (tok < s0 || tok >= s1 || s0 < 0 || s1 > a.tokens) return;   // (a sequence out of the batch has no tokens)
    i = tok - s0;
    at = a.lens[b] - (s1 - s0) + i;
  } else {
    b = tok / a.per_seq;
    i = tok - b * a.per_seq;
    if (APPEND) at = a.lens[b] - a.per_seq + i;
  }
  const int trow = APPEND && a.starts ? tok : i;  // row along the token axis, and the batch index with it
  const int brow = APPEND && a.starts ? 0 : b;

  // first element of this token's head 0, per kind (wave-uniform)
  auto source = [&](const gr_rope_rows& k) { return static_cast<const T*>(k.src) + brow * k.sb + trow * k.st; };
  const T *sq = source(a.q), *sk = source(a.k), *sv = APPEND ? source(a.v) : nullptr;
  gr_rope8<T> x[ITER], y[ITER];
#pragma unroll
  for (int p = 0; p < ITER; ++p) {
    const int r = row0 + p * rpp;
    if (lane_live && r < rows) {
      const T* s = r < h0 ? sq + r * a.q.sh : !APPEND || r < h1 ? sk + (r - h0) * a.k.sh : sv + (r - h1) * a.v.sh;
      x[p].load(s + lo);
      y[p].load(s + hi);
    }
  }

  // where an append puts the token: its page and slot, or nowhere
  long long page = -1;
  int slot = 0;
  if (APPEND) {
    const int pi = at >> a.page_shift;
    if (at >= 0 && pi < a.width) {
      const int id = a.table[b * a.table_stride + pi];
      if (id >= 0 && id < a.pages) page = id;
    }
    slot = at & ((1 << a.page_shift) - 1);
  }

  float sn[8] = {}, cs[8] = {};
  if (a.pairs > 0) {
    int p1 = at, plane = 0;
    if (a.pos) {
      const int* pp = a.pos + brow * a.ps[1] + trow * a.ps[2];
      if (a.naxes == 1) p1 = pp[0];
      else if (lane < a.naxes) plane = pp[lane * a.ps[0]];
    }
    const int u0 = u < ru ? u : 0;
    unsigned long long ax = 0;
    if (a.naxes > 1) ax = *reinterpret_cast<const unsigned long long*>(a.axes + 8 * u0);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      int pe = p1;
      if (a.naxes > 1 && a.pos) pe = __shfl(plane, (int)(ax >> (8 * e)) & 63, 64);
      const unsigned long long t = (unsigned long long)(long long)pe * a.turns[8 * u0 + e];
      gr_turn_sincos((unsigned)(t >> 32), sn[e], cs[e]);
      if (inverse) sn[e] = -sn[e];
    }
  }

  auto target = [&](const gr_rope_rows& k, bool cached) {
    return static_cast<T*>(k.dst) + (cached ? page * k.db + slot * k.dt : brow * k.db + trow * k.dt);
  };
  T *dq = target(a.q, false), *dk = target(a.k, APPEND), *dv = APPEND ? target(a.v, true) : nullptr;
#pragma unroll
  for (int p = 0; p < ITER; ++p) {
    const int r = row0 + p * rpp;
    if (!lane_live || r >= rows) continue;
    if ((!APPEND || r < h1) && u < ru) {
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        if constexpr (INTER) {
          gr_rope8<T>& z = e < 4 ? x[p] : y[p];
          const int k = (2 * e) & 7;              // pairs e, e + 1: elements k .. k + 3
          const float a0 = z.get(k), b0 = z.get(k + 1), a1 = z.get(k + 2), b1 = z.get(k + 3);
          z.put2(k, fmaf(a0, cs[e], -b0 * sn[e]), fmaf(a0, sn[e], b0 * cs[e]));
          z.put2(k + 2, fmaf(a1, cs[e + 1], -b1 * sn[e + 1]), fmaf(a1, sn[e + 1], b1 * cs[e + 1]));
        } else {
          const float a0 = x[p].get(e), a1 = x[p].get(e + 1), b0 = y[p].get(e), b1 = y[p].get(e + 1);
          x[p].put2(e, fmaf(a0, cs[e], -b0 * sn[e]), fmaf(a1, cs[e + 1], -b1 * sn[e + 1]));
          y[p].put2(e, fmaf(a0, sn[e], b0 * cs[e]), fmaf(a1, sn[e + 1], b1 * cs[e + 1]));
        }
      }
    }
    if (APPEND && r >= h0 && page < 0) continue;
    T* d = r < h0 ? dq + r * a.q.dh : !APPEND || r < h1 ? dk + (r - h0) * a.k.dh : dv + (r - h1) * a.v.dh;
    x[p].template store<PAST>(d + lo);
    y[p].template store<PAST>(d + hi);
  }
}
