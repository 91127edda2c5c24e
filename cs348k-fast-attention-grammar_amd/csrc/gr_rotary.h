// gr_rotary.h -- rotation of query and key heads by position, alone or on the
// way into a paged key/value cache, behind a norm of each head or not, the cache's
// rows quantised or not.
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
// Rows that are normed (divided by their root mean square) or quantised are reduced, over
// lanes of a power of two and without LDS. What a token's angles and weights are made of is
// asked for before its rows, and every lane asks for as much, whatever it is for: the
// compiler then knows how many loads are behind the ones it waits for, and angles are
// computed while rows are on their way. (Rows asked for by the lanes that have one, angles'
// turns behind them: 9,668 tokens of 32 + 8 + 8 heads of 128, normed into a quantised
// cache, 53.7 us, now 47.5; without the norm 45.4 and 42.)
//
// Bound by memory once there are tokens enough: 2 x 4,096 tokens of 32 + 32 heads
// of 128 (268 MB, bf16) take 43-52 us, 5.2-6.2 TB/s, where a large copy reaches
// 5.15; 320 tokens of 4 + 4 heads of 64 take 4.0 us, a launch and two trips to
// memory. Normed: 2 x 4,096 tokens of 32 + 8 heads of 128 (168 MB) 28-31 us a launch in a row
// of them, 5.4-6.0 TB/s (34-36 alone, from its first wave to its last), in fp32 61-68; 288
// tokens of 8 + 4 heads of 64 4.0; normed into a quantised cache, the 9,668 tokens above
// (218 MB) 43-47.5, 4.6-5.1 TB/s, and into 16-bit pages (238 MB) 43-47: four waves a SIMD
// (115 registers) with vector work of their own between loads and stores; without the norm,
// six waves, 5.2.
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
  // NORM: weights of the queries' and keys' rows (nullptr: ones), in fp32 or the rows' type
  const void *wq, *wk;
  int w32;
  float eps;
  // Q8: the E8M0 scales of the cache's rows, unit stride along the slots
  unsigned char* scales;
  long long sp, sh, skind;       // page, head, from a key's to a value's
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

// A token's position, from `pos` (several axes: lane i has axis i's), or `at` on every
// axis. (a: gr_rope_args, or what has its members.)
template <class A>
__device__ __forceinline__ int gr_position(const A& a, const int* pos, int at, int lane) {
  if (!pos) return at;
  if (a.naxes == 1) return pos[0];
  return lane < a.naxes ? pos[lane * a.ps[0]] : 0;
}

// What the angles of the 8 pairs of a unit are made of, asked for before a token's rows are,
// so that they are computed while the rows are on their way (loads return in order).
struct gr_unit_turns {
  unsigned long long turns[8], axes;
  template <class A>
  __device__ __forceinline__ void load(const A& a, int u0) {
#pragma unroll
    for (int e = 0; e < 8; ++e) turns[e] = a.turns[8 * u0 + e];
    axes = 0;
    if (a.naxes > 1) axes = *reinterpret_cast<const unsigned long long*>(a.axes + 8 * u0);
  }
  // Sines and cosines at `position`; by_axis: lane i has axis i's.
  __device__ __forceinline__ void angles(int position, bool by_axis, bool inverse, float (&sn)[8], float (&cs)[8]) const {
    int pe[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) pe[e] = position;
    if (by_axis) {
#pragma unroll
      for (int e = 0; e < 8; ++e) pe[e] = __shfl(position, (int)(axes >> (8 * e)) & 63, 64);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const unsigned long long t = (unsigned long long)(long long)pe[e] * turns[e];
      gr_turn_sincos((unsigned)(t >> 32), sn[e], cs[e]);
      if (inverse) sn[e] = -sn[e];
    }
  }
};

// Sum, and largest as whole numbers, over the 1, 2, 4, 8 or 16 lanes of a group (a power of
// two, aligned), for all of them: within four lanes, then by mirrors of 8 and 16, whose
// halves are alike by then.
template <int CTRL>
__device__ __forceinline__ unsigned gr_dpp(unsigned v) {
  return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
__device__ __forceinline__ float gr_group_sum(float v, int lanes) {
  if (lanes > 1) v += __builtin_bit_cast(float, gr_dpp<0xb1>(__builtin_bit_cast(unsigned, v)));    // quad_perm 1 0 3 2
  if (lanes > 2) v += __builtin_bit_cast(float, gr_dpp<0x4e>(__builtin_bit_cast(unsigned, v)));    // quad_perm 2 3 0 1
  if (lanes > 4) v += __builtin_bit_cast(float, gr_dpp<0x141>(__builtin_bit_cast(unsigned, v)));   // row_half_mirror
  if (lanes > 8) v += __builtin_bit_cast(float, gr_dpp<0x140>(__builtin_bit_cast(unsigned, v)));   // row_mirror
  return v;
}
__device__ __forceinline__ unsigned gr_umax(unsigned a, unsigned b) { return a > b ? a : b; }
__device__ __forceinline__ unsigned gr_group_umax(unsigned v, int lanes) {
  if (lanes > 1) v = gr_umax(v, gr_dpp<0xb1>(v));
  if (lanes > 2) v = gr_umax(v, gr_dpp<0x4e>(v));
  if (lanes > 4) v = gr_umax(v, gr_dpp<0x141>(v));
  if (lanes > 8) v = gr_umax(v, gr_dpp<0x140>(v));
  return v;
}

// Lanes of a head row that is reduced: its units, up to a power of two.
__device__ __forceinline__ int gr_row_lanes(int units) { return units > 1 ? 1 << (32 - __builtin_clz(units - 1)) : 1; }

// 16 weights of a lane's unit, from elements lo and hi on: asked for, and as floats. (Loads
// whatever the weights are, from `any` where there are none: loads of one of two ways are
// waited for where the ways join.)
template <class T>
struct gr_unit_weights {
  gr_u32x4 r[4];
  __device__ __forceinline__ void load(const void* w, int w32, int lo, int hi, const void* any) {
    const bool wide = sizeof(T) == 4 || w32;
    const char* const p = static_cast<const char*>(w ? w : any);
    const int size = w ? (wide ? 4 : 2) : 0, next = w && wide ? 16 : 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = gr_ld16(p + (i < 2 ? lo : hi) * size + (i & 1) * next);
  }
  __device__ __forceinline__ void floats(const void* w, int w32, float (&f)[16]) const {
    if (w == nullptr) {
#pragma unroll
      for (int e = 0; e < 16; ++e) f[e] = 1.f;
    } else if (sizeof(T) == 4 || w32) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const unsigned u = r[e >> 2][e & 3];   // (a bit cast of the element itself reads element 0)
        f[e] = __builtin_bit_cast(float, u);
      }
    } else {
      gr_rope8<T> a, b;
      a.w[0] = r[0];
      b.w[0] = r[2];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        f[e] = a.get(e);
        f[8 + e] = b.get(e);
      }
    }
  }
};

// Rotates a unit's 8 pairs by its sines and cosines: elements e and 8 + e, or 2e and 2e + 1.
template <bool INTER>
__device__ __forceinline__ void gr_turn_unit(float (&f)[16], const float (&sn)[8], const float (&cs)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float &x = f[INTER ? 2 * e : e], &y = f[INTER ? 2 * e + 1 : 8 + e];
    const float a = x, b = y;
    x = fmaf(a, cs[e], -b * sn[e]);
    y = fmaf(a, sn[e], b * cs[e]);
  }
}

// Stores a unit of a key's (hr below their heads) or value's row as e4m3 numbers
// with the row's scale; the lanes of a row call it together.
template <class T>
__device__ __forceinline__ void gr_store_e4m3(const gr_rope_args& a, float (&f)[16], int hr, int lanes, int u, bool live, int lo,
                                              int hi, long long page, int slot) {
  unsigned top = 0;                              // the largest magnitude's bits
#pragma unroll
  for (int e = 0; e < 16; ++e) top = gr_umax(top, __builtin_bit_cast(unsigned, f[e]) & 0x7fffffffu);
  top = gr_group_umax(top, lanes);
  const bool finite = top < 0x7f800000u;
  // the largest number of four significant bits in T, 15 2^12 or 15 2^124
  constexpr float MOST = __is_same(T, _Float16) ? 61440.f : 0x1.ep+127f;
#pragma unroll
  for (int e = 0; e < 16; ++e) f[e] = __builtin_amdgcn_fmed3f(f[e], -MOST, MOST);
  top = top < __builtin_bit_cast(unsigned, MOST) ? top : __builtin_bit_cast(unsigned, MOST);
  // 1.m 2^e <= 1.75 2^8 2^k: k = e - 8, or one more where 1.m is above 1.75
  int sb = (int)(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
  sb = !finite ? 255 : sb < 0 ? 0 : sb;
  const float by = __builtin_bit_cast(float, (unsigned)(finite ? 254 - sb : 127) << 23);
  gr_u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int half = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i] * by, f[4 * i + 1] * by, 0, false);
    w[i] = finite ? (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i + 2] * by, f[4 * i + 3] * by, half, true) : 0x7f7f7f7fu;
  }
  if (!live || page < 0) return;
  const bool key = hr < a.k.heads;
  const gr_rope_rows& k = key ? a.k : a.v;
  const int h = key ? hr : hr - a.k.heads;
  unsigned char* const d = static_cast<unsigned char*>(k.dst) + page * k.db + slot * k.dt + h * k.dh;
  *reinterpret_cast<gr_u32x2*>(d + lo) = (gr_u32x2){w[0], w[1]};
  *reinterpret_cast<gr_u32x2*>(d + hi) = (gr_u32x2){w[2], w[3]};
  if (u == 0) a.scales[page * a.sp + h * a.sh + (key ? 0 : a.skind) + slot] = (unsigned char)sb;
}

// PAST: stores go past the caches (of whole 128-byte lines only). NORM: query and
// key rows are divided by their root mean square and multiplied by their
// weights, in fp32, before they are rotated. Q8: key and value rows are stored as
// e4m3 numbers z 2^-k, k the least power (-127 at least) by which the row's
// largest magnitude is at most 448, and k + 127 beside them. z 2^-k is exact, so the only rounding is
// the one to e4m3's four bits, and an attention gets the value back in bf16 or
// fp16 as it is (but for normed or turned keys below the type's normal range, which it
// rounds to the type's smallest steps): rows are clamped to the largest number of four bits
// in the type first, 61,440 in fp16 and 15 2^124 in bf16. A row with a value that is not finite is NaN all over.
template <class T, bool APPEND, bool INTER, int ITER, bool PAST, bool NORM = false, bool Q8 = false>
__device__ __forceinline__ void gr_rope_body(const gr_rope_args& a, bool inverse) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)((blockIdx.x * blockDim.x + threadIdx.x) >> 6));
  const int units = a.D >> 4;                    // of a head row
  const int lanes = NORM || Q8 ? gr_row_lanes(units) : units;
  const int rpp = 64 / lanes;                    // rows a pass
  const int h0 = a.q.heads, h1 = h0 + a.k.heads, rows = h1 + (APPEND ? a.v.heads : 0);
  const int passes = (rows + rpp - 1) / rpp, groups = (passes + ITER - 1) / ITER;
  const int tok = wave / groups;
  if (tok >= a.tokens) return;
  const int row0 = (wave - tok * groups) * ITER * rpp + lane / lanes, u = lane % lanes;
  const int ru = a.pairs >> 3;                   // rotated units
  const bool lane_live = lane < rpp * lanes && u < units;
  const int u0 = !(NORM || Q8) || u < units ? u : 0;   // (a lane without elements reads the first unit's)
  const int lo = u0 < ru ? (INTER ? 16 * u0 : 8 * u0) : 2 * a.pairs + 8 * (u0 - ru);
  const int hi = u0 < ru ? (INTER ? 16 * u0 + 8 : a.pairs + 8 * u0) : lo + 8 * (units - ru);

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
  const int* const pos = a.pos ? a.pos + brow * a.ps[1] + trow * a.ps[2] : nullptr;
  gr_unit_turns unit_turns = {};
  int position = 0;
  if ((NORM || Q8) && a.pairs > 0) {
    unit_turns.load(a, u0 < ru ? u0 : 0);
    // (a load either way: one of two ways to a register would wait where they join)
    position = *(pos ? pos + (a.naxes > 1 ? gr_imin(lane, a.naxes - 1) * a.ps[0] : 0) : a.lens);
  }
  gr_unit_weights<T> uq = {}, uk = {};
  if constexpr (NORM) {
    uq.load(a.wq, a.w32, lo, hi, h0 > 0 ? sq : sk);
    uk.load(a.wk, a.w32, lo, hi, h0 > 0 ? sq : sk);
  }
  gr_rope8<T> x[ITER], y[ITER];
  if constexpr (NORM || Q8) {
    // (in registers: a choice among arguments would become a load from a chosen address)
    long long qsh = a.q.sh, ksh = a.k.sh, vsh = APPEND ? a.v.sh : 0;
    asm("" : "+s"(qsh), "+s"(ksh), "+s"(vsh));
#pragma unroll
    for (int p = 0; p < ITER; ++p) {
      const int r = gr_imin(row0 + p * rpp, rows - 1);             // (rows past the end: the last again)
      const bool is_q = r < h0, is_k = !APPEND || r < h1;
      const T* s = (is_q ? sq : is_k ? sk : sv) + (r - (is_q ? 0 : is_k ? h0 : h1)) * (is_q ? qsh : is_k ? ksh : vsh);
      x[p].load(s + lo);
      y[p].load(s + hi);
    }
  } else {
#pragma unroll
    for (int p = 0; p < ITER; ++p) {
      const int r = row0 + p * rpp;
      if (lane_live && r < rows) {
        const T* s = r < h0 ? sq + r * a.q.sh : !APPEND || r < h1 ? sk + (r - h0) * a.k.sh : sv + (r - h1) * a.v.sh;
        x[p].load(s + lo);
        y[p].load(s + hi);
      }
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
  if ((NORM || Q8) && a.pairs > 0) {
    unit_turns.angles(pos ? position : at, pos && a.naxes > 1, inverse, sn, cs);
  } else if (a.pairs > 0) {
    unit_turns.load(a, u < ru ? u : 0);
    unit_turns.angles(gr_position(a, pos, at, lane), pos && a.naxes > 1, inverse, sn, cs);
  }

  auto target = [&](const gr_rope_rows& k, bool cached) {
    return static_cast<T*>(k.dst) + (cached ? page * k.db + slot * k.dt : brow * k.db + trow * k.dt);
  };
  T* dq = target(a.q, false);
  if constexpr (NORM || Q8) {
    const bool unit = u < units;
    const float inv_d = 1.0f / (float)a.D;
    float wq[16], wk[16];
    if constexpr (NORM) {
      uq.floats(a.wq, a.w32, wq);
      uk.floats(a.wk, a.w32, wk);
    }
#pragma unroll
    for (int p = 0; p < ITER; ++p) {
      const int r = row0 + p * rpp;
      float f[16];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        f[e] = x[p].get(e);
        f[8 + e] = y[p].get(e);
      }
      if (units != lanes) {                      // (lanes without elements add nothing to their row's sum)
#pragma unroll
        for (int e = 0; e < 16; ++e) f[e] = unit ? f[e] : 0.f;
      }
      if constexpr (NORM) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) ss = fmaf(f[e], f[e], ss);
        const float rms = rsqrtf(gr_group_sum(ss, lanes) * inv_d + a.eps);
        // rows of one kind in most passes: a scalar branch instead of a choice of each element
        const int first = (wave - tok * groups) * ITER * rpp + p * rpp;
        if (first + rpp <= h0) {
#pragma unroll
          for (int e = 0; e < 16; ++e) f[e] = f[e] * rms * wq[e];
        } else if (first >= h0 && first + rpp <= h1) {
#pragma unroll
          for (int e = 0; e < 16; ++e) f[e] = f[e] * rms * wk[e];
        } else if (!APPEND || first < h1) {
#pragma unroll
          for (int e = 0; e < 16; ++e) f[e] = APPEND && r >= h1 ? f[e] : f[e] * rms * (r < h0 ? wq[e] : wk[e]);
        }
      }
      if ((!APPEND || r < h1) && u < ru) gr_turn_unit<INTER>(f, sn, cs);
      if (Q8 && r >= h0) {
        gr_store_e4m3<T>(a, f, r - h0, lanes, u, lane_live && r < rows, lo, hi, page, slot);
      } else if (lane_live && r < rows && (!APPEND || r < h0 || page >= 0)) {
        gr_rope8<T> s, t;
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          s.put2(e, f[e], f[e + 1]);
          t.put2(e, f[8 + e], f[9 + e]);
        }
        T* d = dq + r * a.q.dh;
        if (r >= h0) {
          const gr_rope_rows& k = !APPEND || r < h1 ? a.k : a.v;
          d = target(k, APPEND) + (!APPEND || r < h1 ? r - h0 : r - h1) * k.dh;
        }
        s.template store<PAST>(d + lo);
        t.template store<PAST>(d + hi);
      }
    }
    return;
  }
  T *dk = target(a.k, APPEND), *dv = APPEND ? target(a.v, true) : nullptr;
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
