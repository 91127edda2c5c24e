// gr_norm.h -- the gradient of normed and rotated heads (their forward is gr_rope_body
// with NORM).
//
// y = R(t) n, n = w x r, r = 1 / sqrt(mean x^2 + eps). With g = R(-t) dy:
//   dw = sum over rows of g x r,   dx = r (g w - x r^2 mean(g w x)).
//
// Layout: as gr_rope_body, a wave takes a token's head rows in passes (all of them, or
// `per` where tokens are few), and then those of other tokens; lane l has the same unit of 8 + 8
// elements in every pass and token, so that it sums the weights' gradients of
// its elements over all its rows in registers. r is computed again from x, which the
// gradient reads in any case. The rows and position of the next pass are on their way while
// one is worked on, the turns of a lane's pairs are kept, and passes of one kind of rows make
// no choice of weights or sums. At its end a workgroup adds its waves' sums and writes them
// beside the others'; a second launch adds those up, in the order of the workgroups.
//
// Bound by memory where tokens are many: 2 x 4,096 tokens of 32 + 8 heads of 128 (bf16, 252
// MB) 49 us, 5.1 TB/s, by two waves a SIMD (209 registers: sums, weights and two passes'
// rows) with 64 KB a CU on the way, and 4 for the second launch, a chain of trips to
// memory; in fp32 104 and 4. 300 tokens of 8 + 4 heads of 64 take 11.9 with it. Before every pass
// had as many loads, whose number is then known, the first took 62. From 4,096 tokens on a wave
// takes whole tokens, some waves one more than others: of 4,713 tokens of two passes three
// where the mean is 2.3, 20-21 us for 58 MB.
#pragma once
#include "gr_rotary.h"

struct gr_norm_bwd_args {
  gr_rope_rows q, k;             // x and dx
  gr_rope_rows gq, gk;           // dy (dst not used)
  int tokens, per_seq;
  int D, pairs, naxes;
  const unsigned long long* turns;
  const unsigned char* axes;
  const int* pos;
  long long ps[3];
  const void *wq, *wk;
  int w32;
  float eps;
  int per;                       // passes of a token that a wave takes
  float* part;                   // [workgroup][2][D], or nullptr: no weights' gradients
};

constexpr int GR_NORM_WAVES = 4;
template <int V> struct gr_const { static constexpr int value = V; };

template <class T, bool INTER>
__device__ __forceinline__ void gr_norm_bwd_body(const gr_norm_bwd_args& a, float* lds) {
  const int lane = threadIdx.x & 63;
  const int wave_in = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int units = a.D >> 4, lanes = gr_row_lanes(units), rpp = 64 / lanes;
  const int h0 = a.q.heads, rows = h0 + a.k.heads;
  const int passes = (rows + rpp - 1) / rpp, groups = (passes + a.per - 1) / a.per;
  const int u = lane & (lanes - 1), ru = a.pairs >> 3;
  const bool unit = u < units;
  const int u0 = unit ? u : 0;
  const int lo = u0 < ru ? (INTER ? 16 * u0 : 8 * u0) : 2 * a.pairs + 8 * (u0 - ru);
  const int hi = u0 < ru ? (INTER ? 16 * u0 + 8 : a.pairs + 8 * u0) : lo + 8 * (units - ru);
  float wq[16], wk[16], sq[16] = {}, sk[16] = {};
  gr_unit_weights<T> uq, uk;
  uq.load(a.wq, a.w32, lo, hi, a.q.src);
  uk.load(a.wk, a.w32, lo, hi, a.q.src);
  uq.floats(a.wq, a.w32, wq);
  uk.floats(a.wk, a.w32, wk);
  const float inv_d = 1.0f / (float)a.D;

  // A task is `per` passes of a token, the part-th of it; a wave's next one is `step` tasks on.
  const unsigned step = gridDim.x * GR_NORM_WAVES, step_tok = step / (unsigned)groups, step_part = step % (unsigned)groups;
  const int sub = lane / lanes;
  const bool all_units = units == lanes;
  struct pass_rows {
    unsigned tok;
    int part, pass, b, i;          // part and pass of the token's; batch and token
    int position;
    gr_rope8<T> x, y, gx, gy;
  };
  gr_unit_turns turns;
  turns.load(a, u0 < ru ? u0 : 0);
  // (in registers: a choice among arguments would become a load from a chosen address)
  long long qsh = a.q.sh, ksh = a.k.sh, gqsh = a.gq.sh, gksh = a.gk.sh;
  asm("" : "+s"(qsh), "+s"(ksh), "+s"(gqsh), "+s"(gksh));
  const long long paxis = (a.naxes > 1 ? gr_imin(lane, a.naxes - 1) : 0) * a.ps[0];
  // Rows past the token's last and lanes without elements read others': that every pass
  // has as many loads lets the next one's stay in flight while one is worked on.
  auto load = [&](pass_rows& d, unsigned tok, int part, int pass) {
    const int r = gr_imin(pass * rpp + sub, rows - 1);
    d.tok = tok;
    d.part = part;
    d.pass = pass;
    d.b = (int)tok / a.per_seq;
    d.i = (int)tok - d.b * a.per_seq;
    d.position = a.pos[d.b * a.ps[1] + d.i * a.ps[2] + paxis];
    auto source = [&](const gr_rope_rows& k) { return static_cast<const T*>(k.src) + d.b * k.sb + d.i * k.st; };
    const bool query = r < h0;
    const int h = r - (query ? 0 : h0);
    const T* const s = (query ? source(a.q) : source(a.k)) + h * (query ? qsh : ksh);
    const T* const g = (query ? source(a.gq) : source(a.gk)) + h * (query ? gqsh : gksh);
    d.x.load(s + lo);
    d.y.load(s + hi);
    d.gx.load(g + lo);
    d.gy.load(g + hi);
  };
  // Asks for the pass behind d's: of its task, or the first of the wave's next one; d's again
  // and false behind the last.
  auto load_next = [&](pass_rows& to, const pass_rows& d) {
    unsigned tok = d.tok;
    int part = d.part, pass = d.pass + 1;
    if (pass >= passes || pass >= (part + 1) * a.per) {
      tok += step_tok;
      part += (int)step_part;
      if (part >= groups) {
        part -= groups;
        ++tok;
      }
      pass = part * a.per;
    }
    const bool more = tok < (unsigned)a.tokens;
    load(to, more ? tok : d.tok, more ? part : d.part, more ? pass : d.pass);
    return more;
  };
  float sn[8] = {}, cs[8] = {};
  // KIND 0: rows of queries, 1: of keys, all live; 2: any.
  auto work = [&](const pass_rows& in, auto kind_tag) {
    constexpr int KIND = decltype(kind_tag)::value;
    const int r = in.pass * rpp + sub;
    const bool query = KIND == 2 ? r < h0 : KIND == 0, live = KIND < 2 || (unit && r < rows);
    auto weight = [&](int e) { return query ? wq[e] : wk[e]; };
    float f[16], g[16], ss = 0.f, dot = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      f[e] = in.x.get(e);
      f[8 + e] = in.y.get(e);
      g[e] = in.gx.get(e);
      g[8 + e] = in.gy.get(e);
    }
    if (KIND == 2 && !all_units) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        f[e] = unit ? f[e] : 0.f;
        g[e] = unit ? g[e] : 0.f;
      }
    }
    if (u < ru) gr_turn_unit<INTER>(g, sn, cs);
    float h[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      h[e] = g[e] * weight(e);
      ss = fmaf(f[e], f[e], ss);
      dot = fmaf(h[e], f[e], dot);
    }
    ss = gr_group_sum(ss, lanes);
    dot = gr_group_sum(dot, lanes);
    const float rms = rsqrtf(fmaf(ss, inv_d, a.eps));
    const float c = dot * inv_d * rms * rms;
    gr_rope8<T> s, t;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      if constexpr (KIND == 0) {
        sq[e] = fmaf(g[e] * rms, f[e], sq[e]);
      } else if constexpr (KIND == 1) {
        sk[e] = fmaf(g[e] * rms, f[e], sk[e]);
      } else {
        const float v = live ? g[e] * rms * f[e] : 0.f;   // (no differences: a NaN stays in its own sum)
        sq[e] += query ? v : 0.f;
        sk[e] += query ? 0.f : v;
      }
      h[e] = rms * fmaf(-c, f[e], h[e]);
    }
    if (!live) return;
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      s.put2(e, h[e], h[e + 1]);
      t.put2(e, h[8 + e], h[9 + e]);
    }
    const gr_rope_rows& to = query ? a.q : a.k;
    T* const d = static_cast<T*>(to.dst) + in.b * to.db + in.i * to.dt + (query ? r : r - h0) * to.dh;
    s.template store<false>(d + lo);
    t.template store<false>(d + hi);
  };
  auto pass = [&](const pass_rows& in) {
    if (in.pass == in.part * a.per)
      turns.angles(in.position, a.naxes > 1, true, sn, cs);
    const int r0 = in.pass * rpp;
    if (all_units && r0 + rpp <= h0) work(in, gr_const<0>{});
    else if (all_units && r0 >= h0 && r0 + rpp <= rows) work(in, gr_const<1>{});
    else work(in, gr_const<2>{});
  };
  pass_rows one, two;
  const unsigned task = blockIdx.x * GR_NORM_WAVES + (unsigned)wave_in;
  if (task / (unsigned)groups < (unsigned)a.tokens) {
    load(one, task / (unsigned)groups, (int)(task % (unsigned)groups), (int)(task % (unsigned)groups) * a.per);
#pragma unroll 1
    while (true) {
      bool more = load_next(two, one);
      pass(one);
      if (!more) break;
      more = load_next(one, two);
      pass(two);
      if (!more) break;
    }
  }
  if (a.part == nullptr) return;
  // the sums of the wave's rows, then of the workgroup's waves
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    for (int off = lanes; off < 64; off <<= 1) {
      sq[e] += __shfl_xor(sq[e], off, 64);
      sk[e] += __shfl_xor(sk[e], off, 64);
    }
  }
  float* const mine = lds + wave_in * 2 * a.D;
  if (lane < lanes && unit) {
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int at = e < 8 ? lo + e : hi + e - 8;
      mine[at] = sq[e];
      mine[a.D + at] = sk[e];
    }
  }
  __syncthreads();
  for (int at = threadIdx.x; at < 2 * a.D; at += 64 * GR_NORM_WAVES) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < GR_NORM_WAVES; ++w) s += lds[w * 2 * a.D + at];
    a.part[(long long)blockIdx.x * 2 * a.D + at] = s;
  }
}

// Column sums of part [n][2 D] for one weight vector: 16 columns a workgroup, 64 rows side by
// side, 8 of each asked for at once.
template <class W>
__device__ __forceinline__ void gr_norm_dw_body(const float* part, int n, int D, W* dwq, W* dwk) {
  __shared__ float sum[64][17];
  const int col = threadIdx.x & 15, r0 = threadIdx.x >> 4;
  const int at = (int)blockIdx.x * 16 + col;      // of the 2 D
  float s = 0.f;
  for (int r = r0; r < n; r += 64 * 8) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = r + 64 * i < n ? part[(long long)(r + 64 * i) * 2 * D + at] : 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += v[i];
  }
  sum[r0][col] = s;
  __syncthreads();
  for (int half = 32; half > 0; half >>= 1) {
    if (r0 < half) sum[r0][col] += sum[r0 + half][col];
    __syncthreads();
  }
  if (r0 == 0) {
    W* const to = at < D ? dwq : dwk;
    if (to) to[at < D ? at : at - D] = (W)sum[0][col];
  }
}
