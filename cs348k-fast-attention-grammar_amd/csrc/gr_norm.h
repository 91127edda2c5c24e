// gr_norm.h -- the gradient of normed and rotated heads (their forward is gr_rope_body
// with NORM).
//
// y = R(t) n, n = w x r, r = 1 / sqrt(mean x^2 + eps). With g = R(-t) dy:
//   dw = sum over rows of g x r,   dx = r (g w - x r^2 mean(g w x)).
//
// Layout: as gr_rope_body, a wave takes ITER passes over a token's head rows; lane l
// has the same unit of 8 + 8 elements in every pass and token, so that it sums the
// weights' gradients of its elements over all its rows in registers. r is computed
// again from x, which the gradient reads in any case. At its end a
// workgroup adds its waves' sums and writes them beside the others'; a second launch adds
// those up, in the order of the workgroups.
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
  float* part;                   // [workgroup][2][D], or nullptr: no weights' gradients
};

constexpr int GR_NORM_WAVES = 4;

template <class T, bool INTER, int ITER>
__device__ __forceinline__ void gr_norm_bwd_body(const gr_norm_bwd_args& a, float* lds) {
  const int lane = threadIdx.x & 63;
  const int wave_in = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int units = a.D >> 4, lanes = gr_row_lanes(units), rpp = 64 / lanes;
  const int h0 = a.q.heads, rows = h0 + a.k.heads;
  const int passes = (rows + rpp - 1) / rpp, groups = (passes + ITER - 1) / ITER;
  const int u = lane & (lanes - 1), ru = a.pairs >> 3;
  const bool unit = u < units;
  const int u0 = unit ? u : 0;
  const int lo = u0 < ru ? (INTER ? 16 * u0 : 8 * u0) : 2 * a.pairs + 8 * (u0 - ru);
  const int hi = u0 < ru ? (INTER ? 16 * u0 + 8 : a.pairs + 8 * u0) : lo + 8 * (units - ru);
  float wq[16], wk[16], sq[16] = {}, sk[16] = {};
  gr_unit_weights<T>(a.wq, a.w32, lo, hi, wq);
  gr_unit_weights<T>(a.wk, a.w32, lo, hi, wk);
  const float inv_d = 1.0f / (float)a.D;

  const long long tasks = (long long)a.tokens * groups;
#pragma unroll 1
  for (long long task = (long long)blockIdx.x * GR_NORM_WAVES + wave_in; task < tasks; task += (long long)gridDim.x * GR_NORM_WAVES) {
    const int tok = (int)(task / groups), grp = (int)(task - (long long)tok * groups);
    const int row0 = grp * ITER * rpp + lane / lanes;
    const int b = tok / a.per_seq, i = tok - b * a.per_seq;
    auto source = [&](const gr_rope_rows& k) { return static_cast<const T*>(k.src) + b * k.sb + i * k.st; };
    const T *xq = source(a.q), *xk = source(a.k), *yq = source(a.gq), *yk = source(a.gk);
    gr_rope8<T> x[ITER], y[ITER], gx[ITER], gy[ITER];
#pragma unroll
    for (int p = 0; p < ITER; ++p) {
      const int r = row0 + p * rpp;
      x[p] = y[p] = gx[p] = gy[p] = {};
      if (unit && r < rows) {
        const T* s = r < h0 ? xq + r * a.q.sh : xk + (r - h0) * a.k.sh;
        const T* d = r < h0 ? yq + r * a.gq.sh : yk + (r - h0) * a.gk.sh;
        x[p].load(s + lo);
        y[p].load(s + hi);
        gx[p].load(d + lo);
        gy[p].load(d + hi);
      }
    }
    float sn[8] = {}, cs[8] = {};
    gr_unit_angles(a, a.pos + b * a.ps[1] + i * a.ps[2], 0, u0 < ru ? u0 : 0, lane, true, sn, cs);
    T *dq = static_cast<T*>(a.q.dst) + b * a.q.db + i * a.q.dt, *dk = static_cast<T*>(a.k.dst) + b * a.k.db + i * a.k.dt;
#pragma unroll
    for (int p = 0; p < ITER; ++p) {
      const int r = row0 + p * rpp;
      const bool query = r < h0, live = unit && r < rows;
      float f[16], g[16], ss = 0.f, dot = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        f[e] = x[p].get(e);
        f[8 + e] = y[p].get(e);
        g[e] = gx[p].get(e);
        g[8 + e] = gy[p].get(e);
      }
      if (u < ru) gr_turn_unit<INTER>(g, sn, cs);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        ss = fmaf(f[e], f[e], ss);
        dot = fmaf(g[e] * (query ? wq[e] : wk[e]), f[e], dot);
      }
      ss = gr_group_sum(ss, lanes);
      dot = gr_group_sum(dot, lanes);
      const float rms = rsqrtf(fmaf(ss, inv_d, a.eps));
      const float c = dot * inv_d * rms * rms;
      gr_rope8<T> s, t;
      float d[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float v = live ? g[e] * f[e] * rms : 0.f, vq = query ? v : 0.f;
        sq[e] += vq;
        sk[e] += v - vq;
        d[e] = rms * fmaf(-c, f[e], g[e] * (query ? wq[e] : wk[e]));
      }
      if (!live) continue;
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        s.put2(e, d[e], d[e + 1]);
        t.put2(e, d[8 + e], d[9 + e]);
      }
      T* to = query ? dq + r * a.q.dh : dk + (r - h0) * a.k.dh;
      s.template store<false>(to + lo);
      t.template store<false>(to + hi);
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
