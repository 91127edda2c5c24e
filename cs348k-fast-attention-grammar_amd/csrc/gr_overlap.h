// gr_overlap.h -- host check of whether two strided arrays share an element.
// Kernels whose waves read and write rows in no order refuse outputs that
// overlap inputs. Apart, as arrays of their own are, costs two comparisons; slices
// of one buffer (heads of one projection) are decided exactly.
#pragma once
#include <cstdint>

namespace gr {

// Up to 4 dimensions, strides in elements (unit stride along the last included).
struct strided {
  const void* p;
  long long n[4], s[4];
};

// {batch, token or slot, head} strides of heads of `dim` elements.
inline strided heads_of(const void* p, long long b, long long t, long long h, int dim, const long long* st) {
  return {p, {b, t, h, dim}, {st[0], st[1], st[2], 1}};
}

// The same array by the same strides (those of single rows say nothing).
inline bool same_array(const strided& a, const strided& b) {
  bool same = a.p == b.p;
  for (int i = 0; i < 4; ++i) same &= a.n[i] == b.n[i] && (a.n[i] <= 1 || a.s[i] == b.s[i]);
  return same;
}

struct overlap_search {
  typedef __int128 i128;
  int terms = 0, steps = 0;
  long long s[8];                    // strides, largest first, and how often each may be taken
  i128 lo[8], hi[8], least[9], most[9];   // (least, most: what the terms from the k-th on reach)

  static i128 down(i128 a, i128 b) { return a / b - (a % b < 0 ? 1 : 0); }   // b > 0

  // Whether the terms from the k-th on reach r. True where the search gets long.
  bool reach(int k, i128 r) {
    if (r < least[k] || r > most[k]) return false;
    if (k == terms || ++steps > 20000) return true;
    i128 c = -down(most[k + 1] - r, s[k]), e = down(r - least[k + 1], s[k]);
    if (c < lo[k]) c = lo[k];
    if (e > hi[k]) e = hi[k];
    for (; c <= e; ++c)
      if (reach(k + 1, r - c * s[k])) return true;
    return false;
  }
};

// Whether arrays of `size`-byte elements share memory: a whole solution of sum i s_a -
// sum j s_b = (b - a) is searched for from the largest stride down, where nested
// strides leave one or two choices each.
inline bool overlap(const strided& a, const strided& b, int size) {
  typedef __int128 i128;
  const i128 pa = (i128)(uintptr_t)a.p, pb = (i128)(uintptr_t)b.p;
  i128 ea = 1, eb = 1;
  for (int i = 0; i < 4; ++i) {
    if (a.n[i] <= 0 || b.n[i] <= 0) return false;
    ea += (i128)(a.n[i] - 1) * a.s[i];
    eb += (i128)(b.n[i] - 1) * b.s[i];
  }
  if (pa + ea * size <= pb || pb + eb * size <= pa) return false;
  if ((pb - pa) % size) return true;
  overlap_search f;
  for (int side = 0; side < 2; ++side)
    for (int i = 0; i < 4; ++i) {
      const strided& x = side ? b : a;
      if (x.n[i] <= 1 || x.s[i] == 0) continue;
      int k = 0;
      while (k < f.terms && f.s[k] > x.s[i]) ++k;
      if (k == f.terms || f.s[k] != x.s[i]) {
        for (int m = f.terms++; m > k; --m) {
          f.s[m] = f.s[m - 1];
          f.lo[m] = f.lo[m - 1];
          f.hi[m] = f.hi[m - 1];
        }
        f.s[k] = x.s[i];
        f.lo[k] = f.hi[k] = 0;
      }
      if (side) f.lo[k] -= x.n[i] - 1;
      else f.hi[k] += x.n[i] - 1;
    }
  f.least[f.terms] = f.most[f.terms] = 0;
  for (int k = f.terms; k-- > 0;) {
    f.least[k] = f.least[k + 1] + f.lo[k] * f.s[k];
    f.most[k] = f.most[k + 1] + f.hi[k] * f.s[k];
  }
  return f.reach(0, (pb - pa) / size);
}

}  // namespace gr
