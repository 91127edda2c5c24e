// gr_paged_rows.h -- attention of few rows over a quantised paged cache: a decode step's
// tiles of 16 rows (the query heads of a key head), and of 32 (gfx950, head dims 64
// and 128).
//
// Such calls read every key for a handful of rows, so the kernel is to keep up with memory:
// at 5.5 TB/s a SIMD has 3,700 cycles for 32 keys of 128 e4m3 numbers, key and value.
//
//  * A wave has its tiles of BN keys to itself; the KG waves of a workgroup take every
//    KG-th tile and merge through LDS at the end.
//  * S^T = K Q^T on 16 x 16 x 32 MFMAs, a 16-key block at a time: lane (key, g) loads 16-byte
//    pieces g of its key's row straight from the page, turns them into T under
//    its key's scale, and has an operand: which dims a lane group holds is the same
//    for Q, so no order of dims is needed, and keys do not pass through LDS.
//  * O^T = V^T P^T: values are turned into T, rows under their scales, and written to LDS,
//    from where transposing reads fetch 4 keys of a dim for each lane; the scores of 2
//    blocks are already in the order of those keys.
//  * Loads are a tile ahead: a tile's bytes are in registers, whose place the next
//    tile's take as soon as they are converted.
//
// Measured (bf16, 32 / 8 heads of 128). A token each of 64 sequences of 200 to 11,000 keys
// (672 MB) takes 122 us in tiles of 16 rows, 5.5 TB/s, and 4.7 for the merge: bound by memory
// (matrix cores 8 % busy, vector units 26 %). With keys through LDS like values, in tiles of
// 32 rows, 167 in all. Four tokens of 40 / 8 heads each of 12 sequences of 900 to 9,000 keys (111 MB,
// tiles of 32 rows) 28 and 4.2: eight key steps a wave, the first tile's way and the merge
// inside the workgroup. 613 keys of one token (16 heads of 64) 6.1, a launch and a chain of
// trips: length, page id, rows, two or three key steps of eight waves and their merge.
//
// What a row may see, pages that do not exist, values that are not finite, bases
// and sums: as in gr_paged.h, whose tiles and shares this uses.
#pragma once
#include "gr_paged.h"

template <int D, int BN, int RB, int KG>
struct gr_rows_lds {
  static constexpr int SLOT = BN * D * 2;                     // a wave's values
  static constexpr int PART = RB * (D / 16) * 1024 + RB * 512;   // a wave's O, base and sum
  static constexpr int MERGE = (KG - 1) * PART;
  static constexpr int BYTES = KG * SLOT > MERGE ? KG * SLOT : MERGE;
};

// One tile of 16 RB rows over keys [key0, key1), by KG of the workgroup's WAVES;
// place: where its partial result goes, in rows of BM, or -1 for a tile that is done here.
template <class T, int D, int BN, int RB, int KG, int WAVES, int BM>
__device__ __forceinline__ void gr_paged_rows(const gr_paged_args& a, char* lds_all, const gr_paged_tile& t, int hk, int key0,
                                              int key1, int place) {
  typedef gr_mfma<T> MF;
  typedef typename MF::vec8 vec8;
  typedef typename MF::vec2 vec2;
  typedef gr_rows_lds<D, BN, RB, KG> L;
  constexpr bool HALF = gr_is_same<T, _Float16>::value;
  constexpr int KB = BN / 16, DB = D / 16, DS = D / 32;
  constexpr int KL = D / 64;                 // 16-byte pieces of a key's row a lane has
  constexpr int CPR = D / 8, CPR8 = D / 16;  // 16-byte chunks of a row of T, of a cached row
  constexpr int VI = CPR8 / 4;               // load instructions of a block of 16 values
  constexpr int WIN = 64 / KB;

  const int lane = threadIdx.x & 63;
  const int kg = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  if (KG < WAVES && kg >= KG) {              // a wave without a part: the merge's barriers only
    if constexpr (KG > 1) {
      __syncthreads();
      __syncthreads();
    }
    return;
  }
  const int g = lane >> 4, l16 = lane & 15;
  char* const vt = lds_all + kg * L::SLOT;

  // this lane's rows, one of each 16, and the last key that each sees
  const int base_pos = t.len - t.n;
  int token[RB], head[RB], limit[RB];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const int row = gr_imin(t.row0 + 16 * rb + l16, t.nrows - 1);   // rows past the end: copies of the last
    token[rb] = row / a.G;
    head[rb] = hk * a.G + row % a.G;
    limit[rb] = a.causal ? gr_imin(base_pos + token[rb], t.keys - 1) : t.keys - 1;
  }
  const int lim_lo = a.causal ? gr_imin(base_pos + t.row0 / a.G, t.keys - 1) : t.keys - 1;
  const float c = a.scale_log2, shift = gr_paged_shift<T>(t.keys);

  // offsets: a key's row in the cache; values' rows there and in LDS; transposing reads
  const unsigned koff = (unsigned)(l16 * a.k_ss) + g * 16;
  auto vrow = [&](int i) { return gr_value8<D>(lane) + i * (64 / CPR8); };
  unsigned voff[VI];
  int vdst[VI];
#pragma unroll
  for (int i = 0; i < VI; ++i) {
    const int r = vrow(i), c8 = gr_piece8<D>(lane);
    voff[i] = (unsigned)(r * a.v_ss) + c8 * 16;
    vdst[i] = r * (D * 2) + gr_swz_v8<CPR>(r, 2 * c8) * 16;
  }
  const int trow = 4 * g + ((lane >> 2) & 3), tcol = 4 * (lane & 3);
  const int tbase = trow * (D * 2) + gr_swz_v8<CPR>(trow, tcol >> 3) * 16 + (tcol & 7) * 2;
  const int smask = (1 << a.page_shift) - 1;
  const int* const tab = a.table + t.b * a.table_stride;
  const unsigned char* const kp = static_cast<const unsigned char*>(a.k) + hk * a.k_sh;
  const unsigned char* const vp = static_cast<const unsigned char*>(a.v) + hk * a.v_sh;

  const int ntile_all = key1 > key0 ? (key1 - key0 + BN - 1) / BN : 0;
  const int ntile = (ntile_all - kg + KG - 1) / KG;           // of this wave
  auto key_of = [&](int j) { return key0 + (j * KG + kg) * BN; };
  // lane l: where block l % KB of tile j0 + l / KB is, refilled every WIN tiles
  unsigned long long kwin = 0, vwin = 0, swin = 0, badwin = 0;
  auto id_of = [&](int j0) {
    const long long key = key0 + ((long long)(j0 + lane / KB) * KG + kg) * BN + 16 * (lane % KB);
    return tab[key >> a.page_shift < a.width ? (int)(key >> a.page_shift) : a.width - 1];
  };
  auto refill = [&](int j0, int id) {
    const int key = key0 + ((j0 + lane / KB) * KG + kg) * BN + 16 * (lane % KB), slot = key & smask;
    const bool ok = (unsigned)id < (unsigned)a.pages;
    kwin = (unsigned long long)(kp + (ok ? id : 0) * a.k_sp + slot * a.k_ss);
    vwin = (unsigned long long)(vp + (ok ? id : 0) * a.v_sp + slot * a.v_ss);
    swin = (unsigned long long)(a.scales + (ok ? id : 0) * a.s_sp + hk * a.s_sh + slot);
    badwin = __builtin_amdgcn_ballot_w64(!ok && key < key1);
  };
  auto lane64 = [&](unsigned long long w, int l) {
    return (unsigned long long)(unsigned)__builtin_amdgcn_readlane((int)(w >> 32), l) << 32
           | (unsigned)__builtin_amdgcn_readlane((int)(unsigned)w, l);
  };

  typedef const __attribute__((address_space(1))) gr_u32x4 global_u32x4;
  typedef const __attribute__((address_space(1))) unsigned global_u32;
  gr_u32x4 kr[KB][KL], vr[KB][VI];
  unsigned ksb[KB], vsb[KB][VI];               // words of four scales, the row's among them
  const int kshift = 8 * (l16 & 3);
  auto vshift = [&](int i) { return 8 * (vrow(i) & 3); };
  // Asks for tile j's keys and values; rows that are not there are zeros.
  auto load_k = [&](int j, auto whole_tag, unsigned bad) {
    constexpr bool WHOLE = decltype(whole_tag)::value;
    const int at = (j & (WIN - 1)) * KB;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const unsigned long long k0 = lane64(kwin, at + kb), s0 = lane64(swin, at + kb);
      if (!WHOLE) {
        ksb[kb] = 0;
#pragma unroll
        for (int i = 0; i < KL; ++i) kr[kb][i] = (gr_u32x4){0, 0, 0, 0};
      }
      if (WHOLE || (!(bad >> kb & 1) && l16 < key1 - key_of(j) - 16 * kb)) {
#pragma unroll
        for (int i = 0; i < KL; ++i) kr[kb][i] = *(global_u32x4*)(k0 + koff + 64 * i);
        ksb[kb] = *(global_u32*)(s0 + (unsigned)(l16 & ~3));
      }
    }
  };
  auto load_v = [&](int j, auto whole_tag, unsigned bad) {
    constexpr bool WHOLE = decltype(whole_tag)::value;
    const int at = (j & (WIN - 1)) * KB;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const unsigned long long v0 = lane64(vwin, at + kb), s0 = lane64(swin, at + kb);
#pragma unroll
      for (int i = 0; i < VI; ++i) {
        const int r = vrow(i);
        if (!WHOLE) {
          vsb[kb][i] = 0;
          vr[kb][i] = (gr_u32x4){0, 0, 0, 0};
        }
        if (WHOLE || (!(bad >> kb & 1) && r < key1 - key_of(j) - 16 * kb)) {
          vr[kb][i] = *(global_u32x4*)(v0 + voff[i]);
          vsb[kb][i] = *(global_u32*)(s0 + a.s_kind + (unsigned)(r & ~3));
        }
      }
    }
  };

  vec8 qf[RB][DS];
  gr_f32x4 o[RB][DB];
  float m[RB], l[RB], base[RB];              // a row's base, its sum, shift - m c (no base yet: shift)
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
#pragma unroll
    for (int db = 0; db < DB; ++db) o[rb][db] = (gr_f32x4)(0.f);
    m[rb] = -GR_INF;
    l[rb] = 0.f;
    base[rb] = shift;
  }

  // Tiles are asked for in order, keys and then values; those up to `plain` are
  // whole, in the window, and their pages exist.
  constexpr unsigned BLOCKS = (1u << KB) - 1;
  int asked = 0, plain = 0, nwhole = 0;
  unsigned bad = 0;                           // bad blocks of the tile asked for last
  auto ask_k = [&]() {
    if (asked >= ntile) return;
    if (asked > 0 && (asked & (WIN - 1)) == 0) refill(asked, id_of(asked));
    bad = (unsigned)(badwin >> ((asked & (WIN - 1)) * KB)) & BLOCKS;
    load_k(asked, gr_ic<0>{}, bad);
    plain = badwin == 0 ? gr_imin(nwhole, (asked & ~(WIN - 1)) + WIN) : 0;
  };
  auto ask_v = [&]() {
    if (asked < ntile) load_v(asked++, gr_ic<0>{}, bad);
  };

  // One tile, and the loads of the next one as its registers become free. MASKED: any
  // tile, else one that every row sees in full. PLAIN: the next one is.
  auto tile = [&](int j, auto masked_tag, auto plain_tag) {
    constexpr bool MASKED = decltype(masked_tag)::value, PLAIN = decltype(plain_tag)::value;
    const int k0 = key_of(j);
    const unsigned mine = bad;
    gr_f32x4 s[RB][KB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) s[rb][kb] = (gr_f32x4)(0.f);
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      // (taken here: what is made of a loaded word alone would go up to the load, in the
      // tile before, and its wait with it)
      asm volatile("" : "+v"(ksb[kb]));
      const float f = gr_e8m0_of(ksb[kb], kshift);
#pragma unroll
      for (int ds = 0; ds < DS; ++ds) {
        const gr_u32x4 r = kr[kb][ds >> 1];
        const int h = 2 * (ds & 1);
        const vec8 kf = gr_as<vec8>((gr_u32x4){gr_from_e4m3<T, false>(r[h], f), gr_from_e4m3<T, true>(r[h], f),
                                               gr_from_e4m3<T, false>(r[h + 1], f), gr_from_e4m3<T, true>(r[h + 1], f)});
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) s[rb][kb] = MF::mma16(kf, qf[rb][ds], s[rb][kb]);
      }
    }
    if constexpr (!PLAIN) ask_k();
    else load_k(asked, gr_ic<1>{}, 0u);
    // values to LDS (the slot's last reads came before in this wave's order)
    unsigned long long odd = 0;               // MASKED: keys with a value that is not finite
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int i = 0; i < VI; ++i) {
        asm volatile("" : "+v"(vsb[kb][i]));
        const float f = gr_e8m0_of(vsb[kb][i], vshift(i));
        gr_u32x4 w[2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
          w[h] = (gr_u32x4){gr_from_e4m3<T, false>(vr[kb][i][2 * h], f), gr_from_e4m3<T, true>(vr[kb][i][2 * h], f),
                            gr_from_e4m3<T, false>(vr[kb][i][2 * h + 1], f), gr_from_e4m3<T, true>(vr[kb][i][2 * h + 1], f)};
        if constexpr (MASKED) {
          constexpr unsigned EXP = HALF ? 0x7c007c00u : 0x7f807f80u, ONE = HALF ? 0x04000400u : 0x00800080u;
          gr_u32x4 x = ((w[0] & EXP) + ONE) | ((w[1] & EXP) + ONE);
          const bool mine = ((x[0] | x[1] | x[2] | x[3]) & 0x80008000u) != 0;
          if (__builtin_expect(gr_any(mine), 0)) {
            bool row_odd = false;
#pragma unroll 1
            for (int r = 0; r < 16; ++r)      // (rows of this instruction: some of the 16)
              if (gr_any(mine && vrow(i) == r)) {
                odd |= 1ull << (16 * kb + r);
                row_odd |= vrow(i) == r;
              }
            if (row_odd) w[0] = w[1] = (gr_u32x4){0, 0, 0, 0};   // taken out of the product
          }
        }
        gr_st16(vt + kb * (16 * D * 2) + vdst[i], w[0]);
        gr_st16(vt + kb * (16 * D * 2) + (vdst[i] ^ 16), w[1]);
      }
    if constexpr (!PLAIN) ask_v();
    else load_v(asked++, gr_ic<1>{}, 0u);
    vec8 pt[RB][KB / 2];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      bool fresh = m[rb] == -GR_INF;          // no base yet, and a key to take it from
      if constexpr (MASKED) {
        // element r of block kb is key k0 + 16 kb + 4 g + r
        const int delta = limit[rb] - k0 - 4 * g;
        bool sees = false;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          const int d = (mine >> kb) & 1 ? -1 : delta - 16 * kb;
          sees |= d >= 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) s[rb][kb][e] = e <= d ? s[rb][kb][e] : -GR_INF;
        }
        fresh &= sees;
      }
      float lt;
      auto make_p = [&]() {
        const float nmc = HALF ? base[rb] : m[rb] == -GR_INF ? 0.f : -m[rb] * c;
        lt = 0.f;
#pragma unroll
        for (int x = 0; x < KB / 2; ++x) {
          gr_u32x4 pw;
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            const float p0 = gr_exp2(fmaf(s[rb][2 * x + (e >> 2)][e & 3], c, nmc));
            const float p1 = gr_exp2(fmaf(s[rb][2 * x + (e >> 2)][(e & 3) + 1], c, nmc));
            const vec2 pp = __builtin_convertvector((gr_f32x2){p0, p1}, vec2);
            lt = MF::sum2(pp, lt);
            pw[e >> 1] = __builtin_bit_cast(unsigned, pp);
          }
          pt[rb][x] = gr_as<vec8>(pw);
        }
      };
      make_p();
      if (gr_any(fresh || !(lt <= GR_FLASH_SUM_MAX))) {
        float mt = -GR_INF;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int e = 0; e < 4; ++e) mt = fmaxf(mt, s[rb][kb][e]);
        mt = fmaxf(mt, __shfl_xor(mt, 16, 64));
        mt = fmaxf(mt, gr_xor32(mt));
        const float mn = fmaxf(m[rb], mt);
        const float alpha = mn > m[rb] ? gr_exp2((m[rb] - mn) * c) : 1.f;   // m = -inf -> 0
        l[rb] *= alpha;
#pragma unroll
        for (int db = 0; db < DB; ++db) o[rb][db] *= alpha;
        m[rb] = mn;
        if (HALF) base[rb] = mn == -GR_INF ? shift : fmaf(-mn, c, shift);
        make_p();
      }
      l[rb] += lt;
    }
#pragma unroll
    for (int x = 0; x < KB / 2; ++x)
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        typedef short v4s __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) v4s lds_v4s;
        gr_u32x4 r;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const char* p = vt + (tbase ^ (db * 32)) + (2 * x + h) * (16 * D * 2);
          const v4s v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(__attribute__((address_space(3))) char*)(char*)p);
          const gr_u32x2 w = __builtin_bit_cast(gr_u32x2, v);
          r[2 * h] = w[0];
          r[2 * h + 1] = w[1];
        }
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) o[rb][db] = MF::mma16(gr_as<vec8>(r), pt[rb][x], o[rb][db]);
      }
    if constexpr (MASKED) {
      // keys taken out, from memory to the rows that see them
#pragma unroll 1
      for (; __builtin_expect(odd != 0, 0); odd &= odd - 1) {
        const int key = __builtin_ctzll(odd), kb = key >> 4;
        const int id = tab[(k0 + key) >> a.page_shift];       // (in the table: the key was loaded)
        const int slot = (k0 + key) & smask;
        const unsigned char* const row = vp + id * a.v_sp + slot * a.v_ss + 4 * g;
        const float f = gr_e8m0(a.scales[id * a.s_sp + hk * a.s_sh + a.s_kind + slot]);
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
          // the key's weight: element 4 (kb % 2) + key % 4 of block pair kb / 2, in lane group (key / 4) % 4
          unsigned w = 0;
#pragma unroll
          for (int x = 0; x < KB / 2; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (x == kb >> 1 && e == 2 * (kb & 1) + ((key >> 1) & 1)) w = gr_raw(pt[rb][x])[e];
          const unsigned short hw = (unsigned short)((key & 1) ? w >> 16 : w & 0xffffu);
          const float pv = __shfl((float)__builtin_bit_cast(T, hw), l16 + 16 * ((key >> 2) & 3), 64);
          const bool vis = k0 + key <= limit[rb];
#pragma unroll
          for (int db = 0; db < DB; ++db) {
            const unsigned b4 = *reinterpret_cast<const unsigned*>(row + 16 * db);
            const unsigned v01 = gr_from_e4m3<T, false>(b4, f), v23 = gr_from_e4m3<T, true>(b4, f);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const unsigned v = e < 2 ? v01 : v23;
              const float x = (float)__builtin_bit_cast(T, (unsigned short)((e & 1) ? v >> 16 : v & 0xffffu));
              if (vis) o[rb][db][e] = fmaf(pv, x, o[rb][db][e]);
            }
          }
        }
      }
    }
  };

  // page ids first, then this lane's Q rows in the order of the keys' dims
  const int first_id = ntile > 0 ? id_of(0) : 0;
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const T* qp = static_cast<const T*>(a.q) + t.b * a.q_sb + (long long)(t.first + token[rb]) * a.q_st + head[rb] * a.q_sh;
#pragma unroll
    for (int ds = 0; ds < DS; ++ds) qf[rb][ds] = gr_as<vec8>(gr_ld16(qp + 64 * (ds >> 1) + 16 * g + 8 * (ds & 1)));
  }
  // leading tiles of the wave that end before key `end`.
  auto tiles_before = [&](int end) { return end - key0 < (kg + 1) * BN ? 0 : ((end - key0) / BN - kg + KG - 1) / KG; };
  nwhole = gr_imin(ntile, tiles_before(key1));
  if (ntile > 0) refill(0, first_id);
  ask_k();
  ask_v();
  const int nclean = gr_imin(nwhole, tiles_before(lim_lo + 1));
  int j = 0;
#pragma unroll 1
  while (j < nclean && bad == 0) {
#pragma unroll 1
    for (; j < nclean && asked < plain && bad == 0; ++j) tile(j, gr_ic<0>{}, gr_ic<1>{});
    if (j < nclean && bad == 0) tile(j++, gr_ic<0>{}, gr_ic<0>{});
  }
#pragma unroll 1
  for (; j < ntile; ++j) tile(j, gr_ic<1>{}, gr_ic<0>{});

  if constexpr (KG > 1) {
    // the waves' partials through LDS: O as RB DB quads of floats per lane, then
    // base and row sum
    __syncthreads();
    auto at = [&](int grp) { return lds_all + (grp - 1) * L::PART + lane * 16; };
    auto ml_at = [&](int grp, int rb) { return lds_all + (grp - 1) * L::PART + RB * DB * 1024 + rb * 512 + lane * 8; };
    if (kg > 0) {
      char* const w = at(kg);
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
#pragma unroll
        for (int db = 0; db < DB; ++db) *reinterpret_cast<gr_f32x4*>(w + (rb * DB + db) * 1024) = o[rb][db];
        *reinterpret_cast<gr_f32x2*>(ml_at(kg, rb)) = (gr_f32x2){m[rb], l[rb]};
      }
    }
    __syncthreads();
    if (kg > 0) return;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      gr_f32x2 ml[KG];
      float mx = m[rb];
#pragma unroll
      for (int k = 1; k < KG; ++k) {
        ml[k] = *reinterpret_cast<const gr_f32x2*>(ml_at(k, rb));
        mx = fmaxf(mx, ml[k][0]);
      }
      const float to = mx == -GR_INF ? 0.f : mx;
      const float w0 = gr_exp2((m[rb] - to) * c);
      l[rb] *= w0;
#pragma unroll
      for (int db = 0; db < DB; ++db) o[rb][db] *= w0;
      m[rb] = mx;
#pragma unroll
      for (int k = 1; k < KG; ++k) {
        const float wk = gr_exp2((ml[k][0] - to) * c);
        l[rb] = fmaf(wk, ml[k][1], l[rb]);
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          const gr_f32x4 v = *reinterpret_cast<const gr_f32x4*>(at(k) + (rb * DB + db) * 1024);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[rb][db][e] = fmaf(wk, v[e], o[rb][db][e]);
        }
      }
    }
  }

#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    float lt = l[rb] + __shfl_xor(l[rb], 16, 64);
    lt += gr_xor32(lt);
    if (t.row0 + 16 * rb + l16 >= t.nrows) continue;
    if (place >= 0) {
      // unnormalised O and (base, row sum) of these keys
      const long long at = (long long)place * BM + 16 * rb + l16;
      float* const po = a.part_o + at * D;
#pragma unroll
      for (int db = 0; db < DB; ++db) *reinterpret_cast<gr_f32x4*>(po + db * 16 + 4 * g) = o[rb][db];
      if (g == 0) *reinterpret_cast<gr_f32x2*>(a.part_ml + at * 2) = (gr_f32x2){m[rb], lt};
      continue;
    }
    // a row that saw no key: sum 0, result 0, lse -inf
    const float inv = lt == 0.f ? 0.f : 1.0f / lt;
    T* const op = static_cast<T*>(a.o) + t.b * a.o_sb + (long long)(t.first + token[rb]) * a.o_st + head[rb] * a.o_sh;
#pragma unroll
    for (int db = 0; db < DB; ++db)
      *reinterpret_cast<gr_u32x2*>(op + db * 16 + 4 * g) = (gr_u32x2){gr_pack2f<T>(o[rb][db][0] * inv, o[rb][db][1] * inv),
                                                                      gr_pack2f<T>(o[rb][db][2] * inv, o[rb][db][3] * inv)};
    if (a.lse && g == 0) {
      const long long lrow = a.starts ? t.first + token[rb] : (long long)t.b * a.rows + token[rb];
      a.lse[lrow * a.Hq + head[rb]] = lt == 0.f ? -GR_INF : (m[rb] * c + (__builtin_amdgcn_logf(lt) - shift)) * 0.6931471805599453f;
    }
  }
}
