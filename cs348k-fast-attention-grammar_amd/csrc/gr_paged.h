// gr_paged.h -- attention of new tokens over a paged key/value cache (gfx950,
// fp16 and bf16, head dims 64 and 128).
//
// A sequence has `len` keys in pages of a power of two of at least 16 slots
// and n new tokens, token i at position len - n + i. The G = Hq / Hkv query
// heads of a key head share its keys: the n G (token, head) rows of a sequence
// and key head are rows of one matrix, row r token r / G, and a workgroup takes
// a tile of 32 NW of them. A decode step's few heads so fill the rows of an
// MFMA, and a long chunk's tile covers 32 NW / G tokens.
//
//  * The products are the transposed ones of the flash body (gr_flash_fwd.h):
//    S^T = K Q^T and O^T = V^T P^T, so that a lane owns one row's softmax.
//    Scores are scaled on the vector unit in fp32.
//  * Keys come in tiles of BN from their pages straight into LDS. A load
//    instruction of a wave covers 64 / (D / 8) rows inside an aligned block of
//    16, which lies in one page: its base is scalar (page id by a scalar load a
//    tile ahead), the lanes' offsets are constant over the whole call.
//  * KG groups of NW waves each take every KG-th tile and merge through LDS.
//    With NW = 1 a wave reads only tiles that it loaded itself: no barrier.
//  * Keys of a tile are shared out over up to `parts` workgroups, of `chunk`
//    keys at least, which leave partial results for gr_paged_merge_body.
//  * Slots behind the part's last key, and pages whose id is out of range,
//    are written to LDS as zeros: what the cache holds there (NaN, say) does not
//    reach a product. A key that only some of a tile's rows may see, and whose
//    value is not finite, is taken out of the matrix product and added on the
//    vector unit to the rows that see it: 0 x inf would be NaN in the others.
#pragma once
#include "gr_flash_fwd.h"
#include "gr_gemm.h"

struct gr_paged_args {
  const void* q;
  void* o;
  float* lse;                      // [row of the batch][Hq] or nullptr
  long long q_sb, q_st, q_sh;      // batch (uniform batches), token, head
  long long o_sb, o_st, o_sh;
  const void* k;
  const void* v;
  long long k_sp, k_sh, k_ss;      // page, head, slot
  long long v_sp, v_sh, v_ss;
  const int* table;
  long long table_stride;
  const int* lens;
  const int* starts;               // nullptr: uniform batch of `rows` tokens
  int B, rows, width, pages, page_shift;
  int Hq, Hkv, G;
  int causal;
  float scale_log2;
  int tiles;                       // row tiles of a key head in the grid (an upper bound for ragged batches)
  int parts, chunk;                // key parts in the grid; fewest keys of a part (a multiple of 64)
  int chunk_long;                  // the same for sequences of more than one row tile
  float* part_o;                   // [(tile Hkv + key head) parts + part][row of the tile][D]
  float* part_ml;                  // the same, [2]: base (in scores), row sum
};

// A tile's place in the batch.
struct gr_paged_tile {
  int b, first;                    // sequence, its first row in a packed batch
  int n, row0, nrows;              // new tokens, first row of the tile, rows n G of the sequence
  int len, keys;                   // key count as given, and those that the page table can hold
  int kend;                        // keys that the tile's last row sees
  int per, np;                     // keys of a part, parts
};

// The tile-th tile of BM rows; false past the last one.
template <int BM>
__device__ __forceinline__ bool gr_paged_find(const gr_paged_args& a, int tile, int lane, gr_paged_tile& t) {
  int rt = -1;
  if (a.starts) {
    int before = 0;
    t.b = -1;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
      const int b = gr_imin(b0 + lane, a.B - 1);
      const int s0 = a.starts[b], s1 = a.starts[b + 1];
      // starts out of order or out of the batch: no tokens
      const int n = b0 + lane < a.B && s0 >= 0 && s1 > s0 && s1 <= a.rows ? s1 - s0 : 0;
      const int mine = (n * a.G + BM - 1) / BM;
      int upto = mine;                            // inclusive sum over the lanes
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const int x = __shfl_up(upto, off, 64);
        if (lane >= off) upto += x;
      }
      const unsigned long long past = __builtin_amdgcn_ballot_w64(before + upto > tile);
      if (past) {
        const int l = __builtin_ctzll(past);
        t.b = b0 + l;
        t.n = __builtin_amdgcn_readlane(n, l);
        t.first = __builtin_amdgcn_readlane(s0, l);
        rt = tile - before - (__builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(mine, l));
        break;
      }
      before += __builtin_amdgcn_readlane(upto, 63);
    }
    if (t.b < 0) return false;
  } else {
    const int per = (a.rows * a.G + BM - 1) / BM;
    t.b = tile / per;
    rt = tile - t.b * per;
    if (t.b >= a.B) return false;
    t.n = a.rows;
    t.first = 0;
  }
  t.nrows = t.n * a.G;
  const int ntile = (t.nrows + BM - 1) / BM;
  t.row0 = (ntile - 1 - rt) * BM;                 // the tiles that see the most keys first
  t.len = a.lens[t.b];
  const int cap = a.width << a.page_shift;
  t.keys = t.len < 0 ? 0 : gr_imin(t.len, cap);
  const int last = (gr_imin(t.row0 + BM, t.nrows) - 1) / a.G;
  // (len - n + last + 1 cannot wrap: n > last, and len is compared first)
  t.kend = a.causal ? gr_imin(t.keys, t.len < 0 ? 0 : t.len - t.n + last + 1) : t.keys;
  if (t.kend < 0) t.kend = 0;
  const int chunk = ntile > 1 ? a.chunk_long : a.chunk;
  const int even = ((t.kend + a.parts - 1) / a.parts + 63) & ~63;
  t.per = chunk > even ? chunk : even;
  t.np = a.parts == 1 ? 1 : (t.kend + t.per - 1) / t.per;
  if (t.np < 1) t.np = 1;
  return true;
}

// global_load_lds_dwordx4 from a scalar base plus a lane offset in bytes (see
// gr_g2lds16).
__device__ __forceinline__ void gr_g2lds16s(const void* base, unsigned off, unsigned lds) {
  unsigned saved;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %3\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %1, %2\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(saved)
      : "v"(off), "s"(base), "s"(lds)
      : "memory");
}

// A pointer that is the same in every lane, in scalar registers.
template <class P>
__device__ __forceinline__ P gr_uniform(P p) {
  const unsigned long long u = (unsigned long long)p;
  const unsigned lo = __builtin_amdgcn_readfirstlane((int)(unsigned)u), hi = __builtin_amdgcn_readfirstlane((int)(unsigned)(u >> 32));
  return (P)((unsigned long long)hi << 32 | lo);
}

template <int D, int BN, int NW, int KG>
struct gr_paged_lds {
  static constexpr int TILE = BN * D * 2;
  static constexpr int RING = 4 * TILE;                       // two slots of K and of V
  static constexpr int PART = 32 * D * 4 + 64 * 8;            // a wave's O, base and sum
  static constexpr int MERGE = (KG - 1) * NW * PART;
  static constexpr int BYTES = KG * RING > MERGE ? KG * RING : MERGE;
};

template <class T, int D, int BN, int NW, int KG>
__device__ __forceinline__ void gr_paged_body(const gr_paged_args& a, char* lds_all) {
  typedef gr_mfma<T> MF;
  typedef typename MF::vec8 vec8;
  typedef typename MF::vec2 vec2;
  typedef gr_paged_lds<D, BN, NW, KG> L;
  constexpr int BM = 32 * NW, NT = 64 * NW;
  constexpr int KB = BN / 32, DB = D / 32, DS = D / 16;
  constexpr int CPR = D / 8;                 // 16-byte chunks of a row
  constexpr int BLOCKS = BN / 16;            // 16-row blocks of a tile
  constexpr int IPB = 16 * CPR / 64;         // load instructions of a block
  constexpr int PER = BLOCKS * IPB / NW;     // of a wave, for K and for V
  static_assert(BLOCKS * IPB % NW == 0, "whole load instructions");
  constexpr bool SOLO = NW == 1;             // waves independent until the merge

  const int lane = threadIdx.x & 63;
  const int wave_all = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int kg = wave_all / NW, wave = wave_all % NW;
  const int g = lane >> 5, l32 = lane & 31;
  char* const lds = lds_all + kg * L::RING;
  char* const ks0 = lds;
  char* const vt0 = lds + 2 * L::TILE;

  // key head slowest, then the tiles: workgroups of one key head share an XCD's L2
  const int logical = gr_xcd_remap_any((int)blockIdx.x, (int)gridDim.x);
  const int part = logical % a.parts, ti = logical / a.parts;
  const int hk = ti / a.tiles, tile_id = ti - hk * a.tiles;
  gr_paged_tile t;
  if (!gr_paged_find<BM>(a, tile_id, lane, t)) return;
  t.b = __builtin_amdgcn_readfirstlane(t.b);
  if (part >= t.np) return;

  const int key0 = part * t.per;                              // multiples of 64
  const int key1 = gr_imin(t.kend, key0 + t.per);
  const int rw = t.row0 + wave * 32;                          // this wave's first row
  const bool wave_live = rw < t.nrows;
  const int row = gr_imin(rw + l32, t.nrows - 1);             // rows past the end: copies of the last
  const int token = row / a.G, head = hk * a.G + row % a.G;
  // the last key that the row sees; the wave's least and greatest
  const int base_pos = t.len - t.n;
  const int limit = a.causal ? gr_imin(base_pos + token, t.keys - 1) : t.keys - 1;
  const int lim_lo = a.causal ? gr_imin(base_pos + gr_imin(rw, t.nrows - 1) / a.G, t.keys - 1) : t.keys - 1;
  const int lim_hi = a.causal ? gr_imin(base_pos + gr_imin(rw + 31, t.nrows - 1) / a.G, t.keys - 1) : t.keys - 1;

  // this lane's Q row, 8 consecutive dims of every 16
  vec8 qf[DS];
  {
    const T* qp = static_cast<const T*>(a.q) + t.b * a.q_sb + (long long)(t.first + token) * a.q_st + head * a.q_sh;
#pragma unroll
    for (int ds = 0; ds < DS; ++ds) qf[ds] = gr_as<vec8>(gr_ld16(qp + ds * 16 + 8 * g));
  }

  // Load instruction i of the wave: 64 / CPR rows of LDS from row r0, in block
  // j = r0 / 16. K rows are stored with row bits 2 and 3 swapped, V rows as they
  // are; both swizzled (gr_swz for 16-byte row reads, gr_swz_tr for gr_tr_frag).
  unsigned koff[PER], voff[PER];              // lane byte offsets within the block's page slots
  int krow[PER];                              // LDS row of the lane; the key of a K chunk is gr_perm32 of it
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int c = lane + (wave + i * NW) * 64, r = c / CPR, pc = c % CPR;
    krow[i] = r;
    koff[i] = (unsigned)((gr_perm32(r) & 15) * a.k_ss * 2) + gr_swz<CPR>(r, pc) * 16;
    voff[i] = (unsigned)((r & 15) * a.v_ss * 2) + gr_swz_tr<CPR>(r, pc) * 16;
  }
  typedef __attribute__((address_space(4))) const int cint;   // the page table by scalar loads
  cint* const tab = (cint*)(unsigned long long)(a.table + t.b * a.table_stride);
  const int smask = (1 << a.page_shift) - 1;
  const T* const kp = static_cast<const T*>(a.k) + hk * a.k_sh;
  const T* const vp = static_cast<const T*>(a.v) + hk * a.v_sh;

  const int ntile_all = (key1 - key0 + BN - 1) / BN;
  const int ntile = (ntile_all - kg + KG - 1) / KG;           // of this group
  const int niter = SOLO ? ntile : (ntile_all + KG - 1) / KG; // of the workgroup (its barriers are everyone's)
  auto key_of = [&](int j) { return key0 + (j * KG + kg) * BN; };
  struct Ids { int id[BLOCKS]; };
  auto ids_of = [&](int j) {
    Ids x;
#pragma unroll
    for (int bl = 0; bl < BLOCKS; ++bl) x.id[bl] = tab[gr_imin((key_of(j) + 16 * bl) >> a.page_shift, a.width - 1)];
    return x;
  };
  auto bad_blocks = [&](const Ids& x) {       // blocks whose page id is out of range, a bit each
    unsigned m = 0;
#pragma unroll
    for (int bl = 0; bl < BLOCKS; ++bl) m |= ((unsigned)x.id[bl] >= (unsigned)a.pages ? 1u : 0u) << bl;
    return m;
  };
  auto load = [&](int j, int slot, const Ids& x) {
    const int k0 = key_of(j);
    const unsigned bad = bad_blocks(x);
    const bool whole = bad == 0 && k0 + BN <= key1;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int instr = wave + i * NW, bl = instr / IPB;
      int id = x.id[0];                       // (bl depends on the wave: a select, not an indexed read)
#pragma unroll
      for (int e = 1; e < BLOCKS; ++e) id = bl == e ? x.id[e] : id;
      char* const kd = ks0 + slot * L::TILE + instr * 1024;
      char* const vd = vt0 + slot * L::TILE + instr * 1024;
      const long long s = (k0 + 16 * bl) & smask;
      const bool ok = (unsigned)id < (unsigned)a.pages;
      const T* const kb = gr_uniform(kp + (ok ? id : 0) * a.k_sp + s * a.k_ss);
      const T* const vb = gr_uniform(vp + (ok ? id : 0) * a.v_sp + s * a.v_ss);
      const unsigned kl = __builtin_amdgcn_readfirstlane((int)gr_lds_addr(kd));
      const unsigned vl = __builtin_amdgcn_readfirstlane((int)gr_lds_addr(vd));
      if (whole) {
        gr_g2lds16s(kb, koff[i], kl);
        gr_g2lds16s(vb, voff[i], vl);
      } else {
        const int r = krow[i];
        if (ok && k0 + gr_perm32(r) < key1) gr_g2lds16s(kb, koff[i], kl);
        else gr_st16(kd + lane * 16, (gr_u32x4){0, 0, 0, 0});
        if (ok && k0 + r < key1) gr_g2lds16s(vb, voff[i], vl);
        else gr_st16(vd + lane * 16, (gr_u32x4){0, 0, 0, 0});
      }
    }
  };

  gr_f32x16 o[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) o[db] = (gr_f32x16)(0.f);
  float m = -GR_INF, l = 0.f;
  const float c = a.scale_log2;

  // One tile's scores, softmax and P V. MASK: some row may not see all of its keys.
  auto tile = [&](int j, int slot, unsigned bad, auto mask_tag) {
    constexpr bool MASK = decltype(mask_tag)::value;
    const int k0 = key_of(j);
    gr_f32x16 s[KB][1];
    vec8 qv[1][DS];
#pragma unroll
    for (int ds = 0; ds < DS; ++ds) qv[0][ds] = qf[ds];
    gr_flash_qk<T, D, BN, 1>(s, ks0 + slot * L::TILE, qv, l32, g);
    bool sees = true;                                          // whether the row sees any key of the tile
    if constexpr (MASK) {
      // element r of key block kb is key k0 + 32 kb + 16 (r / 8) + 8 g + r % 8
      const int delta = limit - k0 - 8 * g;
      bool any = false;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const bool vis = 32 * kb + 16 * (r >> 3) + (r & 7) <= delta && !(bad >> (2 * kb + (r >> 3)) & 1);
          any |= vis;
          if (!vis) s[kb][0][r] = -GR_INF;
        }
      sees = any;
    }
    vec8 pt[KB][2];
    float lt;
    auto make_p = [&](float nmc) {
      lt = 0.f;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          gr_u32x4 pw;
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            const float p0 = gr_exp2(fmaf(s[kb][0][8 * hf + e], c, nmc));
            const float p1 = gr_exp2(fmaf(s[kb][0][8 * hf + e + 1], c, nmc));
            const vec2 pp = __builtin_convertvector((gr_f32x2){p0, p1}, vec2);
            lt = MF::sum2(pp, lt);
            pw[e >> 1] = __builtin_bit_cast(unsigned, pp);
          }
          pt[kb][hf] = gr_as<vec8>(pw);
        }
    };
    bool ok = !gr_any(m == -GR_INF && sees);
    if (ok) {
      make_p(m == -GR_INF ? 0.f : -m * c);
      ok = !gr_any(!(lt <= GR_FLASH_SUM_MAX));
    }
    if (!ok) {
      float mt = -GR_INF;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) mt = fmaxf(mt, s[kb][0][r]);
      mt = fmaxf(mt, gr_xor32(mt));
      const float mn = fmaxf(m, mt);
      const float alpha = mn > m ? gr_exp2((m - mn) * c) : 1.f;   // m = -inf -> 0
      l *= alpha;
#pragma unroll
      for (int db = 0; db < DB; ++db) o[db] *= alpha;
      m = mn;
      make_p(m == -GR_INF ? 0.f : -m * c);
    }
    l += lt;
    const char* vt = vt0 + slot * L::TILE;
    if constexpr (MASK) {
      // keys with a value that is not finite: exponent bits all ones
      constexpr unsigned EXP = gr_is_same<T, _Float16>::value ? 0x7c007c00u : 0x7f807f80u;
      constexpr unsigned ONE = gr_is_same<T, _Float16>::value ? 0x04000400u : 0x00800080u;
      gr_u32x4 flags[KB][2];
      unsigned all = 0;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          flags[kb][hf] = (gr_u32x4)(0u);
#pragma unroll
          for (int db = 0; db < DB; ++db)
            flags[kb][hf] |= (gr_raw(gr_tr_frag<T, D, false>(vt, kb * 32 + 16 * hf, db * 32, lane)) & EXP) + ONE;
          flags[kb][hf] &= 0x80008000u;
          all |= flags[kb][hf][0] | flags[kb][hf][1] | flags[kb][hf][2] | flags[kb][hf][3];
        }
      if (__builtin_expect(gr_any(all != 0), 0)) {
        unsigned long long odd = 0;                            // those keys, a bit each
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int hf = 0; hf < 2; ++hf)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              // lanes 0-31 hold key e of the 16, lanes 32-63 key 8 + e
              const unsigned long long who =
                  __builtin_amdgcn_ballot_w64((flags[kb][hf][e >> 1] >> ((e & 1) ? 31 : 15)) & 1);
              odd |= ((unsigned long long)((unsigned)who != 0) | (unsigned long long)((who >> 32) != 0) << 8)
                     << (kb * 32 + 16 * hf + e);
            }
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            const unsigned byte = (unsigned)(odd >> (kb * 32 + 16 * hf + 8 * g)) & 0xffu;
            gr_u32x4 keep;                                     // halfwords of the keys that stay in the product
#pragma unroll
            for (int e = 0; e < 4; ++e)
              keep[e] = ((byte >> (2 * e)) & 1 ? 0u : 0x0000ffffu) | ((byte >> (2 * e + 1)) & 1 ? 0u : 0xffff0000u);
#pragma unroll
            for (int db = 0; db < DB; ++db) {
              const gr_u32x4 w = gr_raw(gr_tr_frag<T, D, false>(vt, kb * 32 + 16 * hf, db * 32, lane));
              o[db] = MF::mma32(gr_as<vec8>(w & keep), pt[kb][hf], o[db]);
            }
          }
#pragma unroll 1
        for (; odd; odd &= odd - 1) {
          const int key = __builtin_ctzll(odd);
          float p = 0.f;                                       // this lane's p of the key, if its half has it
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int hf = 0; hf < 2; ++hf)
#pragma unroll
              for (int e = 0; e < 8; ++e)
                if (key == kb * 32 + 16 * hf + 8 * g + e) p = (float)pt[kb][hf][e];
          p += gr_xor32(p);                                    // the other half's is 0
          const bool vis = k0 + key <= limit && !(bad >> (key >> 4) & 1);
          const char* const vr = vt + key * (D * 2);
#pragma unroll
          for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const int d = db * 32 + 8 * (r >> 2) + 4 * g + (r & 3);
              const float v = (float)*reinterpret_cast<const T*>(vr + gr_swz_tr<CPR>(key, d >> 3) * 16 + (d & 7) * 2);
              if (vis) o[db][r] = fmaf(p, v, o[db][r]);
              if ((r & 3) == 3) __builtin_amdgcn_sched_barrier(0);   // not all reads at once: they would spill
            }
        }
        return;
      }
    }
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int hf = 0; hf < 2; ++hf)
#pragma unroll
        for (int db = 0; db < DB; ++db)
          o[db] = MF::mma32(gr_tr_frag<T, D, false>(vt, kb * 32 + 16 * hf, db * 32, lane), pt[kb][hf], o[db]);
  };

  // Iteration j reads slot j & 1; tile j + 1 is on its way to the other. A
  // part-filled tile's zeros are LDS stores, so a wave alone also waits on them.
  Ids cur = {}, nxt = {};
  unsigned bad = 0;
  if (ntile > 0) {
    cur = ids_of(0);
    bad = bad_blocks(cur);
    load(0, 0, cur);
    if (ntile > 1) nxt = ids_of(1);
  }
  // Q has landed before the loop: the compiler cannot see that through the
  // loop's back edge and would wait for every load in flight in each tile
  __builtin_amdgcn_s_waitcnt(0);
  auto step = [&](int j, int slot) {
    if constexpr (SOLO) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");      // the slot's last reads are over
      if (j + 1 < ntile) load(j + 1, slot ^ 1, nxt);
      if (j + 1 < ntile && key_of(j + 1) + BN <= key1) {
        // (a part-filled or bad next tile issues fewer loads: then all are waited for)
        if (bad_blocks(nxt) == 0) gr_wait_vmcnt<2 * PER>();
        else gr_wait_vmcnt<0>();
      } else {
        gr_wait_vmcnt<0>();
      }
      asm volatile("" ::: "memory");
    } else {
      gr_wait_vmcnt<0>();
      __syncthreads();                                         // tile j is there, and the other slot free
      if (j + 1 < ntile) load(j + 1, slot ^ 1, nxt);
    }
    const unsigned bad_now = bad;
    if (j + 1 < ntile) bad = bad_blocks(nxt);
    if (j + 2 < ntile) nxt = ids_of(j + 2);
    const int k0 = key_of(j);
    if (wave_live && j < ntile && k0 <= lim_hi) {
      if (k0 + BN - 1 <= lim_lo && bad_now == 0) tile(j, slot, 0u, gr_ic<0>{});
      else tile(j, slot, bad_now, gr_ic<1>{});
    }
  };
#pragma unroll 1
  for (int j = 0; j < niter; ++j) step(j, j & 1);

  if constexpr (KG > 1) {
    // the groups' partials through LDS: O as 4 DB quads of floats per lane,
    // then base and row sum
    __syncthreads();
    auto at = [&](int grp) { return lds_all + ((grp - 1) * NW + wave) * L::PART + lane * 16; };
    if (kg > 0) {
      char* const w = at(kg);
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int rr = 0; rr < 4; ++rr)
          *reinterpret_cast<gr_f32x4*>(w + (db * 4 + rr) * 1024) =
              (gr_f32x4){o[db][4 * rr], o[db][4 * rr + 1], o[db][4 * rr + 2], o[db][4 * rr + 3]};
      *reinterpret_cast<gr_f32x2*>(w + DB * 4096 - lane * 8) = (gr_f32x2){m, l};
    }
    __syncthreads();
    if (kg > 0) return;
    gr_f32x2 ml[KG];
    float mx = m;
#pragma unroll
    for (int k = 1; k < KG; ++k) {
      ml[k] = *reinterpret_cast<const gr_f32x2*>(at(k) + DB * 4096 - lane * 8);
      mx = fmaxf(mx, ml[k][0]);
    }
    const float base = mx == -GR_INF ? 0.f : mx;
    const float w0 = gr_exp2((m - base) * c);
    l *= w0;
#pragma unroll
    for (int db = 0; db < DB; ++db) o[db] *= w0;
    m = mx;
#pragma unroll
    for (int k = 1; k < KG; ++k) {
      const float wk = gr_exp2((ml[k][0] - base) * c);
      l = fmaf(wk, ml[k][1], l);
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int rr = 0; rr < 4; ++rr) {
          const gr_f32x4 v = *reinterpret_cast<const gr_f32x4*>(at(k) + (db * 4 + rr) * 1024);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[db][4 * rr + e] = fmaf(wk, v[e], o[db][4 * rr + e]);
        }
    }
  }

  const bool live = rw + l32 < t.nrows;
  const float lt = l + gr_xor32(l);
  if (t.np > 1) {
    // unnormalised O and (base, row sum) of this part
    const long long at = ((long long)(tile_id * a.Hkv + hk) * a.parts + part) * BM + wave * 32 + l32;
    if (live) {
      float* const po = a.part_o + at * D;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int rr = 0; rr < 4; ++rr)
          *reinterpret_cast<gr_f32x4*>(po + db * 32 + 8 * rr + 4 * g) =
              (gr_f32x4){o[db][4 * rr], o[db][4 * rr + 1], o[db][4 * rr + 2], o[db][4 * rr + 3]};
      if (g == 0) *reinterpret_cast<gr_f32x2*>(a.part_ml + at * 2) = (gr_f32x2){m, lt};
    }
    return;
  }
  // a row that saw no key: sum 0, result 0, lse -inf
  const float inv = lt == 0.f ? 0.f : 1.0f / lt;
  if (live) {
    T* const op = static_cast<T*>(a.o) + t.b * a.o_sb + (long long)(t.first + token) * a.o_st + head * a.o_sh;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int rr = 0; rr < 4; ++rr) {
        gr_u32x2 w = {gr_pack2f<T>(o[db][4 * rr] * inv, o[db][4 * rr + 1] * inv),
                      gr_pack2f<T>(o[db][4 * rr + 2] * inv, o[db][4 * rr + 3] * inv)};
        *reinterpret_cast<gr_u32x2*>(op + db * 32 + 8 * rr + 4 * g) = w;
      }
    if (a.lse && g == 0) {
      const long long trow = a.starts ? t.first + token : (long long)t.b * a.rows + token;
      a.lse[trow * a.Hq + head] = lt == 0.f ? -GR_INF : (m * c + __builtin_amdgcn_logf(lt)) * 0.6931471805599453f;
    }
  }
}

// Merges the key parts of a tile's rows, a wave to a row: O = sum_p w_p O_p /
// sum_p w_p l_p with w_p = 2^((m_p - max m) c), the parts in order.
template <class T, int D, int BM>
__device__ __forceinline__ void gr_paged_merge_body(const gr_paged_args& a) {
  constexpr int V = D / 64;                  // floats a lane
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), nw = blockDim.x >> 6;
  const int hk = blockIdx.x / a.tiles, tile_id = blockIdx.x - hk * a.tiles;
  gr_paged_tile t;
  if (!gr_paged_find<BM>(a, tile_id, lane, t) || t.np == 1) return;
  const float c = a.scale_log2;
  const int rows = gr_imin(BM, t.nrows - t.row0);
  for (int r = (int)blockIdx.y * nw + wave; r < rows; r += nw * gridDim.y) {
    const long long at = ((long long)(tile_id * a.Hkv + hk) * a.parts) * BM + r;
    float mx = -GR_INF;
    for (int p = lane; p < t.np; p += 64) mx = fmaxf(mx, a.part_ml[(at + (long long)p * BM) * 2]);
    mx = gr_wave_max(mx);
    const float base = mx == -GR_INF ? 0.f : mx;
    float l = 0.f, o[V];
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] = 0.f;
    for (int p = 0; p < t.np; ++p) {
      const long long ap = at + (long long)p * BM;
      const gr_f32x2 ml = *reinterpret_cast<const gr_f32x2*>(a.part_ml + ap * 2);
      const float w = gr_exp2((ml[0] - base) * c);
      l = fmaf(w, ml[1], l);
      float x[V];
      gr_row_load<V>(x, a.part_o + ap * D + lane * V);
#pragma unroll
      for (int e = 0; e < V; ++e) o[e] = fmaf(w, x[e], o[e]);
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] *= inv;
    const int token = (t.row0 + r) / a.G, head = hk * a.G + (t.row0 + r) % a.G;
    gr_row_store<V>(static_cast<T*>(a.o) + t.b * a.o_sb + (long long)(t.first + token) * a.o_st + head * a.o_sh + lane * V, o);
    if (a.lse && lane == 0) {
      const long long trow = a.starts ? t.first + token : (long long)t.b * a.rows + token;
      a.lse[trow * a.Hq + head] = l == 0.f ? -GR_INF : (mx * c + __builtin_amdgcn_logf(l)) * 0.6931471805599453f;
    }
  }
}
