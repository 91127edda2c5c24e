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
//  * Few tiles (`shares` > 0): the work of the call, counted in blocks of 64 keys
//    over all tiles and key heads, is cut into equal runs, one a workgroup, by
//    the lengths as they are on the device. A run covers a tile's end, whole
//    tiles and a tile's start; tiles that several runs cover are merged by
//    gr_paged_merge_body. Many tiles: a workgroup each.
//  * Slots behind the part's last key, and pages whose id is out of range,
//    are written to LDS as zeros: what the cache holds there (NaN, say) does not
//    reach a product. A key that only some of a tile's rows may see, and whose
//    value is not finite, is taken out of the matrix product and added on the
//    vector unit to the rows that see it: 0 x inf would be NaN in the others.
//
// Measured (bf16, 32 / 8 heads of 128). A token each of 48 sequences of 150 to 8,000
// keys (848 MB): 147-150 us, 5.7 TB/s, bound by memory (matrix cores 8 % busy), and
// 4.8 for the merge. 4,096 tokens onto 4,096: 403-440 us by clocks, 940-1,020 TFLOP/s,
// bound by the MFMAs and the softmax of two waves a SIMD taking turns (matrix cores
// 49 % busy, no LDS conflicts). Small grids are bound by a workgroup's chain of steps, 1.2-1.3 us
// for 64 keys of 128 rows: 419 keys of one token (16 heads of 64) take 7.2 us.
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
  int tiles;                       // row tiles of a key head (an upper bound for ragged batches)
  int shares;                      // workgroups that share the work out; 0: a workgroup a tile
  float* part_o;                   // [2 share + place][row of the tile][D]
  float* part_ml;                  // the same, [2]: base (in scores), row sum
};

// A tile's place in the batch.
struct gr_paged_tile {
  int b, first;                    // sequence, its first row in a packed batch
  int n, row0, nrows;              // new tokens, first row of the tile, rows n G of the sequence
  int len, keys;                   // key count as given, and those that the page table can hold
  int kend;                        // keys that the tile's last row sees
  int nb;                          // blocks of 64 keys, 1 at least
  int block;                       // found by block: the block in the tile (from nb on: its cost)
  int x0;                          // blocks of a key head before the tile's
};

// What a tile costs beside its keys (page ids, Q, the first tile's way, the
// merge), in blocks of 64 keys: counted behind its last block. (32 sequences of 320
// to 960 keys, one token each: 29.6 us with 0, 25.5 with 5; 2 and 3 lie between.)
constexpr int GR_PAGED_COST = 5;

// Blocks of 64 keys of a sequence, as its tiles are counted (1 for none: its
// rows are written all the same).
__device__ __forceinline__ int gr_paged_keys(const gr_paged_args& a, int len) {
  return len < 0 ? 0 : gr_imin(len, a.width << a.page_shift);
}
__device__ __forceinline__ int gr_paged_blocks(int keys) { return keys > 64 ? (keys + 63) >> 6 : 1; }

// Sequence b's new tokens and, in a packed batch, its first row. Starts out of
// order or out of the batch: no tokens.
__device__ __forceinline__ int gr_paged_news(const gr_paged_args& a, int b, int& first) {
  first = 0;
  if (!a.starts) return a.rows;
  first = a.starts[b];
  const int s1 = a.starts[b + 1];
  return first >= 0 && s1 > first && s1 <= a.rows ? s1 - first : 0;
}

// Sum over lanes 0 .. l, for every lane l (DPP: a few cycles a step, a tenth of
// what a shuffle through LDS takes).
__device__ __forceinline__ int gr_wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);    // row_shr:1 (rows of 16 lanes)
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);    // row_shr:2
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);    // row_shr:4
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);    // row_shr:8
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);   // row_bcast:15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);   // row_bcast:31 into rows 2 and 3
  return v;
}

// 64 sequences, one a lane, and where their tiles and blocks begin.
template <int BM, bool SMALL>
struct gr_paged_seqs {
  int b0 = -1;
  int only = 0;                    // SMALL: 1 and 2 leave out sequences of at most and of more than 32 rows
  int tiles, blocks;               // before these 64
  int first, n, len, nt, nb;       // of the lane's sequence: tiles, blocks of a tile
  int tsum, bsum;                  // tiles and blocks of the 64 up to and with it
  __device__ __forceinline__ void load(const gr_paged_args& a, int from, int tiles0, int blocks0, int lane) {
    b0 = from;
    tiles = tiles0;
    blocks = blocks0;
    const int b = gr_imin(from + lane, a.B - 1);
    len = a.lens[b];
    n = gr_paged_news(a, b, first);
    const int rows = n * a.G;
    nt = from + lane >= a.B || rows == 0 ? 0 : SMALL && rows <= 32 ? 1 : (rows + BM - 1) / BM;
    if (SMALL && only == (rows <= 32 ? 1 : 2)) nt = 0;
    nb = gr_paged_blocks(gr_paged_keys(a, len));
    // Starts that overlap could make more tiles than the grid, and more blocks than 32
    // bits count (a head's number from them could then be below 0): tiles past the
    // grid's are left out. Starts in order never make them.
    nt = gr_imin(nt, a.tiles);
    tsum = gr_wave_scan(nt);
    if (__builtin_expect(tiles_after() > a.tiles, 0)) {
      const int over = tiles + tsum - a.tiles;
      nt = over <= 0 ? nt : nt > over ? nt - over : 0;
      tsum -= over > 0 ? over : 0;
    }
    bsum = gr_wave_scan((int)((unsigned)nt * (nb + GR_PAGED_COST)));
  }
  __device__ __forceinline__ int tiles_after() const { return tiles + __builtin_amdgcn_readlane(tsum, 63); }
  __device__ __forceinline__ int blocks_after() const { return blocks + __builtin_amdgcn_readlane(bsum, 63); }

  // Tiles of one key head.
  __device__ __forceinline__ int count(const gr_paged_args& a, int lane) {
    load(a, 0, 0, 0, lane);
    int sum = tiles_after();
    if (a.B > 64) {
      gr_paged_seqs more;
      more.only = only;
      for (int from = 64; from < a.B; from += 64) {
        more.load(a, from, sum, 0, lane);
        sum = more.tiles_after();
      }
    }
    return sum;
  }

  // Blocks of one key head over all tiles.
  __device__ __forceinline__ int total(const gr_paged_args& a, int lane) {
    load(a, 0, 0, 0, lane);
    int sum = blocks_after();
    if (a.B > 64) {
      gr_paged_seqs more;
      for (int from = 64; from < a.B; from += 64) {
        more.load(a, from, 0, sum, lane);
        sum = more.blocks_after();
      }
    }
    return sum;
  }

  // BLOCK: the tile of the at-th block of a key head, else the at-th tile;
  // false past the last one.
  template <bool BLOCK>
  __device__ __forceinline__ bool find(const gr_paged_args& a, int at, int lane, gr_paged_tile& t) {
    if (b0 < 0 || (BLOCK ? blocks : tiles) > at) load(a, 0, 0, 0, lane);
    while ((BLOCK ? blocks_after() : tiles_after()) <= at) {
      if (b0 + 64 >= a.B) return false;
      load(a, b0 + 64, tiles_after(), blocks_after(), lane);
    }
    const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64((BLOCK ? blocks + bsum : tiles + tsum) > at));
    t.b = b0 + l;
    t.n = __builtin_amdgcn_readlane(n, l);
    t.first = __builtin_amdgcn_readlane(first, l);
    t.len = __builtin_amdgcn_readlane(len, l);
    t.nb = __builtin_amdgcn_readlane(nb, l);
    const int before = blocks + __builtin_amdgcn_readlane(bsum - (int)((unsigned)nt * (nb + GR_PAGED_COST)), l);
    const int per = t.nb + GR_PAGED_COST;
    const int rt = BLOCK ? (at - before) / per : at - tiles - __builtin_amdgcn_readlane(tsum - nt, l);
    t.x0 = before + rt * per;
    t.block = at - t.x0;
    t.nrows = t.n * a.G;
    const int ntile = (t.nrows + BM - 1) / BM;    // (one, whatever its size, for at most 32 rows)
    t.row0 = (ntile - 1 - rt) * BM;               // the tiles that see the most keys first
    t.keys = gr_paged_keys(a, t.len);
    const int last = (gr_imin(t.row0 + BM, t.nrows) - 1) / a.G;
    // (len - n + last + 1 cannot wrap: n > last, and len is compared first)
    t.kend = a.causal ? gr_imin(t.keys, t.len < 0 ? 0 : t.len - t.n + last + 1) : t.keys;
    if (t.kend < 0) t.kend = 0;
    return true;
  }
};

// The shares of a call's `total` blocks: as many as workgroups, fewer if a share
// would not get 4 blocks; the first `rest` get per + 1 blocks, the others per.
struct gr_paged_cut {
  int W, per, rest;
  __device__ __forceinline__ gr_paged_cut(int total, int shares) {
    W = total >> 2 < shares ? (total + 3) >> 2 : shares;
    per = W > 0 ? total / W : 0;
    rest = total - per * W;
  }
  __device__ __forceinline__ int begin(int w) const { return w * per + gr_imin(w, rest); }
  __device__ __forceinline__ int of(int x) const {               // the share of block x
    const int big = rest * (per + 1);
    return x < big ? x / (per + 1) : rest + (x - big) / per;
  }
};

// global_load_lds_dwordx4 from scalar bases plus lane offsets in bytes (see
// gr_g2lds16); M0 holds the LDS address. The bases come from lane reads, which are
// vector instructions: a memory instruction may read a scalar register no sooner
// than five wait states after one wrote it. The compiler cannot see these loads,
// so the wait (s_nop 4) is part of each group.
__device__ __forceinline__ void gr_g2lds16s(unsigned long long base, unsigned off, unsigned lds) {
  asm volatile(
      "s_mov_b32 m0, %2\n\t"
      "s_nop 4\n\t"
      "global_load_lds_dwordx4 %0, %1"
      :
      : "v"(off), "s"(base), "s"(lds)
      : "memory", "m0");
}

// N loads of K and N of V, the K loads STEP bytes of LDS apart, V's VOFF behind.
template <int N, int STEP, int VOFF>
__device__ __forceinline__ void gr_g2lds16_kv(unsigned long long kb, unsigned long long vb, const unsigned* koff,
                                              const unsigned* voff, unsigned lds) {
  static_assert(N == 1 || N == 2 || N == 4, "loads of a group");
  if constexpr (N == 1)
    asm volatile(
        "s_mov_b32 m0, %4\n\ts_nop 4\n\t"
        "global_load_lds_dwordx4 %0, %2\n\t"
        "s_add_u32 m0, m0, %5\n\ts_nop 0\n\t"
        "global_load_lds_dwordx4 %1, %3"
        :
        : "v"(koff[0]), "v"(voff[0]), "s"(kb), "s"(vb), "s"(lds), "n"(VOFF)
        : "memory", "m0", "scc");
  else if constexpr (N == 2)
    asm volatile(
        "s_mov_b32 m0, %6\n\ts_nop 4\n\t"
        "global_load_lds_dwordx4 %0, %4\n\t"
        "s_add_u32 m0, m0, %7\n\ts_nop 0\n\t"
        "global_load_lds_dwordx4 %1, %4\n\t"
        "s_add_u32 m0, m0, %8\n\ts_nop 0\n\t"
        "global_load_lds_dwordx4 %2, %5\n\t"
        "s_add_u32 m0, m0, %7\n\ts_nop 0\n\t"
        "global_load_lds_dwordx4 %3, %5"
        :
        : "v"(koff[0]), "v"(koff[1]), "v"(voff[0]), "v"(voff[1]), "s"(kb), "s"(vb), "s"(lds), "n"(STEP), "n"(VOFF - STEP)
        : "memory", "m0", "scc");
  else
    asm volatile(
        "s_mov_b32 m0, %10\n\ts_nop 4\n\t"
        "global_load_lds_dwordx4 %0, %8\n\t"
        "s_add_u32 m0, m0, %11\n\ts_nop 0\n\t"
        "global_load_lds_dwordx4 %1, %8\n\t"
        "s_add_u32 m0, m0, %11\n\ts_nop 0\n\t"
        "global_load_lds_dwordx4 %2, %8\n\t"
        "s_add_u32 m0, m0, %11\n\ts_nop 0\n\t"
        "global_load_lds_dwordx4 %3, %8\n\t"
        "s_add_u32 m0, m0, %12\n\ts_nop 0\n\t"
        "global_load_lds_dwordx4 %4, %9\n\t"
        "s_add_u32 m0, m0, %11\n\ts_nop 0\n\t"
        "global_load_lds_dwordx4 %5, %9\n\t"
        "s_add_u32 m0, m0, %11\n\ts_nop 0\n\t"
        "global_load_lds_dwordx4 %6, %9\n\t"
        "s_add_u32 m0, m0, %11\n\ts_nop 0\n\t"
        "global_load_lds_dwordx4 %7, %9"
        :
        : "v"(koff[0]), "v"(koff[1]), "v"(koff[2]), "v"(koff[3]), "v"(voff[0]), "v"(voff[1]), "v"(voff[2]), "v"(voff[3]),
          "s"(kb), "s"(vb), "s"(lds), "n"(STEP), "n"(VOFF - 3 * STEP)
        : "memory", "m0", "scc");
}

// XOR swizzle of K's 16-byte chunks for reads of consecutive rows at one logical
// chunk: 8 and 16 rows of an aligned 16 fall on distinct bank groups, as with
// gr_swz, by row bits 0 to 3 only.
template <int CPR>
__device__ __forceinline__ int gr_paged_swz(int row, int chunk) {
  return CPR >= 16 ? chunk ^ (row & 15) : chunk ^ ((row & 7) ^ ((row >> 3) & 1));
}

// P is rounded to the type before its product with V, as in the flash body, and the
// row sum is taken of the rounded ones, so that what a rounding adds to a key's weight
// divides out in part; sums, bases and partial results are fp32. fp16 alone would
// drop weights below 2^-25 of the base (the row's max when its base was taken)
// and round those below 2^-14 to whole steps of 2^-24, which many alike keys add
// up (131,072 keys of 2^-25.05 beside one of 1: 0.7 % of the result). So fp16's P, row
// sums and O carry a factor of 2^shift, which divides out of O and leaves the
// log-sum-exp at the end, by the sequence's keys: N keys lose N 2^-(25 + shift) of
// the base at most, 2^-14 (an eighth of a rounding of P) for up to 2^26 keys. P then
// overflows 16 - shift powers of two above the base, and the tile is redone from a
// new one: no more shift than is needed (4,096 tokens onto 4,096, 16 heads of 64 with
// scores of deviation 3: 162 us with 0 or the 2 that it takes, 171 with 8, 183 with 12).
template <class T>
__device__ __forceinline__ float gr_paged_shift(int keys) {
  if (!gr_is_same<T, _Float16>::value || keys <= 2048) return 0.f;
  return (float)gr_imin(32 - __builtin_clz((unsigned)(keys - 1)) - 11, 15);
}

template <int D, int BN, int NW, int KG, int NS>
struct gr_paged_lds {
  static constexpr int TILE = BN * D * 2;
  static constexpr int RING = 2 * NS * TILE;                  // NS slots of K, then of V
  static constexpr int PART = 32 * D * 4 + 64 * 8;            // a wave's O, base and sum
  static constexpr int MERGE = (KG - 1) * NW * PART;
  static constexpr int BYTES = KG * RING > MERGE ? KG * RING : MERGE;
};

// One tile over keys [key0, key1), by NW KG waves of the workgroup's WAVES; place:
// where its partial result of BM rows goes, or -1 for a tile that is done here.
template <class T, int D, int BN, int NW, int KG, int NS, int WAVES, int BM>
__device__ __forceinline__ void gr_paged_segment(const gr_paged_args& a, char* lds_all, const gr_paged_tile& t, int hk,
                                                 int key0, int key1, int place) {
  typedef gr_mfma<T> MF;
  typedef typename MF::vec8 vec8;
  typedef typename MF::vec2 vec2;
  typedef gr_paged_lds<D, BN, NW, KG, NS> L;
  constexpr bool SOLO = NW == 1;             // waves independent until the merge
  constexpr bool HALF = gr_is_same<T, _Float16>::value;
  constexpr int KB = BN / 32, DB = D / 32, DS = D / 16;
  constexpr int CPR = D / 8;                 // 16-byte chunks of a row
  constexpr int BLOCKS = BN / 16;            // 16-row blocks of a tile
  constexpr int IPB = 16 * CPR / 64;         // load instructions of a block
  constexpr int PER = BLOCKS * IPB / NW;     // of a wave, for K and for V
  static_assert(BLOCKS * IPB % NW == 0, "whole load instructions");

  const int lane = threadIdx.x & 63;
  const int wave_all = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int kg = wave_all / NW, wave = wave_all % NW;
  if (NW * KG < WAVES && kg >= KG) {          // a wave without a part: the merge's barriers only
    if constexpr (KG > 1) {
      __syncthreads();
      __syncthreads();
    }
    return;
  }
  static_assert(NW * KG == WAVES || SOLO, "the loop's barriers are every wave's");
  const int g = lane >> 5, l32 = lane & 31;
  char* const lds = lds_all + kg * L::RING;
  char* const ks0 = lds;
  char* const vt0 = lds + NS * L::TILE;

  // Load instruction i of the wave is number wave + i NW of the tile: 64 / CPR
  // rows of LDS, part `sub` of the IPB of a block of 16 rows. K rows are stored
  // with row bits 2 and 3 swapped, V rows as they are; both swizzled (gr_paged_swz
  // for 16-byte row reads, gr_swz_tr for gr_tr_frag) by row bits 0 to 3, so that a
  // lane's offset from its block's first slot depends on sub alone.
  constexpr int SUBS = IPB > NW ? IPB / NW : 1;
  auto block_row = [&](int i) { return lane / CPR + ((wave + i * NW) % IPB) * (64 / CPR); };
  unsigned koff[SUBS], voff[SUBS];            // bytes
#pragma unroll
  for (int i = 0; i < SUBS; ++i) {
    const int r = block_row(i), pc = lane % CPR;
    koff[i] = (unsigned)((gr_perm32(r) & 15) * a.k_ss * 2) + gr_paged_swz<CPR>(r, pc) * 16;
    voff[i] = (unsigned)(r * a.v_ss * 2) + gr_swz_tr<CPR>(r, pc) * 16;
  }
  const float c = a.scale_log2, shift = gr_paged_shift<T>(t.keys);
  // LDS addresses of the fragments: the swizzles are XORs of chunk bits, so a
  // fragment's is a lane constant XOR an immediate, plus whole rows.
  //  K (gr_paged_swz): row 32 kb + l32, chunk 2 ds + g
  //  V (gr_tr_frag): rows 16 x + 8 g + 4 h + (lane / 4) % 4, columns 32 db + ...
  const int kbase = l32 * (D * 2) + gr_paged_swz<CPR>(l32, g) * 16;
  const int vcol = 16 * ((lane >> 4) & 1) + 4 * (lane & 3), vrow = 8 * g + ((lane >> 2) & 3);
  const int vbase = vrow * (D * 2) + gr_swz_tr<CPR>(vrow, vcol >> 3) * 16 + (vcol & 7) * 2;
  const int smask = (1 << a.page_shift) - 1;

  const int rw = t.row0 + wave * 32;                          // this wave's first row
  const bool wave_live = rw < t.nrows;
  const int row = gr_imin(rw + l32, t.nrows - 1);             // rows past the end: copies of the last
  const int token = row / a.G, head = hk * a.G + row % a.G;
  // the last key that the row sees; the wave's least and greatest
  const int base_pos = t.len - t.n;
  const int limit = a.causal ? gr_imin(base_pos + token, t.keys - 1) : t.keys - 1;
  const int lim_lo = a.causal ? gr_imin(base_pos + gr_imin(rw, t.nrows - 1) / a.G, t.keys - 1) : t.keys - 1;
  const int lim_hi = a.causal ? gr_imin(base_pos + gr_imin(rw + 31, t.nrows - 1) / a.G, t.keys - 1) : t.keys - 1;

  const int* const tab = a.table + t.b * a.table_stride;
  const T* const kp = static_cast<const T*>(a.k) + hk * a.k_sh;
  const T* const vp = static_cast<const T*>(a.v) + hk * a.v_sh;

  const int ntile_all = key1 > key0 ? (key1 - key0 + BN - 1) / BN : 0;
  const int ntile = (ntile_all - kg + KG - 1) / KG;           // of this group
  const int niter = SOLO ? ntile : (ntile_all + KG - 1) / KG; // of the workgroup (its barriers are everyone's)
  auto key_of = [&](int j) { return key0 + (j * KG + kg) * BN; };
  // Where the blocks of this group's tiles are: lane l has block l % BLOCKS of
  // tile j0 + l / BLOCKS, its K and V addresses and (a bit each) whether its page
  // exists; refilled every 64 / BLOCKS tiles. A tile's loads take their scalar
  // bases from it by lane reads (worked out by scalar multiplications they cost more
  // than the loads). The page ids are read when a window begins, not ahead: kept
  // over the tiles in a register, they made the compiler wait for all loads in
  // every tile.
  constexpr int WIN = 64 / BLOCKS;
  auto id_of = [&](int j0) {
    const long long key = key0 + ((long long)(j0 + lane / BLOCKS) * KG + kg) * BN + 16 * (lane % BLOCKS);
    return tab[key >> a.page_shift < a.width ? (int)(key >> a.page_shift) : a.width - 1];
  };
  unsigned long long kwin = 0, vwin = 0, badwin = 0;
  auto refill = [&](int j0, int id) {
    const int key = key0 + ((j0 + lane / BLOCKS) * KG + kg) * BN + 16 * (lane % BLOCKS), slot = key & smask;
    const bool ok = (unsigned)id < (unsigned)a.pages;
    kwin = (unsigned long long)(kp + (ok ? id : 0) * a.k_sp + slot * a.k_ss);
    vwin = (unsigned long long)(vp + (ok ? id : 0) * a.v_sp + slot * a.v_ss);
    badwin = __builtin_amdgcn_ballot_w64(!ok && key < key1);
  };
  auto lane64 = [&](unsigned long long w, int l) {
    return (unsigned long long)(unsigned)__builtin_amdgcn_readlane((int)(w >> 32), l) << 32
           | (unsigned)__builtin_amdgcn_readlane((int)(unsigned)w, l);
  };
  const unsigned kring = __builtin_amdgcn_readfirstlane((int)gr_lds_addr(ks0));
  // Asks for tile j: 2 PER loads of the wave if all of its keys are there, SUBS of
  // K and of V for each block that it has a part of.
  auto load = [&](int j, int slot, auto whole_tag, unsigned bad) {
    constexpr bool WHOLE = decltype(whole_tag)::value;
    const int at = (j & (WIN - 1)) * BLOCKS;
#pragma unroll
    for (int n = 0; n < PER / SUBS; ++n) {
      const int instr = wave + n * SUBS * NW, bl = instr / IPB;
      const unsigned long long kb = lane64(kwin, at + bl), vb = lane64(vwin, at + bl);
      const unsigned kl = kring + slot * L::TILE + instr * 1024;
      if constexpr (WHOLE) {
        gr_g2lds16_kv<SUBS, NW * 1024, NS * L::TILE>(kb, vb, koff, voff, kl);
      } else {
        const bool ok = !(bad >> bl & 1);
#pragma unroll
        for (int i = 0; i < SUBS; ++i) {
          char* const kd = ks0 + slot * L::TILE + (instr + i * NW) * 1024 + lane * 16;
          const int r = block_row(i), kblk = key_of(j) + 16 * bl;
          if (ok && kblk + gr_perm32(r) < key1) gr_g2lds16s(kb, koff[i], kl + i * NW * 1024);
          else gr_st16(kd, (gr_u32x4){0, 0, 0, 0});
          if (ok && kblk + r < key1) gr_g2lds16s(vb, voff[i], kl + i * NW * 1024 + NS * L::TILE);
          else gr_st16(kd + NS * L::TILE, (gr_u32x4){0, 0, 0, 0});
        }
      }
    }
  };

  vec8 qf[DS];
  gr_f32x16 o[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) o[db] = (gr_f32x16)(0.f);
  float m = -GR_INF, l = 0.f, base = shift;    // the row's base, its sum, shift - m c (no base yet: shift)

  // One tile's scores, softmax and P V. MASKED: some row may not see all of its
  // keys (bad: 16-key blocks of no page, a bit each).
  auto tile = [&](int j, int slot, unsigned bad, auto masked_tag) {
    constexpr bool MASKED = decltype(masked_tag)::value;
    const int k0 = key_of(j);
    const int ka = kbase + slot * L::TILE, va = vbase + slot * L::TILE;
    auto vfrag = [&](int x, int db) -> vec8 {       // 16 keys x, head dims 32 db on
      typedef short v4s __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) v4s lds_v4s;
      gr_u32x4 r;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const char* p = vt0 + (va ^ (db * 64)) + (16 * x + 4 * h) * (D * 2);
        const v4s v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(__attribute__((address_space(3))) char*)(char*)p);
        const gr_u32x2 w = __builtin_bit_cast(gr_u32x2, v);
        r[2 * h] = w[0];
        r[2 * h + 1] = w[1];
      }
      return gr_as<vec8>(r);
    };
    gr_f32x16 s[KB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) s[kb] = (gr_f32x16)(0.f);
#pragma unroll
    for (int ds = 0; ds < DS; ++ds)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        s[kb] = MF::mma32(gr_as<vec8>(gr_ld16(ks0 + (ka ^ (ds * 32)) + kb * 32 * (D * 2))), qf[ds], s[kb]);
      }
    bool fresh = m == -GR_INF;                                // no base yet, and a key to take it from
    if constexpr (MASKED) {
      // element r of key block kb is key k0 + 32 kb + 16 (r / 8) + 8 g + r % 8
      const int delta = limit - k0 - 8 * g;
      bool sees = false;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const int d = (bad >> (2 * kb + hf)) & 1 ? -1 : delta - 32 * kb - 16 * hf;
          sees |= d >= 0;
#pragma unroll
          for (int e = 0; e < 8; ++e) s[kb][8 * hf + e] = e <= d ? s[kb][8 * hf + e] : -GR_INF;
        }
      fresh &= sees;
    }
    vec8 pt[2 * KB];
    float lt;
    auto make_p = [&]() {
      // (kept over the tiles for fp16 alone: without the shift it costs more than it
      // saves, 4,096 tokens onto 4,096, 16 heads of 64 in bf16 152 us to 158)
      const float nmc = HALF ? base : m == -GR_INF ? 0.f : -m * c;
      lt = 0.f;
#pragma unroll
      for (int x = 0; x < 2 * KB; ++x) {
        gr_u32x4 pw;
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const float p0 = gr_exp2(fmaf(s[x >> 1][8 * (x & 1) + e], c, nmc));
          const float p1 = gr_exp2(fmaf(s[x >> 1][8 * (x & 1) + e + 1], c, nmc));
          const vec2 pp = __builtin_convertvector((gr_f32x2){p0, p1}, vec2);
          lt = MF::sum2(pp, lt);
          pw[e >> 1] = __builtin_bit_cast(unsigned, pp);
        }
        pt[x] = gr_as<vec8>(pw);
      }
    };
    make_p();
    if (gr_any(fresh || !(lt <= GR_FLASH_SUM_MAX))) {
      float mt = -GR_INF;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) mt = fmaxf(mt, s[kb][r]);
      mt = fmaxf(mt, gr_xor32(mt));
      const float mn = fmaxf(m, mt);
      const float alpha = mn > m ? gr_exp2((m - mn) * c) : 1.f;   // m = -inf -> 0
      l *= alpha;
#pragma unroll
      for (int db = 0; db < DB; ++db) o[db] *= alpha;
      m = mn;
      if (HALF) base = m == -GR_INF ? shift : fmaf(-m, c, shift);
      make_p();
    }
    l += lt;
    if constexpr (MASKED) {
      // keys with a value that is not finite (exponent bits all ones), a bit each
      constexpr unsigned EXP = gr_is_same<T, _Float16>::value ? 0x7c007c00u : 0x7f807f80u;
      constexpr unsigned ONE = gr_is_same<T, _Float16>::value ? 0x04000400u : 0x00800080u;
      unsigned long long odd = 0;
#pragma unroll 1
      for (int x = 0; x < 2 * KB; ++x) {
        gr_u32x4 f = (gr_u32x4)(0u);
#pragma unroll
        for (int db = 0; db < DB; ++db) f |= (gr_raw(vfrag(x, db)) & EXP) + ONE;
        f &= 0x80008000u;
        if (gr_any((f[0] | f[1] | f[2] | f[3]) != 0)) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            // lanes 0-31 hold key e of the 16, lanes 32-63 key 8 + e
            const unsigned long long who = __builtin_amdgcn_ballot_w64((f[e >> 1] >> ((e & 1) ? 31 : 15)) & 1);
            odd |= ((unsigned long long)((unsigned)who != 0) | (unsigned long long)((who >> 32) != 0) << 8) << (16 * x + e);
          }
        }
      }
      if (__builtin_expect(odd != 0, 0)) {
#pragma unroll 1
        for (int x = 0; x < 2 * KB; ++x) {
          gr_u32x4 p = gr_raw(pt[0]);
#pragma unroll
          for (int y = 1; y < 2 * KB; ++y) p = x == y ? gr_raw(pt[y]) : p;
          const unsigned byte = (unsigned)(odd >> (16 * x + 8 * g)) & 0xffu;
          gr_u32x4 keep;                                       // halfwords of the keys that stay in the product
#pragma unroll
          for (int e = 0; e < 4; ++e)
            keep[e] = ((byte >> (2 * e)) & 1 ? 0u : 0x0000ffffu) | ((byte >> (2 * e + 1)) & 1 ? 0u : 0xffff0000u);
#pragma unroll
          for (int db = 0; db < DB; ++db)
            o[db] = MF::mma32(gr_as<vec8>(gr_raw(vfrag(x, db)) & keep), gr_as<vec8>(p), o[db]);
#pragma unroll 1
          for (unsigned left = (unsigned)(odd >> (16 * x)) & 0xffffu; left; left &= left - 1) {
            const int i = __builtin_ctz(left), key = 16 * x + i;   // key i of the 16: half i / 8, element i % 8
            const unsigned w = (i & 6) == 0 ? p[0] : (i & 6) == 2 ? p[1] : (i & 6) == 4 ? p[2] : p[3];
            const unsigned short hw = (unsigned short)((i & 1) ? w >> 16 : w & 0xffffu);
            const float mine = g == (i >> 3) ? (float)__builtin_bit_cast(T, hw) : 0.f;
            const float pv = mine + gr_xor32(mine);
            const bool vis = k0 + key <= limit && !(bad >> x & 1);
            const char* const vr = vt0 + slot * L::TILE + key * (D * 2);
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
              for (int r = 0; r < 16; ++r) {
                const int d = db * 32 + 8 * (r >> 2) + 4 * g + (r & 3);
                const float v = (float)*reinterpret_cast<const T*>(vr + gr_swz_tr<CPR>(key, d >> 3) * 16 + (d & 7) * 2);
                if (vis) o[db][r] = fmaf(pv, v, o[db][r]);
                if ((r & 3) == 3) __builtin_amdgcn_sched_barrier(0);   // (all reads at once would spill)
              }
          }
        }
        return;
      }
    }
#pragma unroll
    for (int x = 0; x < 2 * KB; ++x)
#pragma unroll
      for (int db = 0; db < DB; ++db) o[db] = MF::mma32(vfrag(x, db), pt[x], o[db]);
  };

  // Iteration j reads slot j % NS; the tiles up to j + NS - 1 are on their way to
  // the others. A part-filled tile's zeros are LDS stores.
  // the page ids first, then this lane's Q row (8 consecutive dims of every 16)
  const int first_id = ntile > 0 ? id_of(0) : 0;
  {
    const T* qp = static_cast<const T*>(a.q) + t.b * a.q_sb + (long long)(t.first + token) * a.q_st + head * a.q_sh;
#pragma unroll
    for (int ds = 0; ds < DS; ++ds) qf[ds] = gr_as<vec8>(gr_ld16(qp + ds * 16 + 8 * g));
  }
  if (ntile > 0) refill(0, first_id);
  // Q has landed (beside the page ids) before the first tile is asked for: its
  // registers taken here, the compiler waits for them here, and not again for
  // every load in flight at each tile's first product, as it cannot see through
  // the loop's back edge that they came
#pragma unroll
  for (int ds = 0; ds < DS; ++ds) asm volatile("" : "+v"(qf[ds]));
  // Leading tiles of the group that end before key `end`.
  auto tiles_before = [&](int end) { return end - key0 < (kg + 1) * BN ? 0 : ((end - key0) / BN - kg + KG - 1) / KG; };
  const int nwhole = gr_imin(ntile, tiles_before(key1));
  // Tiles are asked for in order. Up to `plain` they are whole and their pages
  // are in the window and exist; the next one is looked at closer.
  int asked = 0, to = 0, plain = 0;           // (to: the next one's slot)
  unsigned long long bads = 0;                // bad blocks of the last tiles asked for, newest first
  // A tile that is part-filled or has a bad page issues fewer loads than 2 PER:
  // from the first such one on, every load is waited for.
  bool uneven = false;
  auto ask = [&]() {
    if (asked < plain) {
      load(asked, to, gr_ic<1>{}, 0u);
      bads <<= BLOCKS;
    } else {
      if (asked >= ntile) return;
      if (asked > 0 && (asked & (WIN - 1)) == 0) refill(asked, id_of(asked));
      const unsigned bad = (unsigned)(badwin >> ((asked & (WIN - 1)) * BLOCKS)) & ((1u << BLOCKS) - 1);
      bads = bads << BLOCKS | bad;
      if (bad == 0 && asked < nwhole) {
        load(asked, to, gr_ic<1>{}, 0u);
      } else {
        load(asked, to, gr_ic<0>{}, bad);
        uneven = true;
      }
      plain = badwin == 0 ? gr_imin(nwhole, (asked & ~(WIN - 1)) + WIN) : 0;
    }
    ++asked;
    to = to + 1 == NS ? 0 : to + 1;
  };
  // Waits for all but the tiles behind tile j (a barrier's waves wait before they ask on).
  constexpr int AHEAD = SOLO ? NS - 1 : NS - 2;
  auto arrived = [&](int j) {
    const int behind = uneven ? 0 : asked - 1 - j;
    if (AHEAD >= 2 && behind >= 2) gr_wait_vmcnt<(AHEAD >= 2 ? 4 * PER : 0)>();
    else if (AHEAD >= 1 && behind >= 1) gr_wait_vmcnt<2 * PER>();
    else gr_wait_vmcnt<0>();
    asm volatile("" ::: "memory");
  };
  static_assert(NS <= 3 && 2 * (NS - 1) * PER < 64 && NS * BLOCKS <= 64, "load counters");
  auto barrier = [&] { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
  int j = 0, slot = 0;
#pragma unroll
  for (int i = 0; i < NS - 1; ++i) ask();
  auto enter = [&](int j) {
    if constexpr (SOLO) {
      // the slot's last reads are over (no other wave reads it)
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      ask();
      arrived(j);
    } else {
      arrived(j);
      barrier();                                               // tile j is there, and its predecessor's slot free
      ask();
    }
  };
  auto bad_at = [&](int j) { return (unsigned)(bads >> ((asked - 1 - j) * BLOCKS)) & ((1u << BLOCKS) - 1); };
  // Tiles that every row of the wave sees in full, then the others (they end a
  // row's keys): two loops, for a join of both kinds in one made the compiler
  // copy the accumulators in every tile. The iterations' barriers are alike.
  const int nclean = wave_live ? gr_imin(nwhole, tiles_before(lim_lo + 1)) : 0;
#pragma unroll 1
  for (; j < nclean && !uneven; ++j) {
    enter(j);
    tile(j, slot, 0u, gr_ic<0>{});
    slot = slot + 1 == NS ? 0 : slot + 1;
  }
#pragma unroll 1
  for (; j < niter; ++j) {
    enter(j);
    if (wave_live && j < ntile && key_of(j) <= lim_hi) tile(j, slot, bad_at(j), gr_ic<1>{});
    slot = slot + 1 == NS ? 0 : slot + 1;
  }

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
    const float to = mx == -GR_INF ? 0.f : mx;
    const float w0 = gr_exp2((m - to) * c);
    l *= w0;
#pragma unroll
    for (int db = 0; db < DB; ++db) o[db] *= w0;
    m = mx;
#pragma unroll
    for (int k = 1; k < KG; ++k) {
      const float wk = gr_exp2((ml[k][0] - to) * c);
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
  if (place >= 0) {
    // unnormalised O and (base, row sum) of these keys
    const long long at = (long long)place * BM + wave * 32 + l32;
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
      a.lse[trow * a.Hq + head] = lt == 0.f ? -GR_INF : (m * c + (__builtin_amdgcn_logf(lt) - shift)) * 0.6931471805599453f;
    }
  }
}

// Tiles of BM rows: NW waves by row, KG groups by key, BN keys a step, NS steps in
// LDS. KGS > 0: sequences of at most 32 rows (single tokens in a
// batch with long chunks) take tiles of 32, KGS waves sharing out the keys, 32 a step.
template <class T, int D, int BN, int NW, int KG, int NS, int KGS, bool SHARED>
__device__ __forceinline__ void gr_paged_body(const gr_paged_args& a, char* lds) {
  constexpr int BM = 32 * NW, WAVES = NW * KG;
  const int lane = threadIdx.x & 63;
  const int logical = gr_xcd_remap_any((int)blockIdx.x, (int)gridDim.x);
  gr_paged_tile t;
  gr_paged_seqs<BM, (KGS > 0)> seqs;
  auto segment = [&](int hk, int key0, int key1, int place) {
    if constexpr (KGS > 0) {
      if (t.nrows <= 32) return gr_paged_segment<T, D, 32, 1, KGS, 2, WAVES, BM>(a, lds, t, hk, key0, key1, place);
    }
    gr_paged_segment<T, D, BN, NW, KG, NS, WAVES, BM>(a, lds, t, hk, key0, key1, place);
  };
  if constexpr (!SHARED) {
    // key head slowest, then the tiles: workgroups of one key head share an XCD's L2
    int at = logical, per = a.tiles;          // tile of all heads' and their tiles
    if constexpr (KGS > 0 && D == 64) {
      // in packed batches the tiles of long chunks of all key heads first, so that
      // they spread over the CUs and single tokens fill up: two chunks of 423 and 17
      // tokens, 16 heads 45.7 us to 37.6, three of 800 and 29 77.3 to 68.9, but two of
      // 400 with short contexts and 18 33 to 36 (D 128: 43.9 to 47.4, 124.9 to 131.9)
      if (a.starts) {
        seqs.only = 1;
        const int large = gr_imin(seqs.count(a, lane), a.tiles), first = large * a.Hkv;
        if ((int)blockIdx.x < first) {
          at = gr_xcd_remap_any((int)blockIdx.x, first);
          per = large;
        } else {
          at = gr_xcd_remap_any((int)blockIdx.x - first, (int)gridDim.x - first);
          per = a.tiles - large;
          seqs.only = 2;
          seqs.b0 = -1;
        }
      }
    }
    const int hk = at / per;
    if (seqs.template find<false>(a, at - hk * per, lane, t)) segment(hk, 0, t.kend, -1);
  } else {
    const int per_head = seqs.total(a, lane);
    const gr_paged_cut cut(per_head * a.Hkv, a.shares);
    if (logical >= cut.W) return;
    const int end = cut.begin(logical + 1);
    int place = 2 * logical;
#pragma unroll 1
    for (int x = cut.begin(logical); x < end;) {
      const int hk = x / per_head;
      if (!seqs.template find<true>(a, x - hk * per_head, lane, t)) return;
      const int left = gr_imin(end - x, t.nb + GR_PAGED_COST - t.block);
      const int to = gr_imin(t.block + left, t.nb);
      if (t.block < to) {
        segment(hk, t.block * 64, gr_imin(t.kend, to * 64), to - t.block == t.nb ? -1 : place);
        if (x + left < end) __syncthreads();                  // the rings are free again
      }
      x += left;
      place = 2 * logical + 1;
    }
  }
}

// Merges the parts of a tile's rows: O = sum_p w_p O_p / sum_p w_p l_p with w_p =
// 2^((m_p - max m) c), in an order that the cut alone decides. D / 4 lanes hold a
// part's row. Up to two parts for each row of the tile: every such group of lanes
// has a row of its own and asks for 8 of its parts at once. More (few rows, long
// contexts): the four waves share a row, 256 / D parts a wave at a time, UN such
// loads ahead.
constexpr int GR_PAGED_MAX_SHARES = 512;

template <class T, int D, int BM, bool SMALL>
__device__ __forceinline__ void gr_paged_merge_body(const gr_paged_args& a) {
  constexpr int LPR = D / 4, PPW = 64 / LPR;  // lanes of a row, rows of a wave's load
  constexpr int FEW = 8, UN = 4, NW = 4;
  __shared__ float xm[NW][D];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int hk = blockIdx.x / a.tiles;
  gr_paged_tile t;
  gr_paged_seqs<BM, SMALL> seqs;
  const int per_head = seqs.total(a, lane);
  if (!seqs.template find<false>(a, (int)blockIdx.x - hk * a.tiles, lane, t)) return;
  // the shares that cover the tile's blocks; only the first may have begun in
  // another tile, and then left this one's part in its second place
  const gr_paged_cut cut(per_head * a.Hkv, a.shares);
  const int x0 = hk * per_head + t.x0;
  const int w0 = cut.of(x0), np = cut.of(x0 + t.nb - 1) + 1 - w0;
  if (np <= 1) return;
  const int skew = cut.begin(w0) < x0 ? 1 : 0;
  auto slot = [&](int p, int r) { return (long long)(2 * (w0 + p) + (p == 0 ? skew : 0)) * BM + r; };
  const float c = a.scale_log2, shift = gr_paged_shift<T>(t.keys);
  const int rows = gr_imin(BM, t.nrows - t.row0);
  const int sub = lane / LPR, d4 = (lane % LPR) * 4;
  auto put = [&](int r, gr_f32x4 o, float l, float mx) {
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    const int token = (t.row0 + r) / a.G, head = hk * a.G + (t.row0 + r) % a.G;
    T* const op = static_cast<T*>(a.o) + t.b * a.o_sb + (long long)(t.first + token) * a.o_st + head * a.o_sh + d4;
    *reinterpret_cast<gr_u32x2*>(op) = (gr_u32x2){gr_pack2f<T>(o[0] * inv, o[1] * inv), gr_pack2f<T>(o[2] * inv, o[3] * inv)};
    if (a.lse && d4 == 0) {
      const long long trow = a.starts ? t.first + token : (long long)t.b * a.rows + token;
      a.lse[trow * a.Hq + head] = l == 0.f ? -GR_INF : (mx * c + (__builtin_amdgcn_logf(l) - shift)) * 0.6931471805599453f;
    }
  };
  if (np <= 2 * rows) {
    for (int r0 = ((int)blockIdx.y * NW + wave) * PPW; r0 < rows; r0 += (int)gridDim.y * NW * PPW) {
      const int r = gr_imin(r0 + sub, rows - 1);
      float mx = -GR_INF, l = 0.f;
      gr_f32x4 o = {0.f, 0.f, 0.f, 0.f};
      for (int p0 = 0; p0 < np; p0 += FEW) {
        gr_f32x2 ml[FEW];
        gr_f32x4 x[FEW];
#pragma unroll
        for (int p = 0; p < FEW; ++p)
          if (p0 + p < np) {
            ml[p] = *reinterpret_cast<const gr_f32x2*>(a.part_ml + slot(p0 + p, r) * 2);
            x[p] = *reinterpret_cast<const gr_f32x4*>(a.part_o + slot(p0 + p, r) * D + d4);
          }
        float mn = mx;
#pragma unroll
        for (int p = 0; p < FEW; ++p)
          if (p0 + p < np) mn = fmaxf(mn, ml[p][0]);
        const float base = mn == -GR_INF ? 0.f : mn;
        const float old = gr_exp2((mx - base) * c);       // 0 before the first part
        mx = mn;
        l *= old;
        o *= old;
#pragma unroll
        for (int p = 0; p < FEW; ++p)
          if (p0 + p < np) {
            const float w = gr_exp2((ml[p][0] - base) * c);
            l = fmaf(w, ml[p][1], l);
            o += w * x[p];
          }
      }
      if (r0 + sub < rows) put(r, o, l, mx);
    }
    return;
  }
  for (int r = (int)blockIdx.y; r < rows; r += (int)gridDim.y) {
    // part lane + 64 i: base and sum
    float m[GR_PAGED_MAX_SHARES / 64], w[GR_PAGED_MAX_SHARES / 64];
    float mx = -GR_INF, l = 0.f;
#pragma unroll
    for (int i = 0; i < GR_PAGED_MAX_SHARES / 64; ++i) {
      const int p = lane + 64 * i;
      m[i] = -GR_INF;
      w[i] = 0.f;
      if (p < np) {
        const gr_f32x2 ml = *reinterpret_cast<const gr_f32x2*>(a.part_ml + slot(p, r) * 2);
        m[i] = ml[0];
        w[i] = ml[1];
      }
      mx = fmaxf(mx, m[i]);
    }
    mx = gr_wave_max(mx);
    const float base = mx == -GR_INF ? 0.f : mx;
#pragma unroll
    for (int i = 0; i < GR_PAGED_MAX_SHARES / 64; ++i) {
      const float sum = w[i];
      w[i] = gr_exp2((m[i] - base) * c);
      l = fmaf(w[i], sum, l);
    }
    l = gr_wave_sum(l);
    gr_f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < GR_PAGED_MAX_SHARES / 64; ++i) {   // (w is indexed by constants)
      if (64 * i >= np) break;
      const int end = gr_imin(np - 64 * i, 64);
      for (int p0 = wave * PPW * UN; p0 < end; p0 += NW * PPW * UN) {
        gr_f32x4 x[UN];
#pragma unroll
        for (int k = 0; k < UN; ++k) {
          const int p = gr_imin(p0 + k * PPW + sub, end - 1);
          x[k] = *reinterpret_cast<const gr_f32x4*>(a.part_o + slot(64 * i + p, r) * D + d4);
        }
#pragma unroll
        for (int k = 0; k < UN; ++k) {
          const int p = p0 + k * PPW + sub;
          const float f = __shfl(w[i], p & 63, 64);
          if (p < end) o += f * x[k];
        }
      }
    }
#pragma unroll
    for (int off = LPR; off < 64; off <<= 1)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], off, 64);
    if (sub == 0) *reinterpret_cast<gr_f32x4*>(&xm[wave][d4]) = o;
    __syncthreads();
    if (wave == 0 && sub == 0) {
#pragma unroll
      for (int k = 1; k < NW; ++k) o += *reinterpret_cast<const gr_f32x4*>(&xm[k][d4]);
      put(r, o, l, mx);
    }
    __syncthreads();
  }
}
