/* grammar_rt.h -- C ABI of libgrammar_rt.so, the MI355X (gfx950) runtime of
 * the kernel-grammar descent.
 *
 * The reference has no native library: its generated modules are cuTile
 * Python, JIT-compiled by cuda.tile and launched/timed through cupy. Every
 * entry point below replaces one piece of that Python/vendor boundary; the
 * comment on each names the reference site it stands in for.
 *
 * Conventions
 *  - Plain C types only. Device buffers are raw pointers owned by the caller
 *    (PyTorch-ROCm tensors in the Python layer); the library never frees them.
 *  - Every function returns 0 on success or a negative GR_E* code; the
 *    message of the last failure on the calling thread is gr_last_error().
 *  - `stream` is a hipStream_t passed as void* (NULL = the null stream).
 */
#ifndef GRAMMAR_RT_H
#define GRAMMAR_RT_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- status codes ------------------------------------------------------ */
#define GR_OK 0
#define GR_E_ARG -1       /* invalid argument / unsupported shape */
#define GR_E_COMPILE -2   /* hiprtc compilation failed */
#define GR_E_LOAD -3      /* code object could not be loaded */
#define GR_E_LAUNCH -4    /* kernel launch failed */
#define GR_E_RUNTIME -5   /* any other HIP runtime error */

/* ---- element types ----------------------------------------------------- */
#define GR_F32 0
#define GR_F16 1
#define GR_BF16 2

/* Message describing the last failure on this thread ("" if none). */
const char* gr_last_error(void);

/* Library / toolchain identification, e.g. "gfx950 hiprtc 7.2". The string is
 * part of every on-disk code-object cache key. */
const char* gr_version(void);

/* ---- device properties -------------------------------------------------- */
/* Fills: [0] CU count, [1] max LDS bytes per workgroup, [2] wavefront size,
 * [3] peak engine clock kHz, [4] L2 bytes. For the roofline constants. */
int gr_device_info(int device, long long* out5);

/* ---- compilation (replaces the cuTile JIT: grammar/optimization.py:262-283,
 *      grammar/kernel_ast.py:1228-1229) ------------------------------------ */

/* Compile HIP C++ source `src` with hiprtc for gfx950. Options are passed
 * through (include paths, -D...). On success *code and *code_size receive a
 * malloc'd code object (free with gr_free_code). On a compile error the hiprtc
 * log is copied to `log` (truncated to loglen) and GR_E_COMPILE is returned.
 * Thread-safe: independent programs may be compiled concurrently. No HIP
 * device context is touched. */
int gr_compile(const char* src, const char* name, const char* const* opts, int nopts,
               void** code, size_t* code_size, char* log, size_t loglen);
void gr_free_code(void* code);

typedef struct gr_module gr_module;
typedef struct gr_kernel gr_kernel;

/* Load a code object (from gr_compile or the on-disk cache). */
int gr_module_load(const void* code, size_t code_size, gr_module** out);
void gr_module_free(gr_module* mod);
/* Look up an extern "C" __global__ function by name. The handle lives as long
 * as its module. */
int gr_get_kernel(gr_module* mod, const char* name, gr_kernel** out);

/* ---- launch (replaces ct.launch: grammar/kernel_ast.py:1273-1275) -------- */

/* Launch with every kernel parameter a 64-bit value (device pointers; the
 * renderer bakes every shape into the source). */
int gr_launch(gr_kernel* k, const uint32_t grid[3], const uint32_t block[3], uint32_t lds_bytes,
              void* stream, const uint64_t* args, int nargs);

/* A launch plan: the ordered stage launches of one generated module with
 * their arguments bound (the reference's host fn(*inputs),
 * grammar/kernel_ast.py:1267-1278, minus its per-call cp.zeros allocations:
 * intermediates are allocated once by the caller). */
typedef struct gr_plan gr_plan;
int gr_plan_create(int nsteps, gr_plan** out);
int gr_plan_set_step(gr_plan* p, int i, gr_kernel* k, const uint32_t grid[3], const uint32_t block[3],
                     uint32_t lds_bytes, const uint64_t* args, int nargs);
int gr_plan_run(gr_plan* p, void* stream);
/* gr_plan_run with the arguments of this call, the steps' one after another
 * (nargs = the sum of their counts), instead of the bound ones. The plan is
 * only read: threads may run one plan at the same time. */
int gr_plan_run_args(gr_plan* p, void* stream, const uint64_t* args, int nargs);
void gr_plan_free(gr_plan* p);

/* ---- timing (replaces cp.cuda.Event timing: grammar/optimization.py:284-300,
 *      bench.py:49-74) ------------------------------------------------------ */
#define GR_TIME_BATCH 0   /* one event pair around `iters` back-to-back runs; mean ms */
#define GR_TIME_MIN 1     /* one event pair per run; minimum ms over `iters` */
/* Each event pair is preceded by a short bounded device spin (about 28 us)
 * that holds the stream while the host enqueues the timed launches, so the
 * time is the GPU's, without the host's launch latency. */
int gr_plan_time(gr_plan* p, void* stream, int warmup, int iters, int mode, float* ms_out);

/* ---- hand-written CDNA4 baselines -------------------------------------- */

/* Flash-style attention forward, O = softmax(scale*Q K^T [causal]) V.
 * Replaces the attention module contract fn(KT, Q, V) (bench.py:14-20,
 * pytorch-naive.py:23-65, grammar/kernel_ast.py:1267-1287) and the SDPA
 * reference point (flash-attn2-sota.py:41-62).
 *  dtype: GR_F16 or GR_BF16 (fp32 accumulate). With GR_F16 the kernel
 *  rounds Q * scale * log2(e) to fp16 once (the scores then need no per-score
 *  scaling); that cannot overflow when scale * log2(e) <= 1 (as for the
 *  default 1/sqrt(D) with D >= 3). A larger fp16 scale (e.g. 1 for a
 *  pre-scaled q) takes kernels that keep Q as given and scale every score,
 *  on one tile only: block_m 64, block_n 32 (0 / 0 pick it; N a multiple of
 *  64). bf16 always keeps Q as given. GR_F32 (the reference's own dtype, fp32
 *  throughout on the fp32 matrix cores): non-causal only, N a multiple of 32,
 *  block_m and block_n ignored (a workgroup owns 32 queries and splits its
 *  keys over its waves); not for gr_attn_fwd_train. When B * H * N / 32 query
 *  blocks would leave CUs idle, the keys of a query block are also split over
 *  2, 4 or 8 workgroups (the library picks by D, N, the query blocks and the
 *  CU count) and a second launch merges their partials, which sit in a
 *  workspace the library allocates once per (device, stream) and keeps until
 *  the process ends: 8.5 MB, for a split launch has at most 256 workgroups of
 *  32 queries (4.3 MB), and the splits below have memory of their own. On the
 *  per-thread default stream each host thread has its own. Without memory for
 *  it the call runs unsplit. Under capture only N a multiple of 256 with at
 *  most 128 query blocks is split, over the most of 8, 4 or 2 workgroups that
 *  divide N / 128; call once on a stream before capturing such calls into a
 *  graph, and order its replays on other streams with calls of such splits.
 *  Q, V, O: [B, H, N, D] with strides {batch, head, seq} in elements
 *  (unit stride along D). K: [B, H, N, D] if k_transposed == 0, else KT
 *  [B, H, D, N] whose k_strides = {batch, head, d} (unit stride along N).
 *  D in {64, 128}; N a multiple of block_m and block_n.
 *  block_m: queries per workgroup, 64 / 128 / 256 (one wave per 32 queries;
 *  129 / 257: 128 / 256 with the software-pipelined schedule), 0 = the
 *  largest of 256 / 128 / 64 dividing N. block_n: keys per tile, 32 / 64 /
 *  128 (128 at D = 64 only), 0 = 128 at D = 64 when it divides N, else 64
 *  or 32, but 64 where the two-wave body below applies at block_m 256.
 *  Both 0 (N a multiple of 64): the library picks by B * H, N and the CU count
 *  among those tiles, part-filled last query tiles included, and workgroups of
 *  32 to 128 queries that split the keys over 2 to 8 groups of waves, for
 *  grids that would leave CUs idle; N then need not divide the query tile.
 *  fp16 at D = 64, non-causal, 256 x 64 and N a multiple of 256 runs
 *  the kernel with two waves per SIMD and a hand-ordered main loop (160 KiB
 *  of LDS); so does fp16 or bf16 at D = 128 with K transposed, causal or not,
 *  at 256 x 64 and N a multiple of 256 (D = 128 is the default tile there).
 *  Causal grids run each XCD's query blocks longest-first. */
int gr_attn_fwd(const void* q, const void* k, const void* v, void* o, int dtype, int B, int H,
                int N, int D, const long long* q_strides, const long long* k_strides,
                const long long* v_strides, const long long* o_strides, int k_transposed,
                int causal, float scale, int block_m, int block_n, void* stream);

/* The workgroup that gr_attn_fwd (train != 0: gr_attn_fwd_train) picks for
 * block_m = block_n = 0 at scale log2(e) <= 1: out3 = {queries, key groups, keys
 * per tile}. GR_F16 or GR_BF16, N a multiple of 64. A 256-query pick that divides
 * N runs the named default tile. Host arithmetic on the current device's CU count
 * (256 without a device). No counterpart in the reference. */
int gr_attn_fwd_shape(int dtype, int B, int H, int N, int D, int k_transposed, int causal, int train, int* out3);

/* Training forward: gr_attn_fwd that also writes, per query row, the
 * log-sum-exp of the scaled (masked) scores, natural log, into lse
 * [B*H][N] fp32 (4-byte aligned) for gr_attn_bwd. No counterpart in the
 * reference (forward only); the scope's next-step backward pass. */
int gr_attn_fwd_train(const void* q, const void* k, const void* v, void* o, float* lse, int dtype, int B,
                      int H, int N, int D, const long long* q_strides, const long long* k_strides,
                      const long long* v_strides, const long long* o_strides, int k_transposed, int causal,
                      float scale, int block_m, int block_n, void* stream);

/* Attention backward: dQ, dK, dV of sum(O * dO) for O = softmax(scale Q K^T
 * [causal]) V, from Q, K, V, O, dO and the forward's lse. No counterpart in
 * the reference (forward only); the scope's next-step backward pass.
 *  All nine [B, H, N, D] tensors share `strides` {batch, head, seq} (in
 *  elements, multiples of 8; unit stride along D) and are 16-byte aligned.
 *  D in {64, 128}; N a multiple of 128.
 *  workspace: device memory of gr_attn_bwd_workspace(B, H, N, D) bytes,
 *  16-byte aligned (per-row statistics; the call overwrites it). */
size_t gr_attn_bwd_workspace(int B, int H, int N, int D);
int gr_attn_bwd(const void* q, const void* k, const void* v, const void* o, const void* dout, const float* lse,
                void* dq, void* dk, void* dv, int dtype, int B, int H, int N, int D, const long long* strides,
                int causal, float scale, void* workspace, size_t workspace_bytes, void* stream);

/* Decode-shape attention forward: Nq queries (any count, e.g. 1 for a
 * decode step) against N keys, O = softmax(scale*Q K^T) V, non-causal.
 * No counterpart in the reference, whose attention takes Nq == N
 * (run_attention_search.py:34-114); it is the decode-shape item of the
 * scope's next steps and serves small B*H*Nq, where the query tiles alone
 * cannot fill the GPU.
 *  Q, O: [B, H, Nq, D]; K, V: [B, H, N, D]; strides {batch, head, seq} in
 *  elements (multiples of 8), unit stride along D. N a multiple of 32; D in
 *  {64, 128}; dtype GR_F16 or GR_BF16.
 *  Up to 4 queries run on a streaming kernel (K and V read once straight
 *  into registers, scores on the VALU); more on the flash body's MFMA tiles,
 *  up to 64 of them with four key groups inside the workgroup. With GR_F16,
 *  more than 4 queries and scale * log2(e) > 1, Q is kept as given (as by
 *  gr_attn_fwd) and a workgroup is one wave of 32 queries without groups.
 *  splits: workgroups per head (up to 4 queries) or per query tile that
 *  share out the keys (clamped to N/32, or to the number of 64- or 32-key
 *  tiles); with more than one, the partials go
 *  through `workspace` (device memory of at least
 *  gr_attn_decode_workspace(B, H, Nq, D, splits) bytes, 16-byte aligned;
 *  the call then overwrites it) and a second kernel merges them. */
size_t gr_attn_decode_workspace(int B, int H, int Nq, int D, int splits);
int gr_attn_decode(const void* q, const void* k, const void* v, void* o, int dtype, int B, int H, int Nq,
                   int N, int D, const long long* q_strides, const long long* k_strides,
                   const long long* v_strides, const long long* o_strides, float scale, int splits,
                   void* workspace, size_t workspace_bytes, void* stream);

/* gr_attn_decode without any allocation: no counterpart in the reference.
 * For callers that cannot allocate device memory -- code under HIP graph
 * capture, tight serving loops, harnesses that forbid hipMalloc. Same
 * arguments and results as gr_attn_decode minus the workspace: the key-split
 * partials go to a scratch array inside the library, GR_DECODE_SCRATCH_BYTES
 * (16 MiB) per device, held by each device the library runs on until the
 * process ends. A call whose key split needs more than that
 * (gr_attn_decode_workspace(B, H, Nq, D, splits) after the split is clamped)
 * fails with GR_E_ARG before launching anything. Nothing in the array needs
 * to start at zero: every part overwrites its rows before the merge reads
 * them. All calls on one device share its array, so calls that overlap in
 * time on one device (different streams, threads) race: serialise them. */
#define GR_DECODE_SCRATCH_BYTES (16u << 20)
int gr_attn_decode_noalloc(const void* q, const void* k, const void* v, void* o, int dtype, int B, int H, int Nq,
                           int N, int D, const long long* q_strides, const long long* k_strides,
                           const long long* v_strides, const long long* o_strides, float scale, int splits,
                           void* stream);

/* ---- positions and paged caches ------------------------------------------ */

/* The rotation of queries and keys by position. No counterpart in the reference,
 * whose attention has no positions. Pair j of a head, (x1, x2), becomes
 * (x1 cos t - x2 sin t, x1 sin t + x2 cos t), t = position x (frequency of j).
 *  turns: device array, per pair the frequency in units of 2^-64 turns a
 *         position (radians / 2 pi, modulo one turn); 8-byte aligned.
 *  axes:  device array, per pair the position axis it turns with; 8-byte
 *         aligned; not read with naxes 1. naxes: 1 to 8.
 *  pairs: a multiple of 8, at most head_dim / 2; the first 2 pairs elements of a
 *         head are rotated, the others pass. head_dim: a multiple of 16 up to 256.
 *  interleaved: pair j is elements 2j and 2j + 1, else j and j + pairs. */
typedef struct gr_rotary_spec {
  const uint64_t* turns;
  const uint8_t* axes;
  int pairs, naxes, head_dim, interleaved;
} gr_rotary_spec;

/* Rotates q [B, Hq, N, D] into q_out and, if k is not NULL, k [B, Hk, N, D] into
 * k_out (each may be its own input, by the same strides: the call then works in
 * place; outputs share no other memory with inputs or each other).
 *  Strides {batch, token, head} in elements, non-negative multiples of 8, unit
 *  stride along D; base pointers 16-byte aligned. dtype GR_F16, GR_BF16 (angles,
 *  products and sums in fp32, rounded once) or GR_F32.
 *  positions: int32, any sign; position_strides = {axis, batch, token}.
 *  inverse != 0 rotates by -t, which is also the gradient's way back. */
int gr_rotary(const gr_rotary_spec* rotary, const void* q, void* q_out, int Hq, const long long* q_strides,
              const long long* q_out_strides, const void* k, void* k_out, int Hk, const long long* k_strides,
              const long long* k_out_strides, int dtype, int B, int N, const int* positions,
              const long long* position_strides, int inverse, void* stream);

/* A norm of query and key heads: a row x of D elements becomes w x / sqrt(mean
 * x^2 + eps), w its D weights. q_weight, k_weight: device arrays, 16-byte aligned, of
 * dtype GR_F32 or the rows' type; NULL: ones. eps: not negative (with 0 a row of zeros
 * is NaN, and rows are normed from magnitudes of 2^-60 on). No counterpart in the
 * reference. */
typedef struct gr_head_norm {
  const void* q_weight;
  const void* k_weight;
  int dtype;
  float eps;
} gr_head_norm;

/* gr_rotary of normed heads, in one pass over them; arguments as there. Squares,
 * norm, weights and rotation in fp32 (magnitudes up to 2^59: 256 squares of 2^60 are no
 * fp32 number), rounded once. */
int gr_norm_rotary(const gr_rotary_spec* rotary, const gr_head_norm* norm, const void* q, void* q_out, int Hq,
                   const long long* q_strides, const long long* q_out_strides, const void* k, void* k_out, int Hk,
                   const long long* k_strides, const long long* k_out_strides, int dtype, int B, int N,
                   const int* positions, const long long* position_strides, void* stream);

/* Its gradient: from q, k as gr_norm_rotary took them and the gradients dq_out,
 * dk_out of its results, those of q and k into dq, dk (strides of dq_out, dq, dk_out and
 * dk as q's; dq may be dq_out by the same strides, outputs share no other memory with
 * the call's arrays) and those of the weights, [D] of the weights' type, into dq_weight, dk_weight
 * (NULL: not wanted). k NULL: queries alone. The weights' gradients are summed in fp32 over all
 * tokens and heads, in an order that the sizes alone decide.
 * workspace: device memory of at least gr_norm_rotary_bwd_workspace(...) bytes, 16-byte
 * aligned, not read by calls to come (calls that may overlap in time need one each); not
 * needed without dq_weight and dk_weight. */
size_t gr_norm_rotary_bwd_workspace(int Hq, int Hk, int head_dim, int B, int N);
int gr_norm_rotary_bwd(const gr_rotary_spec* rotary, const gr_head_norm* norm, const void* q, const void* dq_out, void* dq,
                       int Hq, const long long* q_strides, const long long* dq_out_strides, const long long* dq_strides,
                       const void* k, const void* dk_out, void* dk, int Hk, const long long* k_strides,
                       const long long* dk_out_strides, const long long* dk_strides, int dtype, int B, int N,
                       const int* positions, const long long* position_strides, void* dq_weight, void* dk_weight,
                       void* workspace, size_t workspace_bytes, void* stream);

/* A key/value cache in pages. No counterpart in the reference. k and v:
 * [pages][heads][page_size][head_dim] by strides {page, head, slot} in elements
 * (non-negative multiples of 8, unit stride along head_dim, the slot stride below
 * 2^26), 16-byte aligned; dtype GR_F16 or GR_BF16; head_dim 64 or 128; page_size
 * a power of two from 16 to 2^20. */
typedef struct gr_paged_cache {
  void* k;
  void* v;
  long long k_strides[3], v_strides[3];
  int dtype, pages, heads, page_size, head_dim;
} gr_paged_cache;

/* The sequences of a call; the arrays are int32 in device memory.
 *  table:  [B][width] page ids by row stride table_stride: key j of sequence b is
 *          slot j % page_size of page table[b][j / page_size].
 *  lens:   [B] keys of each sequence, the new tokens' among them: new token i
 *          of n stands at position len - n + i.
 *  starts: [B + 1] first row of each sequence's new tokens in a packed batch of
 *          `rows` tokens, rows outside of every sequence being left alone; or
 *          NULL for a uniform batch of `rows` new tokens a sequence.
 *  max_new, max_len: the most new tokens and keys of a sequence, where known (0:
 *          not). They only choose how an attention is shared out.
 * What the arrays hold is bounded on the device: a page id outside of the cache,
 * a position outside of the table or a sequence whose starts are not both in
 * the batch reads and writes nothing (such keys do not exist, such tokens are not
 * stored). Starts are to be in order: where they overlap, nothing else is touched, but
 * which of the sequences a row belongs to is not defined. */
typedef struct gr_paged_batch {
  const int* table;
  long long table_stride;
  const int* lens;
  const int* starts;
  int B, rows, width, max_new, max_len;
} gr_paged_batch;

/* Puts the new tokens' keys and values into their pages and, with a rotation
 * (NULL: none), turns the keys on the way, and the queries, if q is not NULL, from
 * q into q_out (which may be q). Strides {batch, token, head}, as gr_rotary's
 * (a packed batch's batch stride is not read). positions NULL: a token's place
 * len - n + i in its sequence, on every axis; else int32 by {axis, batch, token}
 * (packed: the token axis is the batch's). q_out shares no memory with k, v or
 * the cache, and k and v lie in no page that the call writes. A slot that two
 * tokens of one call fall on ends with either's entry or parts of both. */
int gr_paged_append(const gr_paged_cache* cache, const gr_paged_batch* batch, const gr_rotary_spec* rotary, const void* q,
                    void* q_out, int Hq, const long long* q_strides, const long long* q_out_strides, const void* k,
                    const void* v, const long long* k_strides, const long long* v_strides, const int* positions,
                    const long long* position_strides, void* stream);

/* The scales of a quantised cache. Its k and v hold bytes (e4m3: four significant
 * bits, at most 448) by strides that are multiples of 16, and its dtype is that of the
 * tokens, GR_F16 or GR_BF16. scales: bytes [pages][heads][2: key, value][page_size] by
 * strides {page, head, key to value} that are non-negative multiples of 16, unit stride
 * along the slots, 16-byte aligned, each b standing for 2^(b - 127), or NaN for 255 (E8M0). A row
 * stands for its numbers times its scale, in the tokens' type: where that has no such number
 * (below its normal range, under scales below 2^-15 in fp16 and 2^-124 in bf16, as keys that a
 * norm or a rotation made small can have) the nearest one, a whole number of its smallest steps. */
typedef struct gr_paged_scales {
  void* scales;
  long long strides[3];
} gr_paged_scales;

/* gr_paged_append of normed queries and keys (norm NULL: none) into a cache that
 * is quantised (scales NULL: it is not). A row is quantised after norm and rotation,
 * from fp32: its scale is the least power of two, 2^-127 at least, by which its
 * largest magnitude is at most 448, its numbers are rounded to nearest even. Rows
 * are clamped to 61440 (fp16) or 15 2^124 (bf16) first; a row with a value that is not finite becomes
 * NaN. Other arguments as gr_paged_append's, of which this is the general form. */
int gr_paged_append_with(const gr_paged_cache* cache, const gr_paged_scales* scales, const gr_paged_batch* batch,
                         const gr_rotary_spec* rotary, const gr_head_norm* norm, const void* q, void* q_out, int Hq,
                         const long long* q_strides, const long long* q_out_strides, const void* k, const void* v,
                         const long long* k_strides, const long long* v_strides, const int* positions,
                         const long long* position_strides, void* stream);

/* Reads the batch's sequences back as dense keys and values in the cache's dtype
 * (scales NULL: the cache is not quantised): key j of sequence b goes to token j of
 * batch b of k_out and v_out [B, rows, heads, D] or, with starts, to row starts[b] + j of
 * [rows, heads, D], by strides {batch, token, head} that are multiples of 8. `rows`
 * and `starts` of the batch count keys here, not new tokens. Rows of a sequence behind its
 * keys, and keys whose page is not in the cache, become 0; rows of no sequence are
 * left alone. k_out and v_out share no memory with each other or the cache. */
int gr_paged_read(const gr_paged_cache* cache, const gr_paged_scales* scales, const gr_paged_batch* batch, void* k_out,
                  void* v_out, const long long* k_strides, const long long* v_strides, void* stream);

/* Attention of the new tokens over the cache, O = softmax(scale Q K^T) V; token
 * i sees the keys up to its own position (causal != 0) or all of its sequence's.
 * Hq, a multiple of the cache's heads: query head h reads key head h / (Hq /
 * heads). q, o: strides {batch, token, head} as above. lse: NULL, or [tokens][Hq]
 * fp32 (uniform batches [B][rows][Hq]) for the log-sum-exp of the scaled scores,
 * natural log. A row that sees no key gets 0 and -inf. o may be q, by the same
 * strides; outputs and workspace share no other memory with the call's arrays.
 * workspace: device memory, 16-byte aligned, in which workgroups that share a
 * row's keys leave partial results; gr_paged_attn_workspace names the size for a
 * call's shapes (0 for calls that are not shared out, and for invalid ones). With
 * less the keys are shared out less, with none not at all. The call overwrites
 * it: calls that may overlap in time need one each. */
size_t gr_paged_attn_workspace(const gr_paged_cache* cache, const gr_paged_batch* batch, int Hq);
int gr_paged_attn(const gr_paged_cache* cache, const gr_paged_batch* batch, const void* q, void* o, float* lse, int Hq,
                  const long long* q_strides, const long long* o_strides, int causal, float scale, void* workspace,
                  size_t workspace_bytes, void* stream);

/* The same over a quantised cache: keys and values are taken as the numbers of
 * the tokens' type that they stand for (gr_paged_scales). The workspace has a size of its own. */
size_t gr_paged_attn_scaled_workspace(const gr_paged_cache* cache, const gr_paged_scales* scales, const gr_paged_batch* batch,
                                      int Hq);
int gr_paged_attn_scaled(const gr_paged_cache* cache, const gr_paged_scales* scales, const gr_paged_batch* batch,
                         const void* q, void* o, float* lse, int Hq, const long long* q_strides,
                         const long long* o_strides, int causal, float scale, void* workspace, size_t workspace_bytes,
                         void* stream);

/* Batched GEMM with fused epilogue, C[z] = act(alpha * A[z] @ B[z]).
 * Replaces the grammar's matmul stage (a stage whose body is matmul over a
 * contraction axis, optionally followed by mulc and relu/silu:
 * grammar/kernel_ast.py:168-223 EMIT_RULES/CONST_OPS, :826-845 accumulator
 * and K loop) as rendered for the MLP (run_mlp_search.py:42-127).
 *  dtype: GR_F16 or GR_BF16 (fp32 accumulate), or GR_F32 (fp32 throughout, on
 *  the fp32 matrix cores: tiles (block_m, block_n) in {32, 64, 128}^2, M and
 *  N multiples of the tile, K a multiple of 8, strides multiples of 4);
 *  batch: number of matrices.
 *  A: [batch][M][K], a_strides = {batch, row}; unit stride along K.
 *  B: [batch][K][N] (b_kmajor == 0, unit stride along N) or [batch][N][K]
 *     (b_kmajor != 0, unit stride along K); b_strides = {batch, row}.
 *  C: [batch][M][N], c_strides = {batch, row}; unit stride along N.
 *  Strides are in elements, multiples of 8 (of 4 for GR_F32); batch stride 0 broadcasts.
 *  epilogue: GR_EPI_NONE, GR_EPI_RELU or GR_EPI_SILU, applied to alpha*acc.
 *  (block_m, block_n) in {(128,128), (256,128), (128,256), (256,256)}
 *  (0 = 256; both 0: for fp16/bf16 the library picks the tile by M, N, K and
 *  batch, 32 x 128 and 64 x 128 ones included). Any M; N a multiple of 8; K a multiple of 32 (the square
 *  tiles use 64-deep k tiles when K allows). The 256 x 256 tile runs four
 *  waves of 128 x 128 (one per SIMD); the other tiles run eight waves.
 *  With batch 1, a 256 x 256 launch whose last round of workgroups would
 *  fill at most half of the device's CUs is issued as two launches on the
 *  stream: the columns of the whole rounds, then the rest on 256 x 128
 *  tiles (same results: each output's k order is unchanged).
 *  Edge tiles of C are stored only where valid. */
#define GR_EPI_NONE 0
#define GR_EPI_RELU 1
#define GR_EPI_SILU 2
int gr_gemm(const void* a, const void* b, void* c, int dtype, int batch, int M, int N, int K,
            const long long* a_strides, const long long* b_strides, const long long* c_strides,
            int b_kmajor, int epilogue, float alpha, int block_m, int block_n, void* stream);

/* gr_gemm with block_m = block_n = 0 and device memory to split K over
 * workgroups where the tiles of C alone would leave CUs idle (few rows, narrow
 * C): the parts' fp32 sums go through `workspace` (16-byte aligned, at least
 * gr_gemm_workspace(dtype, batch, M, N, K) bytes; the call overwrites it) and a
 * second kernel adds them in a fixed order and applies the epilogue. With a
 * smaller or NULL workspace the call runs without that split.
 * gr_gemm_workspace is at most 64 MiB, and 0 where no split is picked (GR_F32
 * among them). No counterpart in the reference. */
size_t gr_gemm_workspace(int dtype, int batch, int M, int N, int K);
int gr_gemm_ws(const void* a, const void* b, void* c, int dtype, int batch, int M, int N, int K,
               const long long* a_strides, const long long* b_strides, const long long* c_strides,
               int b_kmajor, int epilogue, float alpha, void* workspace, size_t workspace_bytes, void* stream);

/* Whether gr_gemm with block_m = block_n = 0 runs an fp32 product (K in `ktiles`
 * tiles of 16, or 8 where 16 does not divide it) as 32 x 32 blocks with K over the
 * four waves of a workgroup rather than on block_m x block_n tiles, on `cus`
 * compute units: 1 or 0. Rendered fp32 stages follow the same rule. No counterpart in the reference. */
int gr_gemm_f32_groups(int batch, int M, int N, int ktiles, int b_kmajor, int block_m, int block_n, int cus);

/* MLP block Y = SiLU(X @ W1) @ W2 as two GEMMs, SiLU fused into the first.
 * The grammar's MLP program (run_mlp_search.py:42-127, with silu in place of
 * relu + residual + LayerNorm). X [M][D], W1 [D][F], W2 [F][D], Y [M][D],
 * all row-major and contiguous; h is caller-provided [M][F] workspace. */
int gr_mlp_fwd(const void* x, const void* w1, const void* w2, void* h, void* y, int dtype, int M,
               int D, int F, int block_m, int block_n, void* stream);

/* gr_mlp_fwd with block_m = block_n = 0 and a workspace for its GEMMs' K
 * splits, as gr_gemm_ws (both GEMMs use the same memory, one after the other). */
size_t gr_mlp_fwd_workspace(int dtype, int M, int D, int F);
int gr_mlp_fwd_ws(const void* x, const void* w1, const void* w2, void* h, void* y, int dtype, int M,
                  int D, int F, void* workspace, size_t workspace_bytes, void* stream);

/* Self-test of the 32x32x16 MFMA operand/accumulator layout the kernels
 * assume: one wavefront computes D[32][32] = A[32][16] @ B[16][32] (fp16 in,
 * fp32 out, all row-major device buffers). */
int gr_selftest_mfma32(const void* a, const void* b, float* d, void* stream);

/* Self-test of the fp32 attention's unsplit path: the calling thread's next
 * `lookups` key-split workspaces fail to allocate (each asks the device for
 * more memory than it has), whether or not the stream has one already. */
int gr_selftest_f32_no_workspace(int lookups);

/* Self-test of the check for outputs that overlap inputs, on the host: 1 if two
 * arrays of `size`-byte elements, of 4 sizes and non-negative strides in
 * elements each, share memory, else 0. The addresses are not followed. */
int gr_selftest_overlap(const void* a, const long long* a_sizes, const long long* a_strides, const void* b,
                        const long long* b_sizes, const long long* b_strides, int size);

#ifdef __cplusplus
}
#endif
#endif /* GRAMMAR_RT_H */
