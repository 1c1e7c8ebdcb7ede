/* include/knj_capi.h -- C ABI of the MI355X (gfx950) MoE decode library.
 *
 * Plain C: pointers, sizes, ints.  Device pointers are addresses in the GPU's
 * memory (from knj_malloc, or any HIP allocation); `stream` is a hipStream_t
 * passed as void* (NULL = the default stream).  Every function returns 0 on
 * success or one of the KNJ_E_* codes below, with a message in knj_last_error().
 *
 * The status codes keep the reference's driver exit codes
 * (/root/reference/tools/bench/q4k_moe_ffn.hip:63, tests/test_gemm_w4.hip:11-19):
 * 5 correctness, 6 arch mismatch, 7 environment, 9 HIP error.
 */
#ifndef KNJ_CAPI_H
#define KNJ_CAPI_H

#include <stdint.h>

#include "knj_model.h"

#ifdef __cplusplus
extern "C" {
#endif

#define KNJ_OK 0
#define KNJ_E_CORRECTNESS 5
#define KNJ_E_ARCH 6
#define KNJ_E_ENV 7
#define KNJ_E_HIP 9
#define KNJ_E_ARG 22
#define KNJ_E_STATE 23

/* ------------------------------------------------------------ device gate
 * Replaces the reference's C2 gate: Backend::create's arch guard and
 * DeviceCaps probe (/root/reference/src/device/backend.cpp:54-62,
 * src/device/device_caps.h:69-157).  The guard compares the device's
 * gcnArchName up to the first ':' with the arch this library was compiled for
 * ("gfx950"); if KNJ_BUILD_ARCH is set in the environment it must name the same
 * arch.  Refusals return KNJ_E_ARCH (mismatch) and leave the device untouched. */
typedef struct knj_device_caps {
  char gcn_arch[32];      /* e.g. "gfx950" (the part before ':') */
  char name[64];
  int32_t wave_size;      /* 64 on CDNA */
  int32_t cu_count;
  int32_t clock_khz;
  int32_t lds_per_block;  /* bytes */
  int32_t l2_bytes;
  int32_t arch_ok;
  int32_t has_mfma_bf16;
  int32_t has_mfma_i8;
  int32_t has_fp8;
  uint64_t vram_total;
  uint64_t vram_free;
} knj_device_caps;

int knj_device_open(int device);
int knj_device_close(void);
int knj_device_caps_get(knj_device_caps* out);
/* Arch guard alone, on strings (host-testable without a GPU): 0 when
 * `device_arch` (full gcnArchName) matches `built_arch` and `env_arch` (may be
 * NULL) agrees, else KNJ_E_ARCH. */
int knj_check_arch(const char* device_arch, const char* built_arch, const char* env_arch);
const char* knj_built_arch(void);
const char* knj_last_error(void);

/* ------------------------------------------------------------ memory */
int knj_malloc(void** dptr, uint64_t bytes);
int knj_free(void* dptr);
int knj_memcpy_h2d(void* dst, const void* src, uint64_t bytes);
int knj_memcpy_d2h(void* dst, const void* src, uint64_t bytes);
int knj_memset_zero(void* dst, uint64_t bytes);
int knj_synchronize(void);

/* ------------------------------------------------------------ format / GEMV
 * knj_dequant: n_weights of `type` at w -> f32, bit-exact with
 *   dequant_row_f32 (/root/reference/src/loader/dequant.cpp:1114-1256).
 * knj_gemv: y[j] = sum_i W[j][i] x[i] for the n_out rows of W, the device
 *   counterpart of Model::matmul at m == 1 (/root/reference/src/model/model.cpp:
 *   326-380) and dequant_dot_f32 (dequant.cpp:1075-1112).  `norm_w` (optional)
 *   applies RMSNorm(x, norm_w, eps) to x first (model.cpp:240-271); `resid`
 *   (optional) makes y = resid + W x (the residual adds at model.cpp:624, 652).
 *   Types: Q4_K, Q6_K (rows of n_in/256 blocks), BF16, F32. */
int knj_dequant(int type, const void* w, uint64_t n_weights, float* out, void* stream);
int knj_gemv(int type, const void* w, int n_in, int n_out, const float* x, const float* norm_w,
             float eps, const float* resid, float* y, void* stream);
int knj_rmsnorm(const float* x, const float* w, int n, float eps, float* out, void* stream);

/* ------------------------------------------------------------ MoE (config 1)
 * knj_moe_router: logits = router_w . RMSNorm(x) (norm skipped when norm_w is
 *   NULL), softmax over all experts, top-k by repeated argmax with ties to the
 *   lower index, weights renormalised over the kept k (model.cpp:420-460).
 *   hx receives the normalised input.  topk in selection order.
 * knj_moe_decode_layer: the whole batch-1 MoE FFN: router as above, then for the
 *   k chosen experts gate/up GEMV, silu(gate)*up, down GEMV, and
 *   out = resid + sum_e w_e * down_e, summed in ascending expert index
 *   (model.cpp:462-509, the moe-router/gate/up/act/down/scatter stages).
 *   `resid` may be NULL (out is then the expert branch alone). */
int knj_moe_router(const float* x, const float* norm_w, float eps, const float* router_w,
                   int n_embd, int n_expert, int k, float* hx, float* logits, int32_t* topk_idx,
                   float* topk_w, void* stream);
int knj_moe_decode_layer(const float* x, const float* norm_w, float eps, const float* router_w,
                         const void* gate, const void* up, const void* down, int type_gate_up,
                         int type_down, int n_embd, int n_ff, int n_expert, int k,
                         const float* resid, float* out, float* logits, int32_t* topk_idx,
                         float* topk_w, void* stream);
/* knj_moe_decode_layer_noalloc: knj_moe_decode_layer computed by the same
 *   kernels, with its scratch (hx, then act: n_embd + k * n_ff floats) in a
 *   fixed device array of 32768 floats (128 KiB per device, held until the
 *   process ends) instead of library-allocated memory: the call allocates and
 *   frees nothing.  No counterpart in the reference; it is for callers that
 *   cannot allocate (code under HIP graph capture, tight serving loops,
 *   harnesses that forbid hipMalloc).  Larger shapes return KNJ_E_ARG.  Every
 *   call on a device shares that device's array, so calls that overlap on one
 *   device (other streams, other threads) race; nothing in the array needs to
 *   start at zero.  The device must have been opened with knj_device_open. */
int knj_moe_decode_layer_noalloc(const float* x, const float* norm_w, float eps,
                                 const float* router_w, const void* gate, const void* up,
                                 const void* down, int type_gate_up, int type_down, int n_embd,
                                 int n_ff, int n_expert, int k, const float* resid, float* out,
                                 float* logits, int32_t* topk_idx, float* topk_w, void* stream);

/* ------------------------------------------------------------ MoE over many tokens (config 2)
 * knj_moe_batch_layer: Model::moe on n_tokens rows at once (model.cpp:399-510
 *   with m > 1, the batched matmul of :354-364): per token RMSNorm(x) (norm
 *   skipped when norm_w is NULL), router logits, softmax and top-k as in
 *   knj_moe_router; the (token, expert) pairs grouped by expert so every
 *   expert's weights are read once for all its tokens; gate/up, silu(gate)*up,
 *   down; out[t] = resid[t] + sum over t's experts in ascending index of
 *   w * down.  x, resid, out: [n_tokens][n_embd]; logits: [n_tokens][n_expert];
 *   topk_idx/topk_w: [n_tokens][k].  Q4_K gate/up, Q4_K or Q6_K down; n_embd
 *   and n_ff multiples of 256, at most 4096; n_expert <= 256; k <= 16. */
int knj_moe_batch_layer(const float* x, const float* norm_w, float eps, const float* router_w,
                        const void* gate, const void* up, const void* down, int type_gate_up,
                        int type_down, int n_tokens, int n_embd, int n_ff, int n_expert, int k,
                        const float* resid, float* out, float* logits, int32_t* topk_idx,
                        float* topk_w, void* stream);

/* ------------------------------------------------------------ attention
 * knj_attention_step: the attention block of one decode token
 *   (/root/reference/src/model/model.cpp:567-616 with an f16 cache): per-head
 *   RMSNorm of the raw projections q [n_head][D] and k [n_head_kv][D] with
 *   q_norm / k_norm, NEOX RoPE at `pos` (pairs (i, i+D/2),
 *   theta = pos*base^(-2i/D)), k and v rounded to f16 and stored at slot `pos`
 *   of the [n_head_kv][n_ctx][D] caches, then GQA attention of every query head
 *   over slots [0, pos]: scores q.k/sqrt(D), softmax, out = sum a*v.
 *   q, k, v are not modified.  D is 64 or 128; the GQA group is at most 8. */
int knj_attention_step(const float* q, const float* k, const float* v, const float* q_norm,
                       const float* k_norm, float eps, float rope_base, int pos, int n_head,
                       int n_head_kv, int head_dim, int n_ctx, uint16_t* k_cache, uint16_t* v_cache,
                       float* out, void* stream);

/* ------------------------------------------------------------ speculative step
 * The operators around a step that verifies drafted tokens: rotary positions of
 * any layout and scaling, a cache in f16 or 8 bits written and read back, the
 * attention of a tree of drafts over that cache, and the log probabilities of
 * given tokens.  No counterpart in the reference, which decodes one token at a
 * time.  These calls queue their kernels on `stream` and return: they allocate
 * nothing, synchronise nothing and keep nothing between calls (scratch is the
 * caller's `workspace`), so they can be captured into a HIP graph; two calls
 * that may run at once need a workspace each.  All pointers are memory of the
 * device opened by knj_device_open, which must be the calling thread's current
 * one (KNJ_E_STATE otherwise).  `type` is that of the activations: KNJ_TYPE_F32,
 * KNJ_TYPE_F16 or KNJ_TYPE_BF16; arithmetic is f32 (angles f64; the attention's operands
 * as knj_attention_tree says), results are rounded once.
 * Rows of activations and caches start on 16-byte boundaries, their strides
 * count elements, other arrays are aligned to their types; anything else is refused.
 * head_dim is 64 or 128. */

/* knj_rope: every head of rows q [n_rows][n_head][head_dim] (and k
 *   [n_rows][n_head_kv][head_dim]; n_head_kv 0: none) RMS-normalised with its
 *   norm weight (NULL: not; eps at least 0) and rotated at position pos[row]: the first n_rot
 *   dims (a multiple of 8) in pairs (i, i + n_rot/2) (KNJ_ROPE_HALF) or
 *   (2i, 2i + 1) (KNJ_ROPE_INTERLEAVED) by the angle pos * inv_freq[i], cos and
 *   sin times mscale; the other dims pass.  Angles are formed in f64 (the decode
 *   step's own tables hold f32 angles: they part by up to pos * 2^-24 radians).
 *   An output may be its own input (the same pointer and stride; another stride is
 *   refused) and overlaps no other row.  n_rows < 2^24.
 * knj_rope_freqs (host only): the n_rot/2 frequencies base^(-2i/n_rot) under a
 *   scaling for contexts `factor` (>= 1) times orig_ctx, to be copied to the
 *   device, and mscale.  KNJ_ROPE_LINEAR: / factor.  KNJ_ROPE_NTK: base times
 *   factor^(n_rot/(n_rot-2)).  KNJ_ROPE_YARN: a ramp between the two over the
 *   dims whose wavelength turns p0 (beta_fast, e.g. 32) to p1 (beta_slow, e.g. 1)
 *   times in orig_ctx, mscale 0.1 ln(factor) + 1.  KNJ_ROPE_LLAMA3: / factor for
 *   wavelengths above orig_ctx/p0 (low_freq_factor), kept below orig_ctx/p1
 *   (high_freq_factor), interpolated between. */
#define KNJ_ROPE_HALF 0
#define KNJ_ROPE_INTERLEAVED 1
#define KNJ_ROPE_NONE 0
#define KNJ_ROPE_LINEAR 1
#define KNJ_ROPE_NTK 2
#define KNJ_ROPE_YARN 3
#define KNJ_ROPE_LLAMA3 4
int knj_rope_freqs(int n_rot, double base, int scaling, double factor, int orig_ctx, double p0,
                   double p1, double* inv_freq, float* mscale);
int knj_rope(int type, int layout, int n_rot, const double* inv_freq, float mscale,
             const int32_t* pos, int n_rows, int head_dim, const void* q, int n_head,
             uint64_t q_stride, const float* q_norm, void* q_out, uint64_t q_out_stride,
             const void* k, int n_head_kv, uint64_t k_stride, const float* k_norm, void* k_out,
             uint64_t k_out_stride, float eps, void* stream);

/* One layer's cache of n_seq sequences: k and v [n_head_kv][n_ctx][head_dim] per
 *   sequence, sequence s at element s * seq_stride (the layout of the model's own
 *   f16 cache; seq_stride 0: back to back), in one of three formats.  The 8-bit
 *   ones hold a scale per (slot, kv head) in k_scale and v_scale [n_head_kv][n_ctx]
 *   per sequence, sequence s at s * seq_stride / head_dim:
 *   KNJ_KV_I8: scale = amax/127, codes rint(x * 127/amax);
 *   KNJ_KV_F8: scale = amax/448, codes e4m3(x * 448/amax).
 *   Codes are those of the exact quotient, ties to even.  A row whose largest
 *   magnitude is below 2^-119 is stored as zeros; a row that holds an infinity or
 *   a NaN reads back as NaN (KNJ_KV_F16 keeps them as they are).
 * knj_kv_store: rows t < counts[s] (NULL: n_rows) of sequence s, k and v
 *   [n_seq][n_rows][n_head_kv][head_dim] with row_stride elements from a row to
 *   the next (of both: keys rotated in place in their projections' rows keep the
 *   values' stride), go to slots start[s] + t.  Rows that would fall outside
 *   [0, n_ctx) are not stored.  n_rows * n_head_kv < 2^27, here and in knj_kv_load.
 * knj_kv_load: slots[s][t] (NULL: slot t) of the cache into rows k and v of the
 *   same form, as code * scale rounded to `type`; rows whose slot is outside
 *   [0, n_ctx) are left as they were.  Loaded as f32 and stored again, a row keeps
 *   its codes, and its scale to a rounding (one within a rounding of 2^-119 may come
 *   out as zeros): how an accepted path of drafts moves to the end of the prefix. */
#define KNJ_KV_F16 0
#define KNJ_KV_F8 1
#define KNJ_KV_I8 2
typedef struct knj_kv_cache {
  void* k;
  void* v;
  float* k_scale; /* NULL with KNJ_KV_F16 */
  float* v_scale;
  uint64_t seq_stride;
  int32_t format;
  int32_t n_seq, n_head_kv, n_ctx, head_dim;
} knj_kv_cache;
int knj_kv_store(const knj_kv_cache* cache, int type, const void* k, const void* v,
                 uint64_t row_stride, const int32_t* start, const int32_t* counts, int n_rows,
                 void* stream);
int knj_kv_load(const knj_kv_cache* cache, int type, const int32_t* slots, int n_rows, void* k,
                void* v, uint64_t row_stride, void* stream);

/* knj_attention_tree: attention of up to n_rows drafts per sequence over the
 *   cache, which already holds the drafts' keys and values: draft t of sequence s
 *   is in slot prefix[s] + t (t < counts[s]; NULL: n_rows) and sees the slots
 *   before prefix[s] and those drafts u < counts[s] whose bit u % 64 of word u / 64
 *   of its mask row is set: mask [n_seq][n_rows][ceil(n_rows/64)] words, one
 *   [n_rows][..] for all sequences with mask_shared, NULL for a chain (u <= t).
 *   q, out: [n_seq][n_rows][n_head][head_dim] with q_stride and out_stride
 *   elements per row; out = softmax(scale * q.k) v over the slots seen.  Whatever
 *   unseen slots hold counts for nothing, NaN included; a draft that sees nothing
 *   gives zeros; rows past counts[s] are left as they were.  A draft that sees a
 *   draft whose value row holds an infinity or a NaN gives NaN (all of its dims); one
 *   that sees a key row with either may give NaN.
 *   prefix[s] is held to [0, max_prefix] and counts[s] to [0, n_rows]; max_prefix +
 *   n_rows <= n_ctx and below 2^31 - 256, n_rows <= 1024, scale in [1e-6, 1e6], n_head a
 *   multiple of n_head_kv and at most 1024.
 *   Queries may be of any size that leaves the scores, scale q.k, below 2^25 in magnitude,
 *   with scale |q| below 2^126 and 8-bit keys below 2^100.
 *   out may be q (with out_stride = q_stride; another is refused) and overlaps nothing
 *   else.  On the matrix cores f32 queries, and the softmax's weights with any
 *   activations, keep 22 bits: with an 8-bit cache of the largest product of a weight and
 *   a value scale, down to 2^-80 of the largest weight times the largest scale.
 * knj_attention_tree_workspace: bytes its workspace needs for these sizes (0: none,
 *   or arguments that it refuses); any contents.  Smaller sizes can need more (their
 *   slots are split further), but none more than 262144 * (head_dim + 4). */
int knj_attention_tree(const knj_kv_cache* cache, int type, const void* q, uint64_t q_stride,
                       int n_head, int n_rows, const int32_t* prefix, int max_prefix,
                       const int32_t* counts, const uint64_t* mask, int mask_shared, float scale,
                       void* out, uint64_t out_stride, void* workspace, uint64_t workspace_bytes,
                       void* stream);
uint64_t knj_attention_tree_workspace(const knj_kv_cache* cache, int n_head, int n_rows,
                                      int max_prefix);

/* knj_token_logprobs: of rows of logits [n_rows][n_vocab] (row_stride elements
 *   from a row to the next, any alignment of `type`'s own), with x = logits /
 *   temperature and lse = log sum exp(x):
 *   logprob[row] = x[tokens[row]] - lse (tokens and logprob: both or neither; 0
 *     where the token is negative, NaN where it is n_vocab or above);
 *   entropy[row] = -sum p log p, p = exp(x - lse) (NULL: not computed);
 *   top_idx, top_logprob [n_rows][n_top]: the n_top largest logits, largest first,
 *     ties to the lowest index, with their log probabilities (n_top 0: none; at
 *     most 32 and n_vocab).
 *   -inf rules a token out.  A row with nothing left gives log probabilities of
 *   -inf and an entropy of 0; a row that holds a NaN or +inf gives NaN (in top_idx a
 *   NaN ranks as -inf).  n_vocab <= 2^20, n_rows < 2^24 and
 *   n_rows * ceil(n_vocab / 2048) < 2^26.
 * knj_token_logprobs_workspace: bytes of its workspace; any contents. */
int knj_token_logprobs(int type, const void* logits, uint64_t row_stride, int n_rows, int n_vocab,
                       float temperature, const int32_t* tokens, float* logprob, float* entropy,
                       int n_top, int32_t* top_idx, float* top_logprob, void* workspace,
                       uint64_t workspace_bytes, void* stream);
uint64_t knj_token_logprobs_workspace(int n_rows, int n_vocab);

/* ------------------------------------------------------------ a 4-bit cache in pages
 * A cache of n_layer layers in 4 bits whose slots lie in pages that sequences share: a
 * prompt's pages serve every answer to it, beams take over their parents' pages, and what
 * is written is copied first.  No counterpart in the reference.  The rules of the
 * speculative step's calls hold (stream, no allocation, device, types, alignment); calls
 * that change the table, the counts or a page are ordered by the caller (one stream).
 *
 * Keys and values are held in groups of 32 dims as code * step + low rounded to f16 (one
 *   rounding), step and low f16, code 0 to 15: low is the group's smallest element rounded
 *   to f16, step the largest f16 not above (largest - low) / 15 (0 if that is negative),
 *   code = (x - low) / step in f64, rounded to nearest even and held to [0, 15] (0 where step
 *   is 0).  A group that holds an infinity, a NaN or a magnitude above 65504 reads back as
 *   NaN.
 * data [n_layer][n_page] pages of n_head_kv * page_size * head_dim * 5 / 4 bytes: per kv
 *   head the page's key codes [page_size][head_dim / 2] bytes, its value codes, then a word
 *   a group [page_size][head_dim / 32] for keys and for values (step the low half, low the
 *   high one).  Of eight dims from 8 w on, word w of a row's codes holds dim 8 w + i in bits
 *   4 (i / 2) + 16 (i % 2) and up.
 * table [n_seq][n_table]: the page of a sequence's slots e * page_size to (e + 1) *
 *   page_size - 1; an entry outside [0, n_page) is none.  refs [n_page]: how many entries
 *   hold a page; a page with none is free (a caller who wants a page to outlive its entries
 *   adds a count of its own).  Calls that do not name the table (knj_pages_copy) or the counts
 *   (all but reserve, fork and free) take NULL there.
 * page_size: a power of two from 16 to 256.  n_layer at most 1024, n_seq at most 4096, n_head_kv
 *   at most 64, n_page below 2^26, n_table * page_size below 2^31 - 256, n_seq * n_table below
 *   2^31 - 1024.  data is 16-byte aligned.
 * knj_pages_bytes: bytes of data (0: sizes that are refused); pointers are not looked at. */
typedef struct knj_kv_pages {
  void* data;
  int32_t* table;
  int32_t* refs;
  int32_t n_layer, n_page, page_size, n_head_kv, head_dim;
  int32_t n_seq, n_table;
} knj_kv_pages;
uint64_t knj_pages_bytes(const knj_kv_pages* pages);

/* knj_pages_store, knj_pages_load: as knj_kv_store and knj_kv_load, of one layer.  Rows
 *   whose slot has no page are not stored, and left as they were when loaded.  Rows stored
 *   into a page that has other holders are theirs too (knj_pages_reserve gives a
 *   sequence pages of its own). */
int knj_pages_store(const knj_kv_pages* pages, int layer, int type, const void* k, const void* v,
                    uint64_t row_stride, const int32_t* start, const int32_t* counts, int n_rows,
                    void* stream);
int knj_pages_load(const knj_kv_pages* pages, int layer, int type, const int32_t* slots,
                   int n_rows, void* k, void* v, uint64_t row_stride, void* stream);

/* knj_attention_pages: knj_attention_tree over one layer of pages: its arguments, masks and
 *   limits (n_ctx is n_table * page_size; a decode step is n_rows 1 with its own key stored, a
 *   piece of a prompt n_rows up to 1024 without a mask).  A slot without a page holds NaN.
 *   A value group of a prefix slot that reads back as NaN makes its own 32 dims NaN, of every
 *   row; of a draft's slot, as there, all dims of the rows that see it.  f32 queries keep 22 bits; weights keep 22 bits with any activations, and queries are of
 *   any size that leaves the scores, scale q.k, below 2^25 in magnitude with scale |q| below
 *   2^126. */
int knj_attention_pages(const knj_kv_pages* pages, int layer, int type, const void* q,
                        uint64_t q_stride, int n_head, int n_rows, const int32_t* prefix,
                        int max_prefix, const int32_t* counts, const uint64_t* mask,
                        int mask_shared, float scale, void* out, uint64_t out_stride,
                        void* workspace, uint64_t workspace_bytes, void* stream);
uint64_t knj_attention_pages_workspace(const knj_kv_pages* pages, int n_head, int n_rows,
                                       int max_prefix);

/* knj_pages_reserve: sequence s, which holds length[s] slots, gets a page of its own for every
 *   slot from start[s] (NULL: length[s]) to want[s] - 1: entries that are none, and those
 *   whose page has other holders, take the lowest-numbered free pages, in order of sequence
 *   and entry.  Of a page that is replaced the slots below length[s] are copied, in all
 *   layers; a page that all its holders would replace stays with the last of them.  If there
 *   are not enough free pages nothing changes.  *missing: how many were short (0: done).
 *   Slots past the table's n_table * page_size get none.
 * knj_pages_fork: sequence s becomes the first keep[s] slots (NULL: all) of sequence parent[s]
 *   as it was before the call, for all s at once (parent[s] = s keeps a sequence, one outside
 *   [0, n_seq) empties it).  Pages are shared, not copied.
 * knj_pages_free: sequence s keeps its first keep[s] slots (a negative keep[s]: all) and gives
 *   the pages behind them back.
 * knj_pages_compact: in every layer, the key and value of slot rows[s][i] move to slot
 *   start[s] + i, i < counts[s] (NULL: n_rows); rows [n_seq][n_rows] ascend and rows[s][i] is
 *   at least start[s] + i.  How the accepted path of a tree of drafts moves behind the
 *   prefix, or what is kept of a long context together.  Codes move as they are.  The pages
 *   written to are to be the sequence's own (knj_pages_reserve from start[s] on).  A row
 *   whose slot, old or new, has no page stays.
 * knj_pages_copy: pages src[i] of one pool into pages dst[i] of another of the same n_layer,
 *   page_size, n_head_kv and head_dim, or of the same pool, i < n < 2^24, in all layers.  Pairs with a
 *   number outside its pool are left out; no page that is written may be read or written
 *   by another pair.
 * knj_pages_workspace: bytes of the workspace of reserve and fork; any contents. */
int knj_pages_reserve(const knj_kv_pages* pages, const int32_t* start, const int32_t* length,
                      const int32_t* want, int32_t* missing, void* workspace,
                      uint64_t workspace_bytes, void* stream);
int knj_pages_fork(const knj_kv_pages* pages, const int32_t* parent, const int32_t* keep,
                   void* workspace, uint64_t workspace_bytes, void* stream);
int knj_pages_free(const knj_kv_pages* pages, const int32_t* keep, void* stream);
int knj_pages_compact(const knj_kv_pages* pages, const int32_t* start, const int32_t* rows,
                      const int32_t* counts, int n_rows, void* stream);
int knj_pages_copy(const knj_kv_pages* to, const knj_kv_pages* from, const int32_t* dst,
                   const int32_t* src, int n, void* stream);
uint64_t knj_pages_workspace(const knj_kv_pages* pages);

/* ------------------------------------------------------------ model step
 * The device counterpart of knj::Model (/root/reference/src/model/model.h:55-80):
 * open -> forward(tokens, n) -> logits of the last token, reset(), pos().
 * Weights live in one device image laid out per include/knj_model.h.
 * knj_model_create_synthetic generates the seeded synthetic weights on the GPU
 * (include/knj_synth.h, bit-identical to the host generator);
 * knj_model_create_from_image uploads a host image. */
typedef struct knj_model knj_model;
int knj_model_create_synthetic(const knj_model_config* cfg, uint64_t seed, knj_model** out);
int knj_model_create_from_image(const knj_model_config* cfg, const void* image, uint64_t bytes,
                                knj_model** out);
/* A qwen3moe GGUF file (the reference's Model::open, model.cpp:174-232, and its
 * geometry/tensor checks, :97-172): knj_gguf_probe reads the geometry and the
 * weight types into `out` without a device; knj_model_create_from_gguf also
 * copies every tensor into a device model (Q, K and V rows into one wqkv).
 * Errors: a missing key or tensor, a wrong shape, an unsupported type, n_ctx
 * beyond the trained context -- each with its name in knj_last_error(). */
int knj_gguf_probe(const char* path, int n_ctx, knj_model_config* out);
int knj_model_create_from_gguf(const char* path, int n_ctx, knj_model** out);
int knj_model_config_get(const knj_model* m, knj_model_config* out);
int knj_model_free(knj_model* m);
uint64_t knj_model_image_bytes(const knj_model* m);
const void* knj_model_image_device(const knj_model* m);
/* Fills cache slots [0, n_pos) of every layer with seeded f16 values ~N(0,1)
 * and sets the position to n_pos: a long context without running its prefill
 * (for throughput runs; the decode step's work is the same). */
int knj_model_fill_kv(knj_model* m, int n_pos, uint64_t seed);
/* ------------------------------------------------------------ batched decode (config 4)
 * A knj_batch decodes n_seq sequences in lockstep on one model's weights (the
 * model must outlive it): one step is Model::forward's per-token work
 * (model.cpp:512-672) for n_seq tokens at once, each sequence with its own f16
 * KV cache of n_ctx slots (n_ctx <= the model's) and its own position.  Every
 * weight matrix is read once per step for all sequences (matrix-core GEMMs;
 * the MoE pairs grouped by expert).  Q4_K attention and gate/up, Q4_K or Q6_K
 * expert down, bf16 or Q6_K head.
 * knj_batch_forward: one step on tokens[n_seq]; logits_out [n_seq][n_vocab]
 *   (may be NULL).  knj_batch_decode_greedy: `steps` greedy steps from
 *   first[n_seq]; out_tokens [steps][n_seq].  Hidden states, top-k and caches
 *   of the last step per sequence as for knj_model_*.  No counterpart in the
 *   reference, which decodes one sequence. */
typedef struct knj_batch knj_batch;
int knj_batch_create(knj_model* m, int n_seq, int n_ctx, knj_batch** out);
int knj_batch_free(knj_batch* b);
int knj_batch_pos(const knj_batch* b);
int knj_batch_forward(knj_batch* b, const int32_t* tokens, float* logits_out);
int knj_batch_decode_greedy(knj_batch* b, const int32_t* first, int steps, int32_t* out_tokens);
int knj_batch_fill_kv(knj_batch* b, int n_pos, uint64_t seed);
int knj_batch_hidden(const knj_batch* b, int il, int seq, float* out);
int knj_batch_topk(const knj_batch* b, int il, int seq, int32_t* idx, float* w);
int knj_batch_kv_download(const knj_batch* b, int seq, uint16_t* k, uint16_t* v);
/* One sequence's whole cache ([n_layer][n_head_kv][n_ctx][head_dim] f16, the
 * batch's n_ctx) from the host, e.g. a cache a knj_model prompt pass wrote; and
 * the lockstep position of every sequence. */
int knj_batch_kv_upload(knj_batch* b, int seq, const uint16_t* k, const uint16_t* v);
int knj_batch_set_pos(knj_batch* b, int pos);

/* Byte offsets of layer `il`'s tensors inside the weight image of a model of
 * configuration `c` (the layout of knj_model.h); returns the image size, 0 on a
 * bad argument. */
uint64_t knj_model_layer_offsets(const knj_model_config* c, int il, knj_layer_offsets* out);
int knj_model_download_image(const knj_model* m, void* host, uint64_t bytes);
int knj_model_reset(knj_model* m);
int knj_model_pos(const knj_model* m);
int knj_model_set_pos(knj_model* m, int pos);
/* Model::forward (/root/reference/src/model/model.cpp:512-672): runs n tokens at
 * positions pos .. pos+n-1.  n == 1 is one decode step (the captured graph);
 * n > 1 is the prompt pass: every weight applied to up to 512 rows at once,
 * each row's key and value appended, causal attention (row t over slots
 * 0 .. pos+t), the head on the last row -- for Q4_K attention and gate/up
 * and Q4_K or Q6_K expert down (other tensor types take one decode step per
 * token).  logits_host (n_vocab
 * floats, may be NULL) receives the last token's logits; the per-layer
 * hidden/top-k queries then describe the last token.  Errors: KNJ_E_ARG for
 * token ids out of range or a full context (model.cpp:514-517, 533), nothing
 * run. */
int knj_model_forward(knj_model* m, const int32_t* tokens, int n, float* logits_host);
/* Greedy decode entirely on the device: feeds `first`, then `steps` argmax
 * tokens (first maximum wins, /root/reference/src/cli/main.cpp:126-132) into
 * out_tokens.  Replays one captured HIP graph per step. */
int knj_model_decode_greedy(knj_model* m, int32_t first, int steps, int32_t* out_tokens);
/* Diagnostics of the most recent step: residual stream after layer il
 * (model.cpp:654-658), router choice of layer il, last logits, KV caches. */
int knj_model_hidden(const knj_model* m, int il, float* host_out);
int knj_model_topk(const knj_model* m, int il, int32_t* idx_out, float* w_out);
int knj_model_logits(const knj_model* m, float* host_out);
int knj_model_kv_download(const knj_model* m, uint16_t* k_host, uint16_t* v_host);
int knj_model_kv_upload(knj_model* m, const uint16_t* k_host, const uint16_t* v_host);
/* Times `iters` greedy steps with HIP events on the model's stream (graph
 * replays), returns total milliseconds. */
int knj_model_time_decode(knj_model* m, int iters, float* ms_out);
/* Times the expert GEMV kernels inside real decode steps: `steps` (1..64)
 * greedy tokens from token 0 at the current position, the step's kernels
 * launched directly (no graph); every layer's gate/up and down launch records
 * HIP start/end events of its own execution (hipExtLaunchKernel) on the
 * model's stream, and so does the router launch before them (unused: a launch
 * timed right after one without events reads the earlier launch's drain as
 * its own).  Returns the mean
 * microseconds per launch of each over n_layer * steps launches; advances the
 * position by `steps`. */
int knj_model_time_experts(knj_model* m, int steps, float* us_gateup, float* us_down);

/* ---- device spans for the profiler -------------------------------------------
 * The device event backend of the reference's profiler
 * (/root/reference/src/profiler/profiler.h:98-139: device_span() takes offsets
 * from one epoch event per stream, set_device_floor() a floor measured through
 * the same event path, set_device_dropped() the spans a full ring lost).  One
 * record per kernel launch: the op class it belongs to (the reference's scope
 * names where one kernel does one op -- "embed", "qkv", "attention", "attn-o",
 * "moe-router", "head" -- and joined names for fused kernels:
 * "moe-gate+up+act", "moe-down+scatter", "sample"), the layer (-1 outside the
 * layers), the kernel symbol, and the dispatch's own start/end in nanoseconds
 * after the epoch event. */
typedef struct knj_span {
  char name[32];
  char kernel[40];
  int32_t layer;
  int32_t stream;
  uint64_t start_ns;
  uint64_t end_ns;
} knj_span;

/* Greedy decode exactly as knj_model_decode_greedy (same tokens, same KV
 * writes, position advanced by `steps`), but with the step's kernels launched
 * directly, each with dispatch-recorded start/end events.  Up to `cap` spans
 * are written; *n_dropped counts launches beyond `cap` (a stated loss).
 * cap <= 1 << 20. */
int knj_model_profile(knj_model* m, int32_t first, int steps, int32_t* out_tokens, knj_span* spans,
                      int cap, int* n_spans, uint64_t* n_dropped);

/* Host<->device bytes this model's calls have copied since it was created
 * (weight upload, per-step token state, logits/tokens/diagnostic downloads):
 * the profiler's transfer row. */
int knj_model_transfer_bytes(const knj_model* m, uint64_t* h2d, uint64_t* d2h);

/* The device instrumentation floor: `n` empty kernels (one wave each, after
 * untimed warm-up launches) timed through the same dispatch-event path;
 * *ns_out is their median span. */
int knj_device_floor(int n, uint64_t* ns_out);

#ifdef __cplusplus
}
#endif

#endif /* KNJ_CAPI_H */
