/* C ABI of the MI355X-native cached block-diffusion step (libfdllm.so).
 *
 * Replaces the reference's TVM Relax VM function table for Fast-dLLM v2: the artifact exposes
 * REQUIRED_FNS (fast_dllm_relax/export_utils.py:13-17), called as vm["name"](..., params) by
 * fast_dllm_relax/runtime.py.  Every entry point below keeps the argument meaning, shapes and error
 * behaviour of the reference function it names; shapes are passed as plain ints and tensors as device
 * pointers (the caller owns every buffer; the KV caches are mutated in place, as in the reference).
 *
 * Conventions
 *   - All pointers are device pointers unless stated; `stream` is a hipStream_t (NULL = default).
 *   - Activations/weights/caches are in the context's dtype (bf16 or fp16, 2-byte elements);
 *     logits are fp32; token ids are int32.  Weights, activations, caches and logits must be
 *     16-byte aligned (FDLLM_EINVAL otherwise); id, offset and bias arrays need only their
 *     element alignment.
 *   - KV caches: [num_layers, 1, cap, num_kv_heads, head_dim] rows (contract "inplace_bsnh_v1",
 *     export_utils.py:21-34).
 *   - Return value: 0 on success; FDLLM_EINVAL for a rejected argument (the reference raises
 *     ValueError / a VM shape error); FDLLM_EHIP for a HIP runtime failure; FDLLM_ESTATE when weights
 *     are not bound.  fdllm_last_error() returns this thread's message for the last failure.
 *   - All work is enqueued on `stream`; nothing synchronises the host unless stated.  One context
 *     per stream; a context is not thread-safe.
 */
#ifndef FDLLM_H
#define FDLLM_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define FDLLM_OK 0
#define FDLLM_EINVAL 1
#define FDLLM_EHIP 2
#define FDLLM_ESTATE 3

#define FDLLM_DTYPE_BF16 0
#define FDLLM_DTYPE_F16 1

typedef struct fdllm_ctx fdllm_ctx;

/* Model constants; mirror of FastDLLMRelaxConfig (fast_dllm_relax/model/cuda.py:15-29). */
typedef struct fdllm_config {
  int32_t vocab_size;
  int32_t hidden_size;
  int32_t intermediate_size;
  int32_t num_hidden_layers;
  int32_t num_attention_heads;
  int32_t num_key_value_heads;
  int32_t head_dim;            /* 128 for the HIP attention kernel */
  float rms_norm_eps;
  float rope_theta;
  int32_t tie_word_embeddings;
  int32_t bd_size;             /* block size (32); partial steps use bd_size / 4 rows */
  int32_t dtype;               /* FDLLM_DTYPE_* */
  int32_t max_rows;            /* rows the workspace is sized for at creation (grown on demand) */
} fdllm_config;

/* Replaces tvm.relax.VirtualMachine(load_module(...)) (fast_dllm_relax/runners.py:614-615). */
int fdllm_create(const fdllm_config* cfg, fdllm_ctx** out);
void fdllm_destroy(fdllm_ctx* ctx);

/* Number of packed parameters and their names, in param_names.txt order
 * (fast_dllm_relax/runners.py:947-972; 198 for the tied 1.5B model). */
int fdllm_num_params(const fdllm_ctx* ctx);
const char* fdllm_param_name(const fdllm_ctx* ctx, int index);

/* Binds the packed `params` list (cuda.py:807, "param_mode": "packed"): n device pointers in
 * fdllm_param_name order, each 16-byte aligned (FDLLM_EINVAL otherwise).  The caller keeps them alive
 * while the context uses them. */
int fdllm_bind_weights(fdllm_ctx* ctx, const void* const* ptrs, int n);

/* embed (cuda.py:698-699): ids [seq_len] int32 -> out [seq_len, hidden]. */
int fdllm_embed(fdllm_ctx* ctx, const int32_t* ids, int seq_len, void* out, void* stream);

/* forward_hidden (cuda.py:604-608, 701-702): stateless forward of [1, seq_len, hidden] with the
 * additive attention bias [1, 1, seq_len, seq_len] fp32; bias == NULL means the block-causal bias of
 * build_prefix_block_attention_bias(0, seq_len, block_size=bd_size) (cuda.py:148-177). */
int fdllm_forward_hidden(fdllm_ctx* ctx, const void* input_embed, int seq_len, const float* attention_bias,
                         void* out, void* stream);

/* get_logits (cuda.py:704-711): hidden [rows, hidden] -> logits [rows, vocab] fp32 (rounded to the
 * model dtype first, as the reference's model-dtype GEMM output is). */
int fdllm_get_logits(fdllm_ctx* ctx, const void* hidden, int rows, float* logits, void* stream);

/* build_prefix_cache (cuda.py:610-637, 713-721): writes rows [0, prefix_len) of every layer of the
 * caches in place; prefix_bias as in fdllm_forward_hidden (NULL = block-causal). */
int fdllm_build_prefix_cache(fdllm_ctx* ctx, const void* prefix_embed, int prefix_len, const float* prefix_bias,
                             void* k_cache, void* v_cache, int cap, void* stream);

/* forward_cached (cuda.py:723-738, 639-666 with fast_dllm.attn_inplace, runtime.py:63-73): writes the
 * block's K/V at rows [prefix_len, prefix_len + block_len) and attends over [0, prefix_len + block_len).
 * cache_offset: device int32 scalar, RoPE position of row 0.  out [block_len, hidden]. */
int fdllm_forward_cached(fdllm_ctx* ctx, const void* active_embed, int block_len, void* k_cache, void* v_cache,
                         int cap, const int32_t* cache_offset, int64_t prefix_len, void* out, void* stream);

/* Allocation-free variant of fdllm_forward_cached.  It has no counterpart in the reference: it is for
 * callers that cannot allocate device memory inside a call (code under HIP graph capture, tight serving
 * loops, harnesses that forbid hipMalloc).  Same arguments, semantics and results (bit for bit) as
 * fdllm_forward_cached, but the step's workspace (residual stream, projections, norms, RoPE table and
 * the split partials of the projections and the attention) lives in a fixed 24 MiB device array of the
 * library, one per GPU, held until the process ends, and the call allocates and frees nothing.
 * Limits: at most 32 rows, and the attended keys must fit the scratch (the 1.5B shapes: up to 5120
 * keys through the chunked attention, more through the key-streaming one, in fewer splits where short); larger calls return FDLLM_EINVAL.
 * Every call on one GPU shares that GPU's array and leaves its contents behind: calls that overlap on
 * one GPU (two streams, threads or contexts) race. */
int fdllm_forward_cached_noalloc(fdllm_ctx* ctx, const void* active_embed, int block_len, void* k_cache,
                                 void* v_cache, int cap, const int32_t* cache_offset, int64_t prefix_len, void* out,
                                 void* stream);

/* forward_block_partial_rp{0,8,16,24} (cuda.py:740-788): bd_size/4 rows written at
 * [prefix_len + rp, + bd_size/4), attending over [0, prefix_len + bd_size). */
int fdllm_forward_block_partial(fdllm_ctx* ctx, int replace_position, const void* active_embed, int rows,
                                void* k_cache, void* v_cache, int cap, const int32_t* cache_offset,
                                int64_t prefix_len, void* out, void* stream);
int fdllm_forward_block_partial_rp0(fdllm_ctx* ctx, const void* active_embed, int rows, void* k_cache,
                                    void* v_cache, int cap, const int32_t* cache_offset, int64_t prefix_len,
                                    void* out, void* stream);
int fdllm_forward_block_partial_rp8(fdllm_ctx* ctx, const void* active_embed, int rows, void* k_cache,
                                    void* v_cache, int cap, const int32_t* cache_offset, int64_t prefix_len,
                                    void* out, void* stream);
int fdllm_forward_block_partial_rp16(fdllm_ctx* ctx, const void* active_embed, int rows, void* k_cache,
                                     void* v_cache, int cap, const int32_t* cache_offset, int64_t prefix_len,
                                     void* out, void* stream);
int fdllm_forward_block_partial_rp24(fdllm_ctx* ctx, const void* active_embed, int rows, void* k_cache,
                                     void* v_cache, int cap, const int32_t* cache_offset, int64_t prefix_len,
                                     void* out, void* stream);

/* The reference's attention callbacks, for a model that computes its own projections and RoPE and calls
 * out once per layer for the cache write and the attention (fast_dllm_relax/runtime.py:19-80, called
 * from model/cuda.py through rx.call_inplace_packed).  Tensors are BSNH with batch 1, in the context's
 * dtype: k / v [rows, nkv, head_dim], q / out [rows, nq, head_dim]; the caches [L, 1, cap, nkv,
 * head_dim] are the ones the other entry points take.  Neither call needs bound weights.
 *
 * fast_dllm.kv_write (runtime.py:76-80, _write_rows :51-60): k / v copied byte for byte to cache rows
 * [start, start + rows) of `layer`.  FDLLM_EINVAL: "KV write [s, e) outside cache capacity cap". */
int fdllm_kv_write(fdllm_ctx* ctx, const void* k, const void* v, int rows, void* k_cache, void* v_cache, int cap,
                   int layer, int64_t start, void* stream);

/* fast_dllm.attn_inplace (runtime.py:63-73): the write of fdllm_kv_write at rows [prefix_len + write_rel,
 * + rows), then out = softmax(q K^T / sqrt(head_dim)) V over cache rows [0, prefix_len + attend_rel) of
 * `layer`, no mask, query head h on kv head h / (nq / nkv) (_attend, runtime.py:30-48); like the
 * reference's slice of the cache, the attended rows stop at the capacity.  q must already be rotated.
 * FDLLM_EINVAL: "KV write [s, e) past the attended rows [0, n)" when the written rows end past the
 * attended ones, and the capacity error of fdllm_kv_write.  q, the caches and out must be 16-byte
 * aligned. */
int fdllm_attn_inplace(fdllm_ctx* ctx, const void* q, const void* k, const void* v, int rows, void* k_cache,
                       void* v_cache, int cap, int layer, int64_t prefix_len, int write_rel, int attend_rel,
                       void* out, void* stream);

/* Batched steps: no counterpart in the reference, whose entry points are batch 1
 * (fast_dllm_relax/model/cuda.py:796-836); they serve callers that refine one block per sequence
 * for many sequences at once.  nseq (<= 64) sequences share one cache tensor [L, nseq, cap, nkv, hd]
 * (inplace_bsnh_v1, export_utils.py:21-34, with a batch dimension); active_embed is [nseq, rows, H]
 * and out the same shape.  cache_offset is a device int32 [nseq] (row 0's RoPE position per
 * sequence) and prefix_lens a host int64 [nseq].  Each sequence follows the batch-1 semantics
 * exactly: fdllm_forward_cached_batch writes rows [P_b, P_b + rows) and attends [0, P_b + rows);
 * fdllm_forward_block_partial_batch writes [P_b + rp, + bd_size/4) and attends [0, P_b + bd_size).
 * Window errors name the sequence. */
int fdllm_forward_cached_batch(fdllm_ctx* ctx, const void* active_embed, int nseq, int rows, void* k_cache,
                               void* v_cache, int cap, const int32_t* cache_offset, const int64_t* prefix_lens,
                               void* out, void* stream);
int fdllm_forward_block_partial_batch(fdllm_ctx* ctx, int replace_position, const void* active_embed, int nseq,
                                      int rows, void* k_cache, void* v_cache, int cap, const int32_t* cache_offset,
                                      const int64_t* prefix_lens, void* out, void* stream);
/* build_prefix_cache (cuda.py:610-637) of sequence `seq` into its slice of a batched cache
 * [L, nseq, cap, nkv, hd]; the other sequences' rows are untouched. */
int fdllm_build_prefix_cache_seq(fdllm_ctx* ctx, const void* prefix_embed, int prefix_len, const float* prefix_bias,
                                 void* k_cache, void* v_cache, int cap, int nseq, int seq, void* stream);

/* Fused lm_head + confidence: the device restatement of get_confidence_m{rows}
 * (fast_dllm_relax/model/metal.py:505-528, dispatch runtime.py:136-174).  ids [rows] int32 = first
 * argmax of each row's logits; maxp [rows] fp32 = 1 / sum exp(logit - max).  Unshifted; the caller
 * applies the shift of runtime.py:172-174.  logits may be NULL, or [rows, vocab] fp32 to also receive
 * exactly what fdllm_get_logits returns. */
int fdllm_get_confidence(fdllm_ctx* ctx, const void* hidden, int rows, int32_t* ids, float* maxp, float* logits,
                         void* stream);

/* The same confidence of given fp32 logits [rows, ld] (the host reduction of runtime.py:176-181). */
int fdllm_confidence_from_logits(fdllm_ctx* ctx, const float* logits, int rows, int vocab, int ld, int32_t* ids,
                                 float* maxp, void* stream);

/* Threshold unmask of one sub-block on the device: the rule of fast_dllm_relax/runtime.py:794-805 (the
 * masked rows whose max probability is above `threshold`, else the first masked row of largest
 * probability) with the shift of runtime.py:172-174, replacing the host loop's per-step readback of the
 * confidence (runtime.py:179-181; device-confidence precedent model/metal.py:316-374).
 *   ids, maxp   [rows] unshifted confidence of one model call, as fdllm_get_confidence writes it.
 *   block       [bd_size] int32 ids of the active block (device); block rows [s0, s0 + sub_rows) are the
 *               sub-block, and block row s0 + r reads the shifted confidence row row0 + r (that is, the
 *               prediction of row row0 + r - 1; row 0 its own): row0 = s0 for a full 32-row step,
 *               0 for a partial step.  The selected rows are overwritten with their predicted ids.
 *   threshold   compared as `p > threshold` in fp32 (pass the fp32 rounding toward -inf of the host
 *               threshold to reproduce numpy's fp32-vs-Python-float comparison).
 *   report      optional int32 [4 + bd_size + 2 sub_rows + 4] (device memory, or host memory from
 *               fdllm_host_alloc that the host polls): word 0 = seq, written after everything else;
 *               1 = masked rows left in the sub-block; 2 = rows unmasked; 3 = unshifted argmax of the
 *               last confidence row (the append step's next token, runtime.py:360-363); 4.. = the block
 *               after the update; then the sub-block's shifted ids, their probabilities (fp32 bits), and
 *               the 64-bit masks of the rows that were masked and that were selected, each as a low and
 *               a high word (bit r: sub-block row r).
 * sub_rows = 0 updates nothing (an append step that only needs the report).  bd_size must be <= 64. */
int fdllm_unmask(fdllm_ctx* ctx, const int32_t* ids, const float* maxp, int rows, int row0, int32_t* block, int s0,
                 int sub_rows, int32_t mask_id, float threshold, int32_t* report, int32_t seq, void* stream);

/* The fused north-star head of one decode step: lm_head + max-softmax / first-argmax over the vocabulary
 * (fdllm_get_confidence) + the threshold unmask of fdllm_unmask, in two launches and without a
 * readback.  ids / maxp: optional (both or neither) [rows] outputs of the unshifted confidence. */
int fdllm_get_confidence_unmask(fdllm_ctx* ctx, const void* hidden, int rows, int row0, int32_t* block, int s0,
                                int sub_rows, int32_t mask_id, float threshold, int32_t* ids, float* maxp,
                                int32_t* report, int32_t seq, void* stream);

/* Pinned, device-mapped, coherent host memory for unmask reports (zeroed): the host polls what the
 * device writes there instead of waiting for a copy.  No reference counterpart (the reference reads
 * the confidence back with a blocking copy, runtime.py:179-181). */
int fdllm_host_alloc(size_t bytes, void** host_ptr, void** device_ptr);
void fdllm_host_free(void* host_ptr);

/* ---- a paged cache in 8 bits: no counterpart in the reference, whose caches are one contiguous allocation per
 * sequence in the model's dtype (inplace_bsnh_v1, export_utils.py:21-34).  For programs that keep their own projections
 * (as those of fdllm_kv_write / fdllm_attn_inplace) and many sequences of very different lengths.
 *
 * The cache of all layers: K [L, num_pages, nkv, page, 128] and V [L, num_pages, nkv, 128, page] in e4m3 (OCP; slots
 * innermost in V), 16-byte aligned, and one fp32 scale for each layer, page and kv head, k_scale / v_scale
 * [L, num_pages, nkv]: a byte stands for e4m3(byte) x scale, scales being 2^-100 or more.  page_size is 16, 32, 64 or
 * 128.
 * Position p of sequence b is slot p % page_size of page page_table[b, p / page_size] (int32 device
 * [nseq, pages_per_seq], row stride table_ld).  A page number outside [0, num_pages) is no page: nothing is written there,
 * and the attention leaves its keys out.
 *
 * The rows of a call (q, k, v, out [rows, heads, 128] in the context's dtype; heads contiguous, ld* elements from row to
 * row, multiples of 8, pointers 16-byte aligned) belong to nseq sequences: sequence b has rows [row_start[b],
 * row_start[b + 1]) (int32 device [nseq + 1], ascending; rows behind the last sequence's are neither read nor written),
 * at most max_rows of them (a bound: a launch has workgroups for max_rows rows of every sequence, so a tight one is faster,
 * and a call for more than a launch holds, some 10^8 rows, is refused); with row_start NULL each has max_rows rows and rows = nseq x max_rows.
 * Everything on the device may change between replays of a captured graph; the host arguments (rows, nseq, max_rows,
 * max_len) are what the launches are planned for.  Neither call needs bound weights, allocates or uses the context's
 * workspace. */
typedef struct fdllm_paged_cache {
  void *k, *v;
  float *k_scale, *v_scale;
  int32_t num_pages;
  int32_t page_size;
} fdllm_paged_cache;

/* Appends k / v [rows, nkv, 128] of `layer`, keys before their rotation: sequence b's rows go to positions start[b],
 * start[b] + 1, ... (int32 device [nseq]; a sequence with a negative start is skipped).  Row i of it is rotated by
 * position pos[b] + i (pos NULL: start): the pair (x[d], x[d + 64]) turns by position x rope_theta^(-d / 64) radians,
 * reduced in 64 bits: keys with sine, cosine and products in 64 bits, rounded once to fp32.  So are its queries, where q is
 * given, with sine, cosine and products in fp32: q [rows, nq, 128] into q_out (contiguous; may be q itself where q is),
 * rounded to the context's dtype.
 * Values are stored with one power-of-two scale for each page, kv head and tensor: the least 2^e, e >= -100, with
 * |x| <= 448 x 2^e for the page's new (finite) values.  live[b] (NULL: start) is the number of positions the sequence
 * holds before the call: if other rows of the page are among them they stay; the larger of the page's scale and the new
 * one is then taken, and where that is the new one they are encoded again with it.  Values that are not finite become
 * NaN.  The pages that a call writes must be distinct (pages that sequences share may only be read). */
int fdllm_paged_kv_append(fdllm_ctx* ctx, const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v,
                          int64_t ldv, int rows, const int32_t* row_start, int nseq, int max_rows,
                          const fdllm_paged_cache* cache, int layer, const int32_t* page_table, int pages_per_seq,
                          int64_t table_ld, const int32_t* start, const int32_t* live, const int32_t* pos, void* q_out,
                          void* stream);

/* out = softmax(q K^T / sqrt(128)) V over positions [0, kv_len[b]) (int32 device [nseq]; at most the table's
 * pages_per_seq x page_size) of `layer`, query head h on kv head h / (nq / nkv); q rotated already.  mask_block = 0: no
 * mask, as fdllm_attn_inplace; B > 0: the last row of sequence b is position kv_len[b] - 1, and a row at position p
 * attends positions below (p / B + 1) B (block-causal; 1: causal).  A row with nothing to attend gets zeros.
 * Values past the dtype's own range (fp16's 65504 is stored as 65536) count with their size: a row is infinite only where its
 * average is.
 * max_len: no kv_len is larger (0: the table's capacity); longer ones are attended in full, only less evenly split.
 * out may be q itself where q is contiguous.
 * workspace: fdllm_paged_attn_workspace bytes for the same arguments (may be 0), 16-byte aligned, used by this call until
 * it has run; calls that overlap need their own. */
size_t fdllm_paged_attn_workspace(const fdllm_ctx* ctx, int rows, int nseq, int max_rows, int page_size, int pages_per_seq,
                                  int64_t max_len);
int fdllm_paged_attn(fdllm_ctx* ctx, const void* q, int64_t ldq, int rows, const int32_t* row_start, int nseq,
                     int max_rows, const fdllm_paged_cache* cache, int layer, const int32_t* page_table,
                     int pages_per_seq, int64_t table_ld, const int32_t* kv_len, int64_t max_len, int mask_block,
                     void* out, void* workspace, size_t workspace_bytes, void* stream);

/* Log probabilities of given tokens from logits [rows, vocab] (the reference's loglikelihood reduction on the host,
 * runners.py:876-880: log-softmax, then a gather), with what a scoring or sampling program asks for beside them:
 *   logprob [rows]  log softmax(logits)[ids[r]]; 0 for ids[r] < 0 (a row without a token), NaN for ids[r] >= vocab.
 *                   ids NULL: none, logprob may be NULL
 *   entropy [rows]  -sum p log p
 *   top_ids, top_logprobs [rows, top_n]  the top_n (0 .. 32, at most vocab) most probable tokens, equal logits by
 *                   their index (a NaN logit counts as -inf in this order); may be NULL with top_n = 0
 * logits_type: FDLLM_DTYPE_BF16, FDLLM_DTYPE_F16 or FDLLM_LOGITS_F32; ld >= vocab elements from row to row; logits aligned to
 * their elements.  Any vocab >= 1, not only the context's.  A row with a NaN or +inf logit, or only -inf, has NaN log
 * probabilities and entropy.  workspace as for fdllm_paged_attn (8-byte aligned). */
#define FDLLM_LOGITS_F32 2
size_t fdllm_token_logprobs_workspace(const fdllm_ctx* ctx, int rows, int vocab, int top_n);
int fdllm_token_logprobs(fdllm_ctx* ctx, const void* logits, int logits_type, int rows, int vocab, int64_t ld,
                         const int32_t* ids, int top_n, float* logprob, float* entropy, int32_t* top_ids,
                         float* top_logprobs, void* workspace, size_t workspace_bytes, void* stream);

/* ---- heads normed and rotated, and a paged cache in 4 bits: no counterpart in the reference, whose rotation is inside its
 * compiled step (one layout, whole heads, one base) and whose caches are 16-bit.  For programs that keep their own
 * projections, as the calls above; like those these need no bound weights, allocate nothing and use none of the context's
 * workspace. */

/* How heads are rotated: the first `dim` (a multiple of 16, 0 .. 128) of a head's 128 dims, in pairs: pair j turns by
 * position x freq[j] radians (freq: HOST array of dim / 2, read during the call; at most 1000 in size) and is multiplied by
 * `factor`.  Pair j: dims (j, j + dim / 2), or (2 j, 2 j + 1) where interleaved is 1.  The other dims stay.  A null
 * fdllm_rotary is the model's own: dim 128 in halves, freq[j] = rope_theta^(-j / 64), factor 1. */
typedef struct fdllm_rotary {
  const double* freq;
  int32_t dim;
  int32_t interleaved;
  double factor;
} fdllm_rotary;

/* Heads of q [rows, nq, 128] and k [rows, nkv, 128] (either may be null) normed and rotated into q_out / k_out, as
 * fdllm_attn_inplace, fdllm_kv_write and fdllm_paged_attn take them.  With a norm's weights (128 of the context's dtype, the
 * same for every head; null: none) a head is x w / sqrt(mean x^2 + rms_norm_eps) first.  Row r is at position pos[r] (int32
 * device [rows]), or pos0 + r where pos is null.  Angles are reduced in 64 bits, the rest is fp32 (sums of squares 64 bits),
 * rounded once to the context's dtype.  ld*: elements from row to row (multiples of 8; pointers 16-byte aligned).  A result
 * may be its input (with the same row stride), but not overlap it otherwise. */
int fdllm_rotate_heads(fdllm_ctx* ctx, const void* q, int64_t ldq, const void* k, int64_t ldk, int rows, const int32_t* pos,
                       int64_t pos0, const fdllm_rotary* rotary, const void* q_norm, const void* k_norm, void* q_out,
                       int64_t ldqo, void* k_out, int64_t ldko, void* stream);

/* The 4-bit cache of all layers, 16-byte aligned: K and V [L, num_pages, nkv, page, 64] bytes of two e2m1 codes each (0, 0.5,
 * 1, 1.5, 2, 3, 4, 6; bit 3 the sign), the lower dim in the lower half.  K has one power of two for each block of 32 dims,
 * k_scale [L, num_pages, nkv, page / 16, 4, 4, 4] bytes of its exponent + 127 (255: NaN), at (slot / 16, slot % 4, block,
 * slot / 4 % 4); V one bf16 scale for each slot and head, v_scale [L, num_pages, nkv, page].  A key costs 134 bytes a kv head
 * and layer (256 in 8 bits, 512 in 16).  Page tables, rows and page sizes as for the 8-bit cache.  A row of the cache stands
 * by itself: it is written without reading what else its page holds, so the positions that one call writes must be distinct,
 * but their pages need not be.  Appends and reads are launched by `rows`: a loose max_rows costs them nothing. */
typedef struct fdllm_paged4_cache {
  void *k, *v;
  void *k_scale, *v_scale;
  int32_t num_pages;
  int32_t page_size;
} fdllm_paged4_cache;

/* Appends k / v [rows, nkv, 128] of `layer` at positions start[b], start[b] + 1, ... (int32 device [nseq]; a sequence with a
 * negative start is skipped, its queries too), keys normed and rotated on the way (rotary, norms as fdllm_rotate_heads; row i
 * of sequence b by position pos[b] + i, pos null: start; in 64 bits), and so the queries where given: q
 * [rows, nq, 128] into q_out (contiguous; may be q itself where q is), as fdllm_rotate_heads gives them.
 * Keys: the least 2^e, -60 <= e <= 125, with |x| <= 7 x 2^e for the block's values; values: a sixth of the row's largest,
 * rounded to bf16, at least 2^-60.  Codes are the nearest to x / scale, ties to the even one, at most 6 in size.  A value that
 * is not finite makes its block's (K) or its row's and head's (V) scale NaN. */
int fdllm_paged4_append(fdllm_ctx* ctx, const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v, int64_t ldv,
                        int rows, const int32_t* row_start, int nseq, int max_rows, const fdllm_paged4_cache* cache,
                        int layer, const int32_t* page_table, int pages_per_seq, int64_t table_ld, const int32_t* start,
                        const int32_t* pos, const fdllm_rotary* rotary, const void* q_norm, const void* k_norm, void* q_out,
                        void* stream);

/* Reads positions start[b], start[b] + 1, ... of `layer` back into k_out / v_out [rows, nkv, 128] (ldk, ldv elements from row
 * to row: a contiguous cache's rows will do), rounded once to the context's dtype.  A position in no page gives zeros (so
 * does a negative one); rows behind the last sequence's are left as they are. */
int fdllm_paged4_read(fdllm_ctx* ctx, const fdllm_paged4_cache* cache, int layer, const int32_t* page_table, int pages_per_seq,
                      int64_t table_ld, const int32_t* start, int rows, const int32_t* row_start, int nseq, int max_rows,
                      void* k_out, int64_t ldk, void* v_out, int64_t ldv, void* stream);

/* fdllm_paged_attn over a 4-bit cache: the same arguments, masks, lengths and workspace rules.  What a page holds behind
 * kv_len is never seen, whatever it is.  A query with a value that is not finite gives NaN.  V's scales may be any of the append's (2^-60
 * and more), negative, zero or smaller (a value of a row with a scale under 2^-60 may be taken as another of up to 6 x 2^-60 in size);
 * in a context of float16 one of more than 2^31 in size is NaN. */
size_t fdllm_paged4_attn_workspace(const fdllm_ctx* ctx, int rows, int nseq, int max_rows, int page_size, int pages_per_seq,
                                   int64_t max_len);
int fdllm_paged4_attn(fdllm_ctx* ctx, const void* q, int64_t ldq, int rows, const int32_t* row_start, int nseq,
                      int max_rows, const fdllm_paged4_cache* cache, int layer, const int32_t* page_table,
                      int pages_per_seq, int64_t table_ld, const int32_t* kv_len, int64_t max_len, int mask_block,
                      void* out, void* workspace, size_t workspace_bytes, void* stream);

/* Profiling hook; it has no counterpart in the reference.  Launches one operator of the cached step
 * `iters` times back to back on `stream`, reading and writing the context's own workspace (the values
 * are not meaningful); launch i uses layer (layer + i) % num_layers, as a step walks the layers, so a
 * benchmark can time one kernel with events on the stream it runs on without re-reading one layer's
 * weights from cache.  FDLLM_OP_ATTENTION attends rows [0, attend_len) of each layer of the caches. */
#define FDLLM_OP_QKV 0
#define FDLLM_OP_O_PROJ 1
#define FDLLM_OP_GATE_UP 2
#define FDLLM_OP_DOWN 3
#define FDLLM_OP_ATTENTION 4
#define FDLLM_OP_LM_HEAD_CONFIDENCE 5
int fdllm_bench_op(fdllm_ctx* ctx, int op, int rows, int layer, int iters, void* k_cache, void* v_cache, int cap,
                   int attend_len, void* stream);

/* Diagnostic; it has no counterpart in the reference.  Number of launches this context has run that
 * reduced their own splits (the down projection's k splits, the decode attention's key splits) instead of
 * handing them to a separate split-sum or merge launch.  Such a launch is planned when its whole grid is
 * resident at once (at most one workgroup per compute unit); FDLLM_GROUP_WAITS=0 at fdllm_create turns
 * it off, and so does a timed-out wait (reported by the next entry point as FDLLM_EHIP). */
long long fdllm_group_wait_launches(const fdllm_ctx* ctx);

/* Diagnostic; it has no counterpart in the reference.  Number of layer-loop calls (cached steps, short
 * stateless forwards) this context has run with the activations in MFMA-fragment order: calls of at
 * most 32 rows whose four projections all take the one-shot GEMM, unless FDLLM_XFRAG=0 was set when
 * the context was created.  Results are the same bit for bit either way. */
long long fdllm_frag_calls(const fdllm_ctx* ctx);

/* Message of this thread's last failure ("" if none). */
const char* fdllm_last_error(void);

#ifdef __cplusplus
}
#endif

#endif /* FDLLM_H */
