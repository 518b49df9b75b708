/*
 * seedplane_cuda.h -- C ABI of the B200 (sm_100a) Qwen2 decode engine.
 *
 * This is the native boundary that replaces SeedPlane's Vulkan runtime (`qwen_vk`), which the
 * reference drives through a JSON-lines subprocess (seedplane/native.py:25-90 ->
 * native/vulkan_decode/qwen_vk.cpp:810-855). Plain pointers and sizes only; no C++ or torch types.
 *
 * Conventions
 *   - Every entry point returns 0 (SP_OK) or a negative SP_ERR_* code; the message of the last
 *     failure on the calling thread is sp_last_error(). Nothing calls exit() or throws across the
 *     ABI (the reference aborted the process on Vulkan errors, qwen_vk.cpp:52-53).
 *   - "dev" pointers are CUDA device pointers on the engine's device; "host" pointers are host
 *     memory. Token ids and positions are int32, logits fp32.
 *   - Work is queued on the caller's stream (`stream`, a cudaStream_t; NULL = legacy default
 *     stream). No call synchronizes the device except where documented.
 *   - One engine per device. Calls on one engine come from one host thread at a time.
 *     Engines on different devices are independent and may run concurrently.
 */
#ifndef SEEDPLANE_CUDA_H
#define SEEDPLANE_CUDA_H

#include <stdint.h>
#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

#define SP_OK               0
#define SP_ERR_INVALID     -1   /* bad argument, shape or layout */
#define SP_ERR_CUDA        -2   /* a CUDA runtime call failed (message names it) */
#define SP_ERR_CAPACITY    -3   /* KV cache / position / node limit exceeded */
#define SP_ERR_UNSUPPORTED -4   /* shape not supported by the kernels */
#define SP_ERR_DEVICE      -5   /* a kernel reported an error status (bounded wait, bad index) */

#define SP_F32              0   /* value types of the paged operators and of logits              */
#define SP_F16              1
#define SP_BF16             2

#define SP_WEIGHTS_F16       0  /* fp16 matrices (seedplane-bundle/2 layout)                    */
#define SP_WEIGHTS_I8_B32    1  /* int8 matrices + one fp16 scale per 32 inputs along K          */

/* Architecture. Mirrors the `arch` block of a seedplane-bundle/2 manifest
 * (seedplane/native_bundle.py:129-131) and Qwen2Engine's config reads (qwen_engine.py:44-53). */
typedef struct sp_config {
    int32_t layers, hidden, heads, kv_heads, head_dim, intermediate, vocab;
    int32_t max_positions;     /* RoPE table length (positions are original position ids)      */
    float   rope_theta, rms_norm_eps;
    int32_t tied_embeddings;   /* 1: LM head = embedding matrix                                 */
    int32_t weight_format;     /* SP_WEIGHTS_*                                                  */
} sp_config;

/* One layer's tensors, device pointers in the bundle-v2 layouts (native_bundle.py:112-120):
 * row-major [out, in]. qkv_w rows are q (heads*head_dim), then k, then v (kv_heads*head_dim each).
 * For SP_WEIGHTS_I8_B32 every matrix is int8 and its `_s` pointer holds fp16 scales
 * [out, in/32]; for SP_WEIGHTS_F16 the `_s` pointers are ignored. */
typedef struct sp_layer_weights {
    const void *qkv_w, *qkv_s;   const float *qkv_b;
    const void *o_w, *o_s;
    const void *gate_w, *gate_s;
    const void *up_w, *up_s;
    const void *down_w, *down_s;
    const float *in_norm, *post_norm;
} sp_layer_weights;

typedef struct sp_weights {
    const void *embed;                 /* [vocab, hidden] fp16, device                          */
    const void *lm_head, *lm_head_s;   /* untied head (fp16, or int8 + scales); NULL when tied  */
    const float *final_norm;           /* [hidden] fp32, device                                 */
    const sp_layer_weights *layers;    /* HOST array of `layers` entries                        */
    const float *rope_host;            /* optional HOST table [max_positions][head_dim/2][2] of
                                          (cos, sin) fp32; NULL = computed in double precision  */
} sp_weights;

typedef struct sp_engine sp_engine;
typedef struct sp_kv sp_kv;

/* Last error message of the calling thread ("" if none). */
const char *sp_last_error(void);
/* Library version string. */
const char *sp_version(void);

/* Create an engine on `device`. The library copies the weights into its own arena in the packed
 * layouts its kernels stream (the caller may free its copies on return) and owns all workspace.
 * Replaces qwen_vk's Engine::init (qwen_vk.cpp:283-342). Synchronizes the device. */
int sp_engine_create(const sp_config *cfg, const sp_weights *w, int device, sp_engine **out);
void sp_engine_destroy(sp_engine *e);
/* Bytes of device memory the engine holds (weights arena + workspace). */
int64_t sp_engine_device_bytes(const sp_engine *e);

/* KV cache of `capacity` slots, fp16 [layers][kv_heads][capacity][head_dim] for K and for V.
 * Replaces KVCache.allocate / Qwen2Engine.new_cache (qwen_engine.py:18-29,82-85). */
int sp_kv_create(sp_engine *e, int32_t capacity, sp_kv **out);
void sp_kv_destroy(sp_kv *kv);
int32_t sp_kv_length(const sp_kv *kv);
int32_t sp_kv_capacity(const sp_kv *kv);
/* Truncate (rollback) the committed length, like `cache.length = n` in the reference's linear
 * verifier (experiments/hive_scaling/benchmark_speculative.py:119,127). */
int sp_kv_set_length(sp_kv *kv, int32_t length);

/* Run `n` tokens through the model at cache slots [len, len+n), exactly Qwen2Engine.forward
 * (qwen_engine.py:105-144): tokens_dev[n] int32, positions_dev[n] int32 RoPE positions (NULL =
 * the slots). Token i attends to slots [0, len+i]. Advances the cache length by n.
 * all_logits = 0: logits_dev NULL or fp32 [vocab] of the last token; argmax_dev NULL or int32 [n],
 *   the greedy token after each input token (lowest index on ties).
 * all_logits = 1: logits_dev fp32 [n][vocab] and argmax_dev [n] for every token.
 * all_logits = 2: the last token only (a prompt whose other tokens only fill the cache): logits_dev
 *   [vocab], argmax_dev[0]; the batched pass runs the LM head for that one token. */
int sp_forward(sp_engine *e, sp_kv *kv, const int32_t *tokens_dev, const int32_t *positions_dev,
               int32_t n, float *logits_dev, int32_t all_logits, int32_t *argmax_dev, void *stream);

/* Greedy decode: feed `token` at position `pos` (slot = current length), then feed back each
 * argmax on the device, for `n_steps` steps without host round trips. out_tokens_dev[n_steps]
 * receives the argmax of every step (out[i] is fed at step i+1). logits_dev: NULL or fp32
 * [vocab] = logits of the last step. Advances the cache length by n_steps. Replaces qwen_vk's
 * per-token Session::step + argmax loop (qwen_vk.cpp:519-565,588-613). */
int sp_decode(sp_engine *e, sp_kv *kv, int32_t token, int32_t pos, int32_t n_steps,
              int32_t *out_tokens_dev, float *logits_dev, void *stream);

/* Greedy decode of B independent requests in one batched pass per step (runtime request batching;
 * the reference has none: README.md:67-68, its HIVE agents report batch_size 1, hive/pool.py:465-466).
 * Request b feeds tokens_host[b] at RoPE position positions_host[b] into its own cache kvs[b] (slot =
 * that cache's length, attention over that cache alone), then each step's argmax is fed back on the
 * device for n_steps steps; the weights are streamed once per step for all B requests.
 * out_tokens_dev[n_steps][B] receives every step's argmaxes (row i = the tokens after step i).
 * 1 <= B <= 64, distinct caches of this engine, each with room for n_steps more slots. Advances every
 * cache's length by n_steps. Replaces, for a batch, B calls of sp_decode (the reference's per-request
 * Session::step loop, qwen_vk.cpp:519-565,588-613). */
int sp_decode_batch(sp_engine *e, sp_kv *const *kvs, int32_t B, const int32_t *tokens_host,
                    const int32_t *positions_host, int32_t n_steps, int32_t *out_tokens_dev, void *stream);

/* The prompts of B independent requests in packed batched passes (runtime request batching; see
 * sp_decode_batch): request b appends lens_host[b] tokens (tokens_dev holds the B prompts one after
 * another) to its own cache kvs[b] at slots len .. len + lens_host[b] - 1, RoPE positions = the slots,
 * every token attending to its own cache up to itself. argmax_dev[B]: the greedy token after each
 * prompt's last token (the LM head runs for those rows only). Whole prompts are packed into passes
 * of at most 512 tokens; a longer prompt runs alone through the chunked pass. 1 <= B <= 256,
 * distinct caches of this engine. Advances every cache's length by its prompt's length. Replaces,
 * for a batch, B prompt calls of sp_forward (Qwen2Engine.forward(prompt), qwen_engine.py:105-144). */
int sp_prefill_batch(sp_engine *e, sp_kv *const *kvs, int32_t B, const int32_t *tokens_dev, const int32_t *lens_host,
                     int32_t *argmax_dev, void *stream);

/* Speculative tree verification (no counterpart kernel in the reference; semantics of
 * seedplane/speculative.py:55-92). n nodes in an ancestor-closed order (parent index < own index;
 * -1 = child of the committed prefix). Node i is written to scratch slot len+i at RoPE position
 * base_pos + depth_i - 1 and attends to the committed slots [0, len) and to its ancestors and
 * itself. The cache length is NOT advanced (see sp_kv_commit).
 * argmax_dev[n]: target argmax after each node. logits_dev: NULL or fp32 [n][vocab]. */
int sp_verify_tree(sp_engine *e, sp_kv *kv, const int32_t *tokens_host, const int32_t *parents_host,
                   int32_t n, int32_t base_pos, float *logits_dev, int32_t *argmax_dev, void *stream);

/* Move the K/V of accepted scratch slots into place: for i < n, slot src_slots_host[i] is copied
 * to slot len+i of every layer, then the length becomes len+n. Replaces the reference's KV
 * rollback by truncation (benchmark_speculative.py:119,127) for tree-shaped drafts. */
int sp_kv_commit(sp_kv *kv, const int32_t *src_slots_host, int32_t n, void *stream);

/* Copy the K/V of n consecutive slots, every layer and kv head, from src slots [src_slot0,
 * src_slot0 + n) to dst slots [dst_slot0, dst_slot0 + n). The caches belong to one engine; they may
 * differ in capacity, or be the same cache with disjoint ranges. Lengths are not changed. Replaces
 * the native session's Engine::copy_slots (native/vulkan_decode/qwen_vk.cpp:440-453): a shard
 * window is seeded with the sink tokens' K/V and, in the approximate reuse mode, the halo's
 * (qwen_vk.cpp:512-542). */
int sp_kv_copy(sp_kv *src, int32_t src_slot0, sp_kv *dst, int32_t dst_slot0, int32_t n, void *stream);

/* Greedy argmax of each row of fp32 logits [rows][ld] (device) over the first `cols` columns:
 * argmax_dev[rows] int32, lowest index on ties (NaN is never selected). For logits produced
 * outside the fused LM head, e.g. all-logits verification. Replaces `Qwen2Engine.sample`
 * (qwen_engine.py:147-148) and argmax.comp:8-22. Uses the engine's scratch: calls on one engine
 * are ordered by their stream (one stream per engine). */
int sp_argmax(sp_engine *e, const float *logits_dev, int32_t rows, int32_t cols, int64_t ld, int32_t *argmax_dev,
              void *stream);

/* Per-row top-k of fp32 logits, k in 1..8: indices and values [rows][k] ordered by larger value,
 * lower index on ties (the greedy argmax's rule), and each row's log-sum-exp, so log-probabilities
 * are val - lse. Replaces the drafter-side `torch.topk` + `log_softmax` a tree drafter needs; the
 * reference has no drafter tree (seedplane/speculative.py:18-43 takes given branches). */
int sp_topk(sp_engine *e, const float *logits_dev, int32_t rows, int32_t cols, int64_t ld, int32_t k,
            int32_t *idx_dev, float *val_dev, float *lse_dev, void *stream);

/* Greedy acceptance of a verified draft tree on the device (replaces the selection loop of
 * seedplane/speculative.py:55-92, verify_greedy, fed by one batched pass instead of per-prefix target
 * calls). node_pred_dev: int32 [n] on the engine's device, the target's argmax after each node (the
 * argmax output of sp_verify_tree); root_pred: its argmax after the committed prefix. tokens /
 * parents (host, parents[i] < i, -1 = child of the prefix); path_ends (host, [n_paths]): the last
 * node of each draft branch in input order. Each branch is walked from its root while the target
 * agrees; the first disagreement emits the target's token and rejects the branch; the chosen
 * branch has the most accepted draft tokens, then the most emitted tokens, then the earliest input
 * position; no paths: the one token root_pred. out_host [2n + 5]: emitted count, accepted count,
 * chosen branch (-1: none), the target's token after a fully accepted branch (else -1), emitted
 * tokens [n + 1], accepted node indices [n]. n <= 64, n_paths <= 1024. Synchronises `stream`. */
int sp_accept_greedy(sp_engine *e, const int32_t *node_pred_dev, int32_t root_pred, const int32_t *tokens_host,
                     const int32_t *parents_host, int32_t n, const int32_t *path_ends_host, int32_t n_paths,
                     int32_t *out_host, void *stream);

/* Stochastic acceptance of a draft tree at `temperature` with a counter-based RNG (seed, counter):
 * recursive rejection sampling (children tried in node order, accept with min(1, p/q), residual
 * max(p - q, 0) after a rejection, a draw from the residual when every child is rejected). The
 * reference has no stochastic verifier (seedplane/speculative.py:46-92 is greedy only); the rule
 * and its fp64 arithmetic are restated bit for bit in the repository's CPU oracle.
 * target_logits / draft_logits: device fp32 [n + 1][ld], row 0 = after the committed prefix,
 * row i + 1 = after node i. tokens / parents (host, parents[i] < i, -1 = root child). out_host
 * [2n + 3]: emitted count, accepted count, emitted tokens [n + 1], accepted node indices [n].
 * Synchronises `stream`. */
int sp_accept_stochastic(sp_engine *e, const float *target_logits_dev, const float *draft_logits_dev, int64_t ld,
                         int32_t vocab, const int32_t *tokens_host, const int32_t *parents_host, int32_t n,
                         double temperature, uint64_t seed, uint64_t counter, int32_t *out_host, void *stream);

/* The batched pass's projection on its own: y[t][n] = alpha * W[n, :] . (x[t] + x[lo_row0 + t]),
 * t < t, n < n, over k inputs, on the tcgen05 multi-column GEMM of the engine's device (no reference
 * counterpart: it is the contraction under sp_forward's prompt chunks and sp_verify_tree, which
 * replace qwen_vk.cpp:417-436's gemm_b.comp batch and speculative.py:55-92's per-prefix target calls;
 * exposed for callers and tests of that contraction). W: row-major fp16 [n, k] (w_lo_dev: optional
 * second fp16 half, W = w + w_lo); x: fp16 rows [x_rows, k], token t's hi half at row t, its lo
 * half at row lo_row0 + t. mode 0: y[t * ldy + n] = ...; 1: y[t * ldy + n] += ...; 2 (SwiGLU): rows
 * 2i, 2i + 1 are gate i, up i, and a = SiLU(gate) * up goes to act_hi[t * ld_act + i] = fp16(a),
 * act_lo[...] = fp16(a - hi). t <= 512; k a multiple of 8; the engine's GEMM workspace is used,
 * so calls on one engine are ordered on one stream. */
int sp_mcol_gemm(sp_engine *e, int32_t mode, const void *w_dev, const void *w_lo_dev, float alpha, int32_t n, int32_t k,
                 const void *x_dev, int32_t x_rows, int32_t lo_row0, int32_t t, float *y_dev, int32_t ldy,
                 void *act_hi_dev, void *act_lo_dev, int32_t ld_act, void *stream);

/* Top-k / top-p filter of one logits row before a draw (replaces the masking steps of
 * seedplane/qwen_engine.py:147-156, Qwen2Engine.sample): z_dev[j] = logits_dev[j] / temperature
 * (fp32); then, if top_k > 0, -inf below the top_k-th largest z (ties at the cut kept); then, if
 * top_p < 1, -inf for every entry whose preceding probability mass in descending order (softmax
 * over the entries still kept) exceeds top_p (a group of equal values at the cut is kept whole).
 * Draw from z_dev with sp_accept_stochastic (n = 0, temperature 1). One launch of one CTA on
 * `stream`, no engine, no allocation. vocab in [1, 524288], temperature > 0, top_k >= 0,
 * top_p in [0, 1], else SP_ERR_INVALID. */
int sp_sample_filter(const float *logits_dev, int32_t vocab, double temperature, int32_t top_k, double top_p,
                     float *z_dev, void *stream);

/* ---- K / V in pages shared by requests (runtime request batching after a common prefix) --------
 * No reference counterpart: the reference keeps one contiguous cache per session
 * (seedplane/qwen_engine.py:18-29) and decodes requests one at a time (README.md:67-68).
 *
 * One layer's pages. K (and V) of kv head g at slot j of page p is the head_dim elements at
 * p * page_stride + g * head_stride + j * slot_stride (elements; multiples of 8, and k_dev, v_dev
 * 16-byte aligned). head_dim 64 or 128, dtype SP_F16 or SP_BF16, any page_size >= 1.
 * status_dev: int32 on the device, or NULL. A kernel that meets a bad page number, length or
 * position stores 3 there (an expired wait inside a kernel: 1) and goes on: slots it cannot reach are not
 * written, and read as zeros. */
typedef struct sp_pages {
    void *k_dev, *v_dev;
    int64_t page_stride, head_stride, slot_stride;
    int32_t n_pages, page_size, kv_heads, head_dim, dtype;
    int32_t *status_dev;
} sp_pages;

/* A ragged batch over pages. Request b's tokens of this call are the rows q_start[b] ..
 * q_start[b + 1] - 1 of the call's matrices (q_start int32 [batch + 1], q_start[0] = 0; NULL: max_q
 * rows each; a request may have none). lens[b]: its own keys, these tokens among them, which are the
 * last: token i has own key lens[b] - q_len + i. Own key j is slot j % page_size of page
 * tables[b * table_stride + j / page_size]. Before its own keys every request sees the shared prefix:
 * keys [0, prefix_len) in the pages of prefix_dev, in order. The arrays are device memory and are read
 * by the kernels, so a captured graph serves new contents; the sizes are the host's: `tokens` rows at
 * most (rows at and behind q_start[batch] are neither read nor written), max_q rows of one request at
 * most. */
typedef struct sp_page_batch {
    int32_t batch, tokens, max_q;
    const int32_t *q_start_dev, *lens_dev, *tables_dev;
    int64_t table_stride;
    int32_t table_width;
    const int32_t *prefix_dev;
    int32_t prefix_len;
} sp_page_batch;

/* Append a pass's keys and values to their pages with the position rotation on the way. x =
 * qkv row + bias (bias fp32 [(heads + 2 kv_heads) * head_dim] or NULL); row = q heads, then k, then v
 * (the fused QKV order of sp_layer_weights), row_stride elements apart. Of every q and k head the
 * first rot_dim dims (even, <= head_dim) are rotated in pairs (a, b) -> (a c - b s, b c + a s), pairs
 * (j, j + rot_dim / 2) or, `interleaved`, (2j, 2j + 1); (c, s) = rope_dev[pos][j], fp32
 * [rope_positions][rot_dim / 2][2] (sp_weights.rope_host's layout; a scaled table gives scaled
 * positions). pos = positions_dev[row], or prefix_len + own key when NULL. q goes to q_out [row][heads
 * * head_dim] (q_stride elements apart) in the rows' type; k and v are rounded to the cache's type.
 * dtype: SP_F32 (either cache type), or the cache's own type. All arithmetic is fp32. `device`: the
 * device of every pointer; the calling thread's current device is put back. Nothing is allocated;
 * the call can be captured into a graph. */
int sp_pages_append(int device, const sp_pages *pages, const sp_page_batch *batch, int32_t heads, const void *qkv_dev,
                    int32_t dtype, int64_t row_stride, const float *bias_dev, const float *rope_dev,
                    int32_t rope_positions, int32_t rot_dim, int32_t interleaved, const int32_t *positions_dev,
                    void *q_out_dev, int64_t q_stride, void *stream);

/* Bytes of workspace sp_pages_attention needs for these sizes (0 is possible), or SP_ERR_*. */
int64_t sp_pages_attention_workspace(const sp_pages *pages, const sp_page_batch *batch, int32_t heads, int32_t dtype);

/* Attention of a batch whose requests share a prefix: out[row] = softmax(scale * q . K) V over the
 * prefix's keys and the request's own keys up to the row's own; the prefix's pages are read once for
 * the whole batch. q, out: [row][heads * head_dim], q_stride / out_stride elements apart (multiples of
 * 8, 16-byte aligned). dtype of q and out: SP_F32 over SP_F16 pages (scores and values then carry the
 * queries and probabilities as two fp16 halves: 2^-22 of each, and of a query 2^-39 of its row's
 * largest), or the pages' own type (probabilities rounded to it; sums, maxima and outputs fp32, rounded
 * once). Over SP_F16 pages a probability is off by 2^-36 (fp32 queries) or 2^-32 of the row's largest
 * besides, fp16's least steps. q . K must stay within fp32's range. fp32 queries: the products'
 * accumulators cut off 2^-23 of a sum for 16 keys at most, over ranges of 4,096 keys; a prefix (or a
 * request) of more than 131,072 keys is cut into 32 ranges, and the error grows with them. A row that
 * sees no key gives zeros. Slots that hold no key may hold anything; the values of keys that another row
 * of the request sees must be finite.
 * lse_dev: NULL or fp32 [row][heads], the log-sum-exp of the scaled scores (-inf for such a row).
 * workspace_dev: as many bytes as sp_pages_attention_workspace says, 16-byte aligned, contents free,
 * not shared by calls that may overlap in time. Can be captured into a graph. */
int sp_pages_attention(int device, const sp_pages *pages, const sp_page_batch *batch, int32_t heads, const void *q_dev,
                       int32_t dtype, int64_t q_stride, float scale, void *out_dev, int64_t out_stride, float *lse_dev,
                       void *workspace_dev, int64_t workspace_bytes, void *stream);

/* One packed pass of a ragged batch through the model over pages: row i of the batch is token
 * tokens_dev[i] (int32, on the engine's device), its K / V go to its request's pages (sp_pages_append) and it
 * attends to the shared prefix and its request's own keys (sp_pages_attention), at RoPE position
 * prefix_len + own key. layer_pages: HOST array of the engine's `layers` entries, SP_F16, with the engine's
 * kv_heads and head_dim (their status_dev is not used: sp_device_status reports). argmax_dev int32 [batch]:
 * the greedy token after each request's last row; logits_dev: NULL or fp32 [batch][vocab]. Every request
 * has at least one row; batch 1 .. 256, tokens 1 .. 512 (and exactly q_start[batch]). Like sp_prefill_batch
 * and sp_decode_batch, for caches that share a prefix. The engine's workspace is used, and grows with the
 * passes: a stream that is being captured is refused. */
int sp_forward_pages(sp_engine *e, const sp_pages *layer_pages, const sp_page_batch *batch, const int32_t *tokens_dev,
                     float *logits_dev, int32_t *argmax_dev, void *stream);

/* Greedy decode of a batch over pages, fed back on the device: n_steps passes of one row per request. On
 * entry tokens_dev[batch] (int32, device) holds each request's next token and lens_dev its own keys so far;
 * every step appends the token (lens_dev[b] += 1) and replaces it by its argmax, also stored at
 * out_tokens_dev[step][batch]. batch->lens_dev and tokens_dev are written; batch->q_start_dev must be NULL,
 * max_q 1, tokens = batch <= 64; the tables must have room for the steps. */
int sp_decode_pages(sp_engine *e, const sp_pages *layer_pages, const sp_page_batch *batch, int32_t *tokens_dev,
                    int32_t n_steps, int32_t *out_tokens_dev, void *stream);

/* Bytes of workspace sp_accept_chains needs, or SP_ERR_*. */
int64_t sp_accept_chains_workspace(int32_t batch, int32_t drafts, int32_t vocab);

/* Verification of every request's chain of drafted tokens with given random numbers, a whole batch in
 * one call and without a synchronisation (sp_accept_stochastic: one request's tree, its own random
 * numbers, on the host's time; the reference verifies greedily, seedplane/speculative.py:55-92).
 * Request b drafted tokens_dev[b][0 .. n), n = counts_dev[b] (NULL: all `drafts`). With p_i =
 * softmax(target row i / T_b) and q_i = softmax(draft row i / T_b) (draft_dev NULL: the drafter is
 * certain, q_i = 1 at its token), draft i is accepted when u[b][i] * q_i(x_i) < p_i(x_i). After the
 * first refusal i the next token is drawn from max(p_i - q_i, 0), or from p_i where that is zero
 * everywhere; after n acceptances from p_n. A draw from weights r is the first index whose running
 * sum exceeds u[b][drafts] * (their sum). T_b = temperature_dev[b] (fp32; NULL: 1); T_b <= 0 or NaN: greedy,
 * p_i is 1 at the row's first maximum. NaN logits weigh nothing, nor do those below 2^-1000 of the row's
 * largest; a row without a finite or +inf logit accepts nothing and draws -1; a drafted token outside [0, vocab)
 * is refused.
 * target_dev: [b][drafts + 1][vocab], rows target_ld and requests target_bs elements apart; draft_dev:
 * [b][drafts][vocab], draft_ld, draft_bs; dtype SP_F32, SP_F16 or SP_BF16; u_dev fp64 [b][drafts + 1] in
 * [0, 1). out_tokens_dev int32 [b][drafts + 1]: the accepted tokens, the drawn one, then -1;
 * accepted_dev int32 [b]. drafts 0 .. 64 (0: a draw for every request). What is decided is decided in fp64: the
 * fp32 sums of the one pass over the logits settle only the drafts that they cannot be wrong about. workspace_dev as
 * above. */
int sp_accept_chains(int device, int32_t batch, int32_t drafts, int32_t vocab, const void *target_dev, int64_t target_bs,
                     int64_t target_ld, const void *draft_dev, int64_t draft_bs, int64_t draft_ld, int32_t dtype,
                     const int32_t *tokens_dev, const int32_t *counts_dev, const double *u_dev,
                     const float *temperature_dev, int32_t *out_tokens_dev, int32_t *accepted_dev, void *workspace_dev,
                     int64_t workspace_bytes, void *stream);

/* sp_argmax without an engine and without any allocation (no reference counterpart: the
 * reference allocates nothing on this path; this entry point exists for callers that must not
 * allocate device memory, e.g. inside a memory-capped serving process or before an engine
 * exists). Same result as sp_argmax. Runs on `device` and sets the calling thread's current
 * device back to what it was before returning; logits_dev and argmax_dev must be device memory
 * of `device` (else SP_ERR_INVALID). Its scratch is a fixed 33,280-byte __device__ array of the
 * library (one per device), so:
 *   - rows <= 128, else SP_ERR_CAPACITY (nothing is launched);
 *   - it clears the row counters it uses (a memset on `stream`) before each launch;
 *   - calls that overlap in time on one device (different streams or threads) race on the same
 *     scratch: order them on one stream;
 *   - the first call on a device looks the scratch up (cudaGetSymbolAddress): make it before any
 *     stream capture. The address is kept for the life of the device's primary context; a
 *     process that resets the device (cudaDeviceReset) must not call this entry point again. */
int sp_argmax_noalloc(int device, const float *logits_dev, int32_t rows, int32_t cols, int64_t ld,
                      int32_t *argmax_dev, void *stream);

/* Kernel timeline of the last step, when the engine was created with SEEDPLANE_TRACE=1: for each
 * GEMV of the step (4 per layer, then the LM head) and each CTA, kernel-start / dependency-wait /
 * prologue / stream / epilogue stamps and per-unit issue and ready stamps of %globaltimer (ns).
 * host_out NULL: returns the number of 64-bit words; else copies them (synchronizes the device)
 * and returns the count. Returns 0 when tracing is off. With SEEDPLANE_MCOL_TRACE=1 (and no step
 * trace) it returns the last sp_mcol_gemm launch's per-CTA phase stamps instead (16 words per CTA,
 * 148 CTAs). The reference had no GPU timestamps
 * (experiments/v18/RESULTS.md:29-30). */
int64_t sp_trace_read(sp_engine *e, uint64_t *host_out, int64_t capacity);

/* Wait for `stream`, then report (and clear) a device-side error status recorded by a kernel since
 * the last call: SP_ERR_DEVICE with a message, or SP_OK. Kernels never trap; a bad token id, an
 * out-of-table position or an expired bounded wait is recorded here instead. */
int sp_device_status(sp_engine *e, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* SEEDPLANE_CUDA_H */
