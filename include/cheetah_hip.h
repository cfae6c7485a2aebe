/*
 * cheetah_hip.h — C-ABI of the MI355X (gfx950) decoder-forward backend for
 * Cheetah's `ModelForward` boundary (CHEETAH_DEVICE=hip).
 *
 * Conventions follow the reference's device C-ABI (cheetah_vulkan.h):
 *  - int status: 0 on success, -1 on failure; the failure sentence is kept
 *    per thread and read with cheetah_hip_last_error() (the Rust wrapper maps
 *    it to Err(String), as src/native.rs:1860-1870 does for Vulkan);
 *  - caller-owned output buffers, plain pointers and sizes, opaque handles;
 *  - every argument error is rejected before any device work.
 *
 * Pointers documented as "device" point to memory from cheetah_hip_alloc();
 * everything else is host memory.
 */
#ifndef CHEETAH_HIP_H
#define CHEETAH_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ------------------------------------------------------------------------
 * Lifecycle. Replaces init_vulkan_device / shutdown_vulkan_device
 * (cheetah_vulkan.h:15-16). Fails on anything but a gfx950 device.
 * ---------------------------------------------------------------------- */
int cheetah_hip_init(int device);
void cheetah_hip_shutdown(void);
/* Backend label for the banner (registry.rs:62 ModelForward::device_name). */
const char *cheetah_hip_device_name(void);
const char *cheetah_hip_last_error(void);

/* ------------------------------------------------------------------------
 * Device memory. Replaces vk_alloc_vram / vk_free_vram
 * (cheetah_vulkan.h:22-23). All copies are synchronous.
 * ---------------------------------------------------------------------- */
void *cheetah_hip_alloc(size_t bytes);
int cheetah_hip_free(void *device_ptr);
int cheetah_hip_upload(void *device_dst, const void *host_src, size_t bytes);
int cheetah_hip_download(void *host_dst, const void *device_src, size_t bytes);
/* Device-to-device copy. No counterpart in the reference; measurement
 * helper (the plain copy whose byte counters calibrate the HBM traffic of
 * the other kernels). */
int cheetah_hip_copy(void *device_dst, const void *device_src, size_t bytes);
int cheetah_hip_synchronize(void);

/* ------------------------------------------------------------------------
 * Op-level entry points (device pointers; run on the library stream and
 * return after the work is queued — call cheetah_hip_synchronize() or a
 * download before reading results).
 *
 * Weight layouts are the reference's own:
 *  - BF16: row-major [rows][cols] uint16 bits;
 *  - Q8:  rows f32 row scales, then rows payload rows of (cols+3)/4*4 int8
 *         codes (src/chat/precision/q8.rs:1-25);
 *  - Q4:  rows f32 row scales, then rows payload rows of
 *         ceil(ceil((cols+1)/2)/4)*4 bytes, two int4 codes per byte, low
 *         nibble = even column (src/chat/precision/q4.rs:1-52).
 * ---------------------------------------------------------------------- */

/* y[rows] = W[rows, cols] · x[cols]. Replaces gemv (ops.rs:246), gemv_q8
 * (ops.rs:544), gemv_q4 (ops.rs:586) and the resident Vulkan matmuls
 * (vk_matmul_{bf16,q8,q4}_transposed_resident_checked, native.rs:987-1030). */
int cheetah_hip_gemv_bf16(const uint16_t *w, size_t rows, size_t cols, const float *x, float *y);
int cheetah_hip_gemv_q8(const uint8_t *w, size_t rows, size_t cols, const float *x, float *y);
int cheetah_hip_gemv_q4(const uint8_t *w, size_t rows, size_t cols, const float *x, float *y);

/* Y[n, rows] = X[n, cols] · Wᵀ. Replaces gemm (ops.rs:308) and the
 * per-row quantized linear_batch loop (ops.rs:1244-1326). */
int cheetah_hip_gemm_bf16(const uint16_t *w, size_t rows, size_t cols, const float *x, size_t n, float *y);
int cheetah_hip_gemm_q8(const uint8_t *w, size_t rows, size_t cols, const float *x, size_t n, float *y);
int cheetah_hip_gemm_q4(const uint8_t *w, size_t rows, size_t cols, const float *x, size_t n, float *y);

/* Row-wise quantization of a BF16 matrix into the reference layouts,
 * bit-exact to q8::quantize (q8.rs:91-125) / q4::quantize (q4.rs:126-161).
 * out_len must equal the layout's byte length. */
size_t cheetah_hip_q8_buffer_bytes(size_t rows, size_t cols);
size_t cheetah_hip_q4_buffer_bytes(size_t rows, size_t cols);
int cheetah_hip_quantize_q8(const uint16_t *w_bf16, size_t rows, size_t cols, uint8_t *out, size_t out_len);
int cheetah_hip_quantize_q4(const uint16_t *w_bf16, size_t rows, size_t cols, uint8_t *out, size_t out_len);
/* out[rows, cols] = scale[row] * code[row, col] (Q8Matrix/Q4Matrix::
 * dequant_value, q8.rs / q4.rs:101-110): the in-register dequantization
 * the GEMV/GEMM kernels use, written out for bit-exact checks. */
int cheetah_hip_dequant_q8(const uint8_t *w, size_t rows, size_t cols, float *out);
int cheetah_hip_dequant_q4(const uint8_t *w, size_t rows, size_t cols, float *out);

/* Paged BF16 KV cache view. K and V pools are
 * [pages][kv_heads][page_size][head_dim] BF16; page_table maps logical page
 * (position / page_size) to a physical page (device int32). */
typedef struct cheetah_hip_kv_view {
    const uint16_t *k_pages;
    const uint16_t *v_pages;
    const int32_t *page_table;
    uint32_t page_size;
    uint32_t kv_heads;
    uint32_t head_dim;
} cheetah_hip_kv_view;

/* GQA causal attention (ops.rs:1357-1467 attention / attention_head) for
 * `rows` query rows at absolute positions offset .. offset+rows-1; query row
 * i attends to cached positions [0, offset+i] (their K/V already in the
 * cache). q: device f32 [rows][q_heads*head_dim] (post-rope); out: device
 * f32 [rows][q_heads*head_dim]. Decode is rows == 1. */
int cheetah_hip_attention(const float *q, const cheetah_hip_kv_view *kv, uint32_t q_heads, size_t rows,
                          size_t offset, float *out);
/* cheetah_hip_attention that allocates nothing. No counterpart in the
 * reference: it is for callers that cannot allocate device memory (tight
 * serving loops, harnesses that forbid hipMalloc). The split partials live
 * in a fixed 48 MiB device array per GPU instead of a buffer the library
 * grows on demand; a call that needs more (rows * q_heads * splits *
 * (head_dim + 2) floats) is rejected with an error before any device work.
 * Same kernels and split choice, so the same results as
 * cheetah_hip_attention. Like every op-level entry point it launches on the
 * library's own stream (created by cheetah_hip_init; cheetah_hip_synchronize
 * waits for it), not on a stream of the caller's: it is not captured by a
 * graph capture the caller runs on its own stream. Calls within a process
 * are therefore ordered on that one stream and do not overlap on the
 * device; the array keeps the last call's partials. */
int cheetah_hip_attention_noalloc(const float *q, const cheetah_hip_kv_view *kv, uint32_t q_heads, size_t rows,
                                  size_t offset, float *out);

/* ------------------------------------------------------------------------
 * Drafted tokens and scoring, op level. No counterpart in the reference (it
 * decodes one token at a time and reads the last row's logits). Buffers the
 * calls read or write may be any memory of the library's device; work on them
 * that runs on other streams must have finished, as for every op-level call.
 * ---------------------------------------------------------------------- */

/* Most nodes of a tree of drafted tokens. */
#define CHEETAH_HIP_MAX_TREE_NODES 256
/* Attention for a tree of n drafted tokens that continue a cached sequence of
 * `offset` positions. parents (device int32 [n]) holds each node's parent, an
 * earlier node; a value outside [0, i) makes node i a root. Node i's K/V row is
 * already in the cache, at position offset + i. Every node attends to the
 * positions [0, offset), its ancestors and itself: never to other branches or to
 * positions past the tree, whatever their rows hold (NaN, unwritten memory). An
 * infinity or NaN in a V row that a node does see shows in that element of its
 * output (NaN where the row's weight rounds to 0); finite rows of any size average
 * to finite outputs. Rows with such values are slow (computed key by key).
 * kv: the paged view of cheetah_hip_attention; kv_format 0 = BF16 pools, 1 =
 * f32 (k_pages / v_pages then point to f32 elements). Page size a multiple of
 * 64, head_dim 64 or 128, 1 to 8 query heads per KV head, 16-byte aligned
 * buffers. q: device f32 [n][q_heads*head_dim] (each rotated for its own
 * position, offset + depth); out: device f32, the same shape. */
int cheetah_hip_tree_attention(const float *q, const cheetah_hip_kv_view *kv, uint32_t kv_format, uint32_t q_heads,
                               const int32_t *parents, size_t n, size_t offset, float *out);
/* Keeps one branch of a tree: in each of the nviews caches (one per layer) the
 * K/V rows of positions offset + nodes[j] move to offset + j, j = 0 .. count-1.
 * nodes (host) is strictly increasing and below CHEETAH_HIP_MAX_TREE_NODES: a
 * root and its descendants in order. The views (host array) may have page
 * tables of their own but one page size, KV head count and head_dim; a cache
 * listed twice (a pool with the same page table) is refused. Rows past the branch
 * are left as they are. */
int cheetah_hip_tree_commit(const cheetah_hip_kv_view *views, size_t nviews, uint32_t kv_format, size_t offset,
                            const uint32_t *nodes, size_t count);

/* ------------------------------------------------------------------------
 * An 8-bit K/V cache, op level. No counterpart in the reference (its caches are
 * f32). A cached value is an E4M3 code (sign, 4 bits of exponent, 3 of fraction,
 * no infinities) times the scale of its block: CHEETAH_HIP_KV8_BLOCK consecutive
 * positions of one KV head, K and V apart. A scale is 2^e, kept as the byte
 * e + 127, e in [-117, 119]: every value is a normal f32 and an exact BF16 one.
 *   codes  [pages][kv_heads][page_size / 32][32 * head_dim] bytes; a K block is
 *          [head_dim / 32][32 positions][32 dims], a V block [head_dim][32 positions]
 *   scales [pages][kv_heads][page_size / 32] bytes
 * page_size is a multiple of 64, head_dim 64 or 128; codes are 16-byte aligned,
 * the four pools do not overlap. page_table (device int32) maps logical pages;
 * entries of pages that a call neither writes nor reads may hold anything. The
 * pages that one append writes differ.
 * ---------------------------------------------------------------------- */
#define CHEETAH_HIP_KV8_BLOCK 32
typedef struct cheetah_hip_kv8_view {
    uint8_t *k_codes;
    uint8_t *v_codes;
    uint8_t *k_scales;
    uint8_t *v_scales;
    const int32_t *page_table;
    uint32_t page_size;
    uint32_t kv_heads;
    uint32_t head_dim;
} cheetah_hip_kv8_view;
/* Quantises `rows` K and V rows into positions offset .. offset + rows - 1. k, v:
 * device rows of kv_heads * head_dim values, `stride` >= that many elements apart
 * (k and v may point into packed projections), row_format 0 = BF16, 1 = f32. A
 * block's scale is the least with |x| <= 448 * 2^e for its rows, codes round to
 * nearest (ties to even). Rows of the block before `offset` (written before, from
 * its first on) keep their values; a scale that later rows raise rounds them again
 * (only values below 2^-13 of the block's largest move, by at most 2^-16 of it), and
 * it does not fall before the block's first position is written again. Rows behind
 * the last new one keep their codes, not their values. An infinity or a NaN is kept
 * as NaN and does not count for the scale; magnitudes past 448 * 2^119 become that. */
int cheetah_hip_kv8_append(const void *k, const void *v, uint32_t row_format, size_t rows, size_t stride, size_t offset,
                           const cheetah_hip_kv8_view *kv);
/* The cached K and V rows of positions begin .. begin + n - 1 as [n][kv_heads *
 * head_dim] values (device, 16-byte aligned), row_format 0 = BF16, 1 = f32; both
 * exact. */
int cheetah_hip_kv8_read(const cheetah_hip_kv8_view *kv, size_t begin, size_t n, uint32_t row_format, void *k_out,
                         void *v_out);
/* GQA causal attention over an 8-bit cache for `rows` query rows at positions
 * offset .. offset + rows - 1 (their K/V already in the cache), q and out as
 * cheetah_hip_attention's, 16-byte aligned. With window 0 row i sees the
 * positions [0, offset + i]; with a window the last `window` of these and the
 * first `sinks` positions (sinks is 0 without a window). 1 to 8 query heads per
 * KV head. Positions that a row does not see do not count, whatever they hold
 * (NaN, unwritten memory); a NaN in a row that it does see shows. Pages that no row
 * sees are not read. */
int cheetah_hip_kv8_attention(const float *q, const cheetah_hip_kv8_view *kv, uint32_t q_heads, size_t rows,
                              size_t offset, size_t window, size_t sinks, float *out);

/* Most alternatives a row of cheetah_hip_logprobs returns. */
#define CHEETAH_HIP_MAX_TOP 64
/* For each of `rows` rows of `vocab` logits (device, `stride` >= vocab elements
 * apart; logit_format 0 = BF16, 1 = f32), in natural logarithms:
 *   logprobs[r] = x[tokens[r]] - log sum exp x   (tokens: device uint32 [rows];
 *                 NaN where the id is not below vocab)
 *   entropy[r]  = - sum p log p
 *   top_ids[r][i], top_logprobs[r][i], i < top: the `top` largest logits in
 *                 descending order, equal ones by ascending id.
 * top is at most CHEETAH_HIP_MAX_TOP and vocab. Outputs are device arrays; any
 * may be null (tokens too, without logprobs), but not all of them, and top_ids
 * and top_logprobs go together with top > 0. -inf logits have probability 0; a
 * row of nothing else has log probabilities of -inf and entropy 0. A row that
 * holds a NaN or +inf has NaN for each log probability and its entropy; its
 * alternatives are ordered with NaN as -inf. */
int cheetah_hip_logprobs(const void *logits, uint32_t logit_format, size_t rows, size_t vocab, size_t stride,
                         const uint32_t *tokens, uint32_t top, float *logprobs, float *entropy, uint32_t *top_ids,
                         float *top_logprobs);

/* ------------------------------------------------------------------------
 * Model: the HIP implementation of ModelForward (registry.rs:57-85) for the
 * qwen2 and llama families (registrations/qwen2.rs, llama.rs).
 * ---------------------------------------------------------------------- */
typedef struct cheetah_hip_config {
    uint32_t family; /* 0 = qwen2, 1 = llama */
    uint32_t num_layers;
    uint32_t hidden_size;
    uint32_t q_heads;
    uint32_t kv_heads;
    uint32_t head_dim;
    uint32_t rotary_dim;
    uint32_t intermediate_size;
    uint32_t vocab_size;
    uint32_t tie_word_embeddings;
    uint32_t sliding_window; /* 0 = whole cache; others with an 8-bit KV cache (kv_format 2) only */
    float rope_theta;
    float rms_eps;
} cheetah_hip_config;

typedef struct cheetah_hip_model cheetah_hip_model;
typedef struct cheetah_hip_snapshot cheetah_hip_snapshot;

/* Creates a model shell. quant_format: 0 = stored precision (BF16), 4 = q8,
 * 5 = q4 (CHEETAH_QUANT_Q8 / CHEETAH_QUANT_Q4, precision.rs:333-356; linear
 * projections only — embedding, head, norms and biases keep BF16,
 * ops.rs:1533-1537). kv_format: element type of the paged KV cache, 0 = BF16
 * (half the KV bytes), 1 = f32 (the reference's own cache precision,
 * ops.rs:995-999), 2 = 8 bits (a quarter; cheetah_hip_kv8_append's codes and
 * scales: K and V are rounded, by up to 2^-4 of a value; values below 2^-13.8 of
 * the largest of their block, by up to 2^-17.8 of that, so that small ones can
 * vanish). Over an 8-bit cache a position's results depend, in their last bits, on
 * how the text was cut into chunks and, behind a prefix restored up to a position
 * inside a block, on the rows cut off (the block's scale stays theirs), and drafted
 * tokens are refused. kv_capacity: positions the KV pool holds across this
 * model, its clones and its snapshots (0 = 65536). max_chunk_rows: largest
 * prefill chunk (0 = 1024). */
cheetah_hip_model *cheetah_hip_model_create(const cheetah_hip_config *cfg, uint32_t quant_format,
                                            uint32_t kv_format, size_t kv_capacity, size_t max_chunk_rows);
/* Uploads one weight unit (host bytes, as MmapWeightStore::slice serves
 * them, store.rs:189-203). dtype: 1 = BF16 (the only stored precision
 * served). Unit ids are the safetensors names ("model.layers.3.mlp.up_proj.weight"). */
int cheetah_hip_model_set_unit(cheetah_hip_model *m, const char *unit_id, const void *bytes, size_t nbytes,
                               uint32_t dtype, const uint64_t *shape, size_t ndim);
/* Checks every unit is present with its shape, builds the fused device
 * layouts and quantizes (the load-time half of ops.rs:1199-1226). */
int cheetah_hip_model_finalize(cheetah_hip_model *m);

/* ModelForward::forward (registry.rs:60): runs tokens[0..n) from absolute
 * position `offset` (must equal the cached length, transformer.rs:799-810)
 * and writes the final position's logits (vocab_size floats) to logits_out.
 * n == 1 runs the decode step; n > 1 runs chunked prefill in chunks of
 * chunk_rows (0 = 256, CHEETAH_PREFILL_CHUNK default, ops.rs:519-535). */
int cheetah_hip_forward(cheetah_hip_model *m, const uint32_t *tokens, size_t n, size_t offset,
                        size_t chunk_rows, float *logits_out);
/* forward + greedy sampling on the device (engine.rs:2247-2253: argmax,
 * ties to the last index). logits_out may be NULL. */
int cheetah_hip_forward_greedy(cheetah_hip_model *m, const uint32_t *tokens, size_t n, size_t offset,
                               size_t chunk_rows, uint32_t *next_token, float *logits_out);
/* The greedy decode loop of Engine::generate_inner (engine.rs:1920-1961)
 * kept on the device: starting from `token` at position `offset`, runs
 * `steps` decode forwards, each feeding its argmax to the next, and writes
 * the sampled ids to tokens_out[steps]. */
int cheetah_hip_decode_greedy(cheetah_hip_model *m, uint32_t token, size_t offset, size_t steps,
                              uint32_t *tokens_out);
/* Verification of drafted tokens (speculative decoding; no counterpart in the
 * reference; refused over an 8-bit KV cache). A tree of candidate tokens is run in one forward behind the
 * cached positions. tokens[n]; parents[n]: parents[i] in [-1, i), -1 for a child
 * of the cached text; n at most CHEETAH_HIP_MAX_TREE_NODES and max_chunk_rows.
 * Node i attends to the cache, its ancestors and itself, at position offset +
 * depth; offset must equal the cached length, and offset + n must fit the
 * capacity.
 *   forward_tree: next_tokens[n] (or NULL) receives every node's argmax (ties
 *     to the last index), logits_out[n * vocab_size] (or NULL) every node's
 *     logits. The cached length stays; the nodes' K/V rows wait behind it until
 *     commit_tree or until anything else runs on this instance or clears or
 *     restores its cache, which drops them.
 *   commit_tree: keeps a branch of that tree, nodes[count] from a child of the
 *     cached text to any node, each followed by a child of it; the cache then
 *     holds the branch's tokens, as if they had been run alone (up to the
 *     rounding of a chunk's products). count 0 drops the tree.
 *   verify_tree: forward_tree and commit_tree in one call, greedily. Node 0 is
 *     the only root: the last token sampled, not yet in the cache. From it the
 *     walk goes to the child whose token is the argmax while there is one (the
 *     first such child). accepted[n] receives the walk's nodes, *count (at least
 *     1) their number, *next_token the argmax behind the last of them: what
 *     `count` steps of greedy decoding would have sampled (but for near ties: a
 *     tree's products are a chunk's, which round otherwise than a decode step's).
 *     The cache then holds the accepted tokens. */
int cheetah_hip_forward_tree(cheetah_hip_model *m, const uint32_t *tokens, const int32_t *parents, size_t n,
                             size_t offset, uint32_t *next_tokens, float *logits_out);
int cheetah_hip_commit_tree(cheetah_hip_model *m, const uint32_t *nodes, size_t count);
int cheetah_hip_verify_tree(cheetah_hip_model *m, const uint32_t *tokens, const int32_t *parents, size_t n,
                            size_t offset, uint32_t *accepted, size_t *count, uint32_t *next_token);
/* forward that scores every position (cheetah_hip_logprobs of each one's
 * logits; no counterpart in the reference): targets[n] are the tokens whose
 * log probabilities go to logprobs[n] (both may be NULL; for a text's own tokens
 * targets[i] = the token after tokens[i]; one past the vocabulary gives NaN),
 * entropy[n] may be NULL, top_ids and top_logprobs [n * top] are NULL when top
 * is 0. Chunks and cache as cheetah_hip_forward, bit for bit: one token is a
 * decode step, and its scores are of that step's logits. */
int cheetah_hip_forward_logprobs(cheetah_hip_model *m, const uint32_t *tokens, size_t n, size_t offset,
                                 size_t chunk_rows, const uint32_t *targets, uint32_t top, float *logprobs,
                                 float *entropy, uint32_t *top_ids, float *top_logprobs);
/* ModelForward::clear_cache (registry.rs:62). */
void cheetah_hip_clear_cache(cheetah_hip_model *m);
/* Boxed clone per generation (registry.rs:95-117, ops.rs:1017-1029): shares
 * weights and the KV page pool, starts with an empty cache. */
cheetah_hip_model *cheetah_hip_clone(const cheetah_hip_model *m);
size_t cheetah_hip_kv_len(const cheetah_hip_model *m);
/* ModelForward::kv_snapshot / restore_kv_prefix (registry.rs:68-79). A
 * snapshot holds references to the model's KV pages (no copy); a restore
 * maps the first `positions` positions into an empty model and copies a
 * page only when it is next written (copy on write). */
int cheetah_hip_kv_snapshot(const cheetah_hip_model *m, cheetah_hip_snapshot **out, size_t *positions);
int cheetah_hip_restore_kv_prefix(cheetah_hip_model *m, const cheetah_hip_snapshot *s, size_t positions);
void cheetah_hip_snapshot_free(cheetah_hip_snapshot *s);
/* Cached K and V rows of positions [pos_begin, pos_begin + n) of one layer,
 * written to host buffers of n * kv_heads * head_dim floats each in the
 * reference's per-layer cache layout [pos][kv_head][dim] (ops.rs:995-999,
 * the rows KvSnapshot carries, registry.rs:48-55). BF16 and 8-bit pages widen
 * exactly.
 * Waits for the model's queued work. */
int cheetah_hip_kv_download(const cheetah_hip_model *m, uint32_t layer, size_t pos_begin, size_t n, float *k_out,
                            float *v_out);
void cheetah_hip_model_free(cheetah_hip_model *m);

/* Ant tier control (AntTierControl::page_in_unit / evict_unit,
 * registry.rs:87-93; called from engine.rs:1210-1226). The movable units
 * are the per-layer linear weights, model.layers.{l}.self_attn.{q,k,v,o}_proj
 * .weight and model.layers.{l}.mlp.{gate,up,down}_proj.weight; q, k and v
 * name one fused matrix and move together.
 *   evict:   the device buffer is released and a pinned host copy becomes
 *            authoritative (vulkan/transformer.rs:578-583). Forwards keep
 *            working: each such layer's matrices are copied into one of two
 *            device slots on a second stream, one streamed layer ahead of
 *            the compute, with the same kernels reading them there (results
 *            are bit-identical). While any unit is evicted, decode runs the
 *            per-kernel path (no persistent kernel, no captured graph).
 *   page_in: the unit returns to HBM and its host copy is freed; `tier` is
 *            accepted and ignored, as every reference implementation does
 *            (vulkan/transformer.rs:572-576).
 * Both return 1 when the id names a movable unit (also when it already sits
 * in the requested tier), 0 for any other id, -1 on error. They wait for the
 * device to go idle and change weights shared with every clone: they must
 * not overlap a forward on any instance sharing them. */
int cheetah_hip_evict_unit(cheetah_hip_model *m, const char *unit_id);
int cheetah_hip_page_in_unit(cheetah_hip_model *m, const char *unit_id, int32_t tier);
/* Where a unit sits: 1 = HBM, 2 = pinned host memory, 0 = not a movable
 * unit, -1 on error. Has no reference counterpart (the reference's Ant
 * bookkeeping tracks tiers on the engine side); for tests and monitoring. */
int cheetah_hip_unit_tier(const cheetah_hip_model *m, const char *unit_id);

/* ------------------------------------------------------------------------
 * Measurement hooks (events on the stream the kernels run on).
 * ---------------------------------------------------------------------- */
/* Times `iters` launches of one op-level GEMV over `nbuf` rotating weight
 * buffers (defeats the 256 MB Infinity Cache); returns the mean
 * milliseconds per launch in *ms. fmt: 1 = BF16, 4 = q8, 5 = q4. */
int cheetah_hip_time_gemv(uint32_t fmt, const void *const *w, size_t nbuf, size_t rows, size_t cols,
                          const float *x, float *y, size_t iters, float *ms);
/* Times `iters` launches of the op-level GEMM (n input rows) over `nbuf`
 * rotating weight buffers; mean milliseconds per launch in *ms. */
int cheetah_hip_time_gemm(uint32_t fmt, const void *const *w, size_t nbuf, size_t rows, size_t cols,
                          const float *x, size_t n, float *y, size_t iters, float *ms);
/* Times `iters` launches of cheetah_hip_attention over `nviews` rotating KV
 * caches (views[i]); mean milliseconds per launch in *ms. */
int cheetah_hip_time_attention(const float *q, const cheetah_hip_kv_view *views, size_t nviews, uint32_t q_heads,
                               size_t rows, size_t offset, float *out, size_t iters, float *ms);
/* Times `steps` greedy decode steps of a model already holding `offset`
 * cached positions (the decode graph replayed back to back), and the
 * model's largest GEMV alone over the same steps; both in ms per step. */
int cheetah_hip_time_decode(cheetah_hip_model *m, uint32_t token, size_t offset, size_t steps,
                            float *ms_per_step, float *gemv_ms_per_launch, uint32_t *tokens_out);

#ifdef __cplusplus
}
#endif

#endif
