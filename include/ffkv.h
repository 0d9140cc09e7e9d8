/*
 * ffkv.h - C ABI of the MI355X (gfx950) paged KV-cache path.
 *
 * This is the drop-in boundary for Firefly's paged KV-cache hot path: appending new K/V tokens into
 * block-table-addressed pages (optionally quantizing to int8 or OCP fp8 e4m3, optionally fused with the rotary
 * embedding of q and k) and PagedAttention decode (GQA, split-K, online softmax).  Plain pointers and sizes
 * only; no C++ or HIP types appear here, so ctypes / cgo / JNI / N-API callers can bind it directly.  `stream` is a hipStream_t passed as void*
 * (NULL = the legacy default stream).
 *
 * Layout contract (identical to the reference):
 *   K/V pages       [num_blocks, block_size=16, num_kv_heads, head_dim], element (p, o, h, d) at
 *                   ((p*16 + o)*num_kv_heads + h)*head_dim + d        (src/model/qwen_model.cu:41-42,
 *                                                                       src/kernels/attention.cu:347-348)
 *   block_table     int32 [batch, max_blocks], row stride max_blocks  (src/kernels/attention.cu:334)
 *   context_lens    int32 [batch], tokens already cached BEFORE this step's append
 *                   (src/model/qwen_model.cu:32-33, src/kernels/attention.cu:320)
 *   append source   [batch, seq_len, num_kv_heads, head_dim]          (src/model/qwen_model.cu:39)
 *   q               [batch, 1, num_heads, head_dim]; out [batch, 1, num_heads*head_dim]
 *   GQA head map    kv_head = q_head / (num_heads / num_kv_heads)     (src/kernels/attention.cu:304)
 *
 * Quantized caches (no counterpart in the reference, which is fp16-only):
 *   FFKV_DTYPE_I8       symmetric int8, scale per (page, slot, kv_head): fp32 [num_blocks, 16, num_kv_heads],
 *                       scale = absmax/127 (IEEE fp32 divide), q = clamp(rint_half_even(x/scale), -127, 127),
 *                       absmax == 0 gives scale 0 and q 0.  Scales are WRITTEN by ffkv_append.
 *   FFKV_DTYPE_FP8_E4M3 OCP e4m3 (bias 7, max 448, NaN = S.1111.111), scale per kv_head: fp32 [num_kv_heads],
 *                       q = e4m3_round_half_even_satfinite(x/scale).  Scales are READ by ffkv_append.
 *
 * Invalid addressing is defined instead of undefined (the reference writes/reads block -1 for padded rows,
 * src/engine.cc:298-300 with src/model/qwen_model.cu:37,41-45): a block-table entry < 0 or >= num_blocks,
 * a logical block index >= max_blocks, or a negative position is skipped by append and masked out by decode;
 * a decode row with no valid token produces zeros.
 *
 * All entry points are asynchronous on `stream`, never synchronize the host, and are safe to capture in a
 * hipGraph: nothing is allocated inside a capture, so give captured calls a workspace (a decode without one splits no
 * rows there, and the others say below what they do).  Return 0 on success or a negative
 * FFKV_ERR_* code; ffkv_last_error() gives a message for the calling thread.
 */
#ifndef FFKV_H_
#define FFKV_H_

#include <stddef.h>
#include <stdint.h>

#ifndef FFKV_API
#define FFKV_API __attribute__((visibility("default")))
#endif

#ifdef __cplusplus
extern "C" {
#endif

#define FFKV_BLOCK_SIZE 16

/* dtype codes: equal to the firefly::DType enumerators F32, F16, BF16, I8 (include/firefly/types.h:16-26 in
 * the reference, whose enum continues I32, I64, U8, UNKNOWN = 7), plus FP8_E4M3 = 8, which the reference lacks. */
#define FFKV_DTYPE_F32 0
#define FFKV_DTYPE_F16 1
#define FFKV_DTYPE_BF16 2
#define FFKV_DTYPE_I8 3
#define FFKV_DTYPE_FP8_E4M3 8

#define FFKV_OK 0
#define FFKV_ERR_INVALID_ARGUMENT -1
#define FFKV_ERR_UNSUPPORTED -2
#define FFKV_ERR_WORKSPACE -3
#define FFKV_ERR_HIP -4

/*
 * Scatter new K/V tokens into their pages.  Replaces the reference's unexported append kernel launch
 * `append_kv_cache<<<(seq_len, Hkv, B), 128, 0, stream>>>(k, v, k_cache, v_cache, block_table, context_lens,
 * max_blocks, Hkv, D)` (src/model/qwen_model.cu:21-47, launched at :138-143).
 *
 * Token t of row b goes to position pos = context_lens[b] + t (context_lens == NULL means 0), i.e. page
 * block_table[b*max_blocks + pos/16], slot pos%16.  src_dtype is F32, F16 or BF16; cache_dtype is F32, F16,
 * BF16 (copy, rounding to nearest even when narrowing), I8 or FP8_E4M3 (quantize, see above).
 * k_scale / v_scale: I8 -> written, [num_blocks, 16, num_kv_heads]; FP8 -> read, [num_kv_heads]; else unused.
 * head_dim is a multiple of 8 up to 128 (the reference's append takes any head_dim up to its 128-thread block),
 * or 256; block_size must be 16.  Source and cache pointers must be 16-byte aligned.
 */
FFKV_API int ffkv_append(const void* k_src, const void* v_src, int src_dtype, void* k_cache, void* v_cache, int cache_dtype,
                float* k_scale, float* v_scale, const int32_t* block_table, const int32_t* context_lens, int batch,
                int seq_len, int num_kv_heads, int head_dim, int block_size, int max_blocks, int num_blocks,
                void* stream);

/*
 * Bytes one pool block (16 tokens of one layer, K and V) takes in a cache of cache_dtype, its scales included:
 * what an engine divides its memory budget by to size the pools.  Replaces the 16-bit element size in the
 * reference's `max_num_blocks = 0.9 * free / (num_layers * 16 * Hkv * D * 2 * 2)` (src/engine.cc:90-96, pools
 * allocated at :104-113):
 *   F32        16 * Hkv * D * 4 * 2
 *   F16, BF16  16 * Hkv * D * 2 * 2
 *   I8         16 * Hkv * (D + 4) * 2   codes and the per-token-per-head fp32 scales [num_blocks, 16, Hkv]
 *   FP8_E4M3   16 * Hkv * D * 2         codes; the per-head scales (2 * Hkv * 4 bytes per layer) do not grow
 *                                       with the pool
 * Returns 0 for another dtype or a non-positive size.  No counterpart in the reference (fp16 pools only).
 */
FFKV_API size_t ffkv_kv_block_bytes(int cache_dtype, int num_kv_heads, int head_dim);

/*
 * Bytes of scratch ffkv_paged_decode needs for split-K partial results at these sizes.  max_context_len is
 * an upper bound on context_lens[b] + 1 (<= 0 means max_blocks * 16).  No counterpart in the reference, whose
 * decode kernel has no split-K (src/kernels/attention.cu:475-485).
 */
FFKV_API size_t ffkv_decode_workspace_bytes(int batch, int num_heads, int head_dim, int max_blocks, int max_context_len);


/*
 * PagedAttention decode: out[b, h, :] = softmax(scale * q[b,h] . K_j) V_j over the context_lens[b] + 1 cached
 * tokens of row b (the +1 is the token appended this step).  Replaces `firefly::kernels::attention(q, k_cache,
 * v_cache, out, block_table, kv_head_num, seq_len, max_context_blocks, context_lens)` on its decode branch
 * (include/firefly/kernels.h:83-84, src/kernels/attention.cu:452-493 -> paged_attention_kernel :291-447).
 *
 * qo_dtype (q and out) is F32, F16 or BF16; cache_dtype as for ffkv_append.  scale <= 0 selects
 * 1/sqrt(head_dim) (src/kernels/attention.cu:458).  num_heads must be a multiple of num_kv_heads (any group
 * size for 16- and 8-bit caches at head_dim 64, 80, 96, 112, 128 and 256, at most 16 otherwise)
 * and at most 65535; head_dim a multiple of 8 up to 128 (as the reference's decode,
 * src/kernels/attention.cu:307-316), or 256: 64, 80, 96, 112, 128 and 256 run the matrix-core kernels, the others a
 * vector kernel; q, out, cache and workspace pointers 16-byte aligned.  Rows are
 * split over the context and the pieces merged; the partials live in `workspace` (ffkv_decode_workspace_bytes;
 * any initial contents), or, when workspace is NULL, in stream-ordered memory the library allocates and frees on
 * `stream`; while `stream` is being captured a call without a workspace leaves its rows whole instead, equal up to rounding,
 * which is slower for few or long rows (1 row of 32000 tokens at 32/8 heads 366 us against 33, 64 rows of 512 to 4096 114
 * against 95).  Calls sharing one workspace must not overlap in time (use one workspace per stream).  Rows whose
 * context_lens[b] + 1 exceeds max_context_len are truncated to it.
 */
FFKV_API int ffkv_paged_decode(const void* q, void* out, int qo_dtype, const void* k_cache, const void* v_cache,
                      int cache_dtype, const float* k_scale, const float* v_scale, const int32_t* block_table,
                      const int32_t* context_lens, int batch, int num_heads, int num_kv_heads, int head_dim,
                      int block_size, int max_blocks, int num_blocks, int max_context_len, float scale,
                      void* workspace, size_t workspace_bytes, void* stream);

/*
 * ffkv_paged_decode without any device allocation: the split-K partials live in a static scratch array that the
 * library holds on every GPU it runs on (FFKV_NOALLOC_SCRATCH_BYTES each, until the process ends), so the call
 * never allocates or frees device memory, whatever `workspace` contract the caller could keep.  No counterpart in
 * the reference; it is for callers that cannot allocate: code under hipGraph capture without a workspace, tight serving
 * loops, hosts that forbid allocation after start-up.  Arguments and results are those of ffkv_paged_decode (same kernels, same
 * split, bit-identical outputs).  Sizes whose partials exceed the scratch (roughly (work items + batch) *
 * num_heads * (head_dim + 2) * 4 bytes with the matrix-core kernel, batch * num_heads * chunks * (head_dim + 2) *
 * 4 with fp32 caches) return FFKV_ERR_WORKSPACE.  All calls on one GPU share its scratch: calls that overlap in
 * time on one GPU (two streams, two threads) race and must be serialized by the caller.
 */
#define FFKV_NOALLOC_SCRATCH_BYTES (32u << 20)

FFKV_API int ffkv_paged_decode_noalloc(const void* q, void* out, int qo_dtype, const void* k_cache,
                                       const void* v_cache, int cache_dtype, const float* k_scale,
                                       const float* v_scale, const int32_t* block_table, const int32_t* context_lens,
                                       int batch, int num_heads, int num_kv_heads, int head_dim, int block_size,
                                       int max_blocks, int num_blocks, int max_context_len, float scale,
                                       void* stream);

/*
 * ffkv_append of one token per row (seq_len 1) followed by ffkv_paged_decode, as one call: the decode step of
 * the reference's model (src/model/qwen_model.cu:138-146, append launch then kernels::attention).  k_new / v_new
 * [batch, 1, num_kv_heads, head_dim] in src_dtype; the other arguments as for the two functions.  When the
 * step's k/v already have the cache's 16-bit type it is a single launch: the decode work item that holds a
 * row's last page reads the new token from k_new / v_new instead of the page, attends it, and writes it to its
 * page slot (rows cut short by max_context_len get the token copied to its slot without attending it).  In that
 * form a row's slot for its new token is its own: no other row of the call may attend it (rows that do, such as
 * several tokens of one sequence, take ffkv_append and ffkv_paged_decode).
 * Otherwise it runs the two functions in turn.  Either way the pages are
 * bit-identical to ffkv_append's and the output is ffkv_paged_decode's on them.  No counterpart in the
 * reference (two launches there).
 */
FFKV_API int ffkv_append_paged_decode(const void* k_new, const void* v_new, int src_dtype, const void* q, void* out,
                                      int qo_dtype, void* k_cache, void* v_cache, int cache_dtype, float* k_scale,
                                      float* v_scale, const int32_t* block_table, const int32_t* context_lens,
                                      int batch, int num_heads, int num_kv_heads, int head_dim, int block_size,
                                      int max_blocks, int num_blocks, int max_context_len, float scale,
                                      void* workspace, size_t workspace_bytes, void* stream);

/*
 * ffkv_paged_decode for a batch whose rows share a prefix of pages (the radix tree's shared blocks): entries
 * 0 .. shared_blocks - 1 of every row's block table are the same physical pages, read from row 0's table.  The
 * prefix is attended once for all rows as a matrix product (every row's queries of a kv head against each
 * prefix page, split into chunks of pages), the rest of each row by the decode kernel, and the split-K merge
 * folds both: each shared page is read once per call instead of once per row.  Results equal ffkv_paged_decode
 * on the same inputs up to floating-point summation order (same tolerance).  Rows shorter than the prefix
 * attend only their own tokens.  The split applies to F16/BF16/I8/FP8 caches; fp32 caches run
 * ffkv_paged_decode unchanged.  No counterpart in the reference, whose decode reads shared blocks once per row
 * (src/kernels/attention.cu:332-335).  Workspace: ffkv_decode_shared_prefix_workspace_bytes, or NULL as for
 * ffkv_paged_decode (a captured call without one attends the prefix with each row).
 */
FFKV_API size_t ffkv_decode_shared_prefix_workspace_bytes(int batch, int num_heads, int num_kv_heads, int head_dim,
                                                          int max_blocks, int max_context_len, int shared_blocks);

FFKV_API int ffkv_paged_decode_shared_prefix(const void* q, void* out, int qo_dtype, const void* k_cache,
                                             const void* v_cache, int cache_dtype, const float* k_scale,
                                             const float* v_scale, const int32_t* block_table,
                                             const int32_t* context_lens, int batch, int num_heads, int num_kv_heads,
                                             int head_dim, int block_size, int max_blocks, int num_blocks,
                                             int max_context_len, float scale, int shared_blocks, void* workspace,
                                             size_t workspace_bytes, void* stream);

/*
 * Causal prefill attention over the paged cache (chunked prefill with prefix reuse).  Replaces the prefill branch
 * of `firefly::kernels::attention` (kv_cache_block_table == nullptr: flash_attn_wmma_kernel,
 * src/kernels/attention.cu:22-286, dispatched at :460-474) and extends it to cached prefixes, which the
 * reference's model skips (src/model/qwen_model.cu:147-151 routes every multi-token batch-1 step to the
 * contiguous kernel).
 *
 * q [batch, seq_len, num_heads, head_dim], out [batch, seq_len, num_heads*head_dim], both qo_dtype.  With a
 * block table, query token t of row b sits at position context_lens[b] + t and attends the row's keys
 * 0 .. context_lens[b] + t read from the pages (context_lens = tokens cached BEFORE this chunk, whose K/V must
 * already be appended, e.g. by ffkv_append with the same context_lens); keys on invalid pages or at or beyond
 * min(context_lens[b] + seq_len, max_context_len or max_blocks*16) are skipped, and a query with no key gives
 * zeros.  With block_table == NULL, k_cache / v_cache are the chunk's contiguous [batch, seq_len, num_kv_heads,
 * head_dim] tensors and positions start at 0: the reference's causal prefill.  seq_len = 1 is decode attention.
 * cache_dtype F16, BF16, I8 or FP8_E4M3 (scales as for ffkv_paged_decode); any GQA group; scale <= 0 selects
 * 1/sqrt(head_dim).  No workspace; pointers 16-byte aligned.  fp8 per-head K scales may be any finite value (0
 * weighs the keys uniformly, a negative one negates the scores, as in decode).  int8 caches: the attention
 * weights (below 2^8) meet their V scales in f16, so a per-token V scale of 256 or more can overflow; a workgroup
 * whose results overflow reruns with its weights scaled by 2^-12, which takes V scales up to 2^20 (|V| up to about
 * 1.3e8).  bf16 caches: V enters the products in f16 (a workgroup that meets |V| >= 65520 reruns in bf16), so V values
 * below 2^-14 carry an absolute error of at most 2^-25.  16-bit caches: an infinite V value also makes NaN, in
 * its dim, the outputs of the queries whose causal limit masks its key (it meets them with weight 0 in the tile
 * products), as in the reference's prefill, whose P.V tile product (src/kernels/attention.cu:232-243) takes every
 * key of its 16-key tile, the causally masked ones with p = 0 (:173-174).
 */
FFKV_API int ffkv_paged_prefill(const void* q, void* out, int qo_dtype, const void* k_cache, const void* v_cache,
                                int cache_dtype, const float* k_scale, const float* v_scale, const int32_t* block_table,
                                const int32_t* context_lens, int batch, int seq_len, int num_heads, int num_kv_heads,
                                int head_dim, int block_size, int max_blocks, int num_blocks, int max_context_len,
                                float scale, void* stream);

/*
 * ffkv_paged_prefill with scratch: a call with too few blocks of 128 query rows to fill the GPU (one request's chunk
 * over a long context, a short prompt) splits their keys into pieces that run side by side, whose partial results
 * live in `workspace` (ffkv_prefill_workspace_bytes; 16-byte aligned, any initial contents), and merges them.  Results
 * equal ffkv_paged_prefill's up to rounding: the sums take another order, and a piece rounds its attention weights to
 * their 11 bits against a maximum of its own (together 1e-3 of the result in bf16, both equally far from the exact one);
 * rows that are NaN are the same.  Equal calls give equal bits.
 * The bound on a row (max_context_len, or the table's width) decides whether a split is planned:
 * ffkv_prefill_workspace_bytes is 0 where it is not; with workspace NULL, or fewer bytes than that, the call runs unsplit,
 * as ffkv_paged_prefill.  A planned call whose rows turn out too short is not split, but pays 1 to 2 us for the launch of
 * a merge without work: give max_context_len where the rows' lengths are known and the table is wide.
 * Calls sharing one workspace must not overlap in time.  paged: whether the call has a block table.
 */
FFKV_API size_t ffkv_prefill_workspace_bytes(int qo_dtype, int cache_dtype, int batch, int seq_len, int num_heads,
                                             int num_kv_heads, int head_dim, int paged, int max_blocks,
                                             int max_context_len);

FFKV_API int ffkv_paged_prefill_ws(const void* q, void* out, int qo_dtype, const void* k_cache, const void* v_cache,
                                   int cache_dtype, const float* k_scale, const float* v_scale,
                                   const int32_t* block_table, const int32_t* context_lens, int batch, int seq_len,
                                   int num_heads, int num_kv_heads, int head_dim, int block_size, int max_blocks,
                                   int num_blocks, int max_context_len, float scale, void* workspace,
                                   size_t workspace_bytes, void* stream);

/*
 * Rotary position embedding of q and k in place.  Replaces `firefly::kernels::apply_rope(q, k, head_dim, seq_len,
 * theta, context_lens)` (include/firefly/kernels.h:68, src/kernels/rope.cu:22-137, called at
 * src/model/qwen_model.cu:136).  q [batch, seq_len, num_heads, head_dim] and k [batch, seq_len, num_kv_heads,
 * head_dim] share `dtype` (F32, F16 or BF16); q may be NULL (then num_heads is ignored).  Token t of row b is
 * at position context_lens[b] + t (t when context_lens is NULL).  Rotate-half form: pair i (dims i, i + D/2) is
 * rotated by pos * inv_freq_i with inv_freq_i = theta^(-2i/head_dim):
 *     x_i' = x_i cos - x_{i+D/2} sin,   x_{i+D/2}' = x_{i+D/2} cos + x_i sin.
 * inv_freq, cos and sin are evaluated in double precision and rounded once to fp32, the angle is one fp32
 * product of float(pos) and inv_freq, the rotation uses separately rounded fp32 products and sums, and the
 * result is rounded to nearest even in `dtype`.  q and k must be 16-byte aligned.
 */
FFKV_API int ffkv_rope(void* q, void* k, int dtype, const int32_t* context_lens, int batch, int seq_len, int num_heads,
                       int num_kv_heads, int head_dim, float rope_theta, void* stream);

/*
 * ffkv_rope followed by ffkv_append of the rotated k (as rounded in src_dtype) and v, in one pass: the
 * reference's `kernels::apply_rope` + append launch pair (src/model/qwen_model.cu:136-143) fused, saving a
 * launch and a read of k.  Arguments as for ffkv_rope and ffkv_append; q may be NULL.  k is rotated in place
 * (as apply_rope leaves it) and v is only read.  The page contents are bit-identical to ffkv_rope followed by
 * ffkv_append.
 */
FFKV_API int ffkv_rope_append(void* q, void* k, const void* v, int src_dtype, void* k_cache, void* v_cache,
                              int cache_dtype, float* k_scale, float* v_scale, const int32_t* block_table,
                              const int32_t* context_lens, int batch, int seq_len, int num_heads, int num_kv_heads,
                              int head_dim, int block_size, int max_blocks, int num_blocks, float rope_theta,
                              void* stream);

/*
 * ---- attention under a score rule --------------------------------------------------------------------------------
 * For the query at position i, head h and the key at position j, with s = scale * q.k:
 *   score_cap  > 0: s becomes score_cap * tanh(s / score_cap) (caps below 7e-31 as 7e-31); 0: left as it is
 *   slopes     fp32 [num_heads], not NULL: s becomes s - slopes[h] * |i - j| (after the cap); finite values
 *   window     > 0: keys j <= i - window are hidden (a query sees its own and the window - 1 positions before it)
 *   key_begin  int32, not NULL: keys before key_begin of the query are hidden
 * A hidden key has weight 0 whatever its K and V hold, NaN and infinities included, and a query that sees no key gives
 * zeros.  No counterpart in the reference, whose attention is plain causal (src/kernels/attention.cu:173-174, :347-360).
 *
 * ffkv_paged_decode_scored is ffkv_paged_decode under a rule (key_begin int32 [batch]), with two options:
 *   k_new / v_new  (both or neither; src_dtype theirs) the step's new tokens, appended first as
 *                  ffkv_append_paged_decode does: in the decode's own launch where they have the cache's 16-bit dtype
 *                  and a head_dim of the matrix cores (no other row of the call may then attend a row's new slot)
 *   weights        fp32 [batch, num_kv_heads, weight_stride]: the attention weight that each cached token j of row b gets,
 *                  summed over the query heads of a KV head, is added to what it had:
 *                    weights[b, kvh, j] = decay * prior[b, kvh, j] + sum of softmax(s)_j    j < context_lens[b]
 *                    weights[b, kvh, j] = sum of softmax(s)_j                               j = context_lens[b]
 *                  prior may be weights itself, or NULL (nothing earlier); tokens past the row's end, or at or beyond
 *                  max_context_len, are left as they were.  weight_stride is at least min(max_blocks * 16,
 *                  max_context_len); decay is finite and not negative.
 * q, out, caches, scales, tables, sizes, scale and errors as for ffkv_paged_decode; positions and distances count the
 * row's cached tokens.  ffkv_decode_scored_workspace_bytes is enough for every type, KV head count and window at these
 * sizes; ffkv_decode_scored_scratch_bytes is what the one call needs (0 for small batches, which take one launch).  With
 * weights the workspace holds the scores of all visible keys (4 bytes per query head and token
 * of the bound on a row): give max_context_len where the block table is wide.  workspace NULL: stream-ordered memory,
 * or FFKV_ERR_WORKSPACE where the stream is being captured (and any is needed).  The calls that share a workspace must not
 * overlap in time.
 */
FFKV_API size_t ffkv_decode_scored_workspace_bytes(int batch, int num_heads, int head_dim, int max_blocks,
                                                   int max_context_len, int with_weights);

FFKV_API size_t ffkv_decode_scored_scratch_bytes(int qo_dtype, int cache_dtype, int batch, int num_heads, int num_kv_heads,
                                                 int head_dim, int max_blocks, int max_context_len, int window,
                                                 int with_weights);

FFKV_API int ffkv_paged_decode_scored(const void* q, void* out, int qo_dtype, void* k_cache, void* v_cache,
                                      int cache_dtype, float* k_scale, float* v_scale, const int32_t* block_table,
                                      const int32_t* context_lens, int batch, int num_heads, int num_kv_heads,
                                      int head_dim, int block_size, int max_blocks, int num_blocks, int max_context_len,
                                      float scale, float score_cap, const float* slopes, int window,
                                      const int32_t* key_begin, const void* k_new, const void* v_new, int src_dtype,
                                      float* weights, const float* prior, float decay, int64_t weight_stride,
                                      void* workspace, size_t workspace_bytes, void* stream);

/*
 * ffkv_paged_prefill_ws under a score rule (see above): query token t of row b at position i = context_lens[b] + t (t
 * without a block table) sees the keys j of its row with lo <= j < hi,
 *   lo = max(0, key_begin[b, t], i - window + 1),  hi = min(the row's tokens, key_end[b, t])  (key_end NULL: i + 1, causal)
 * where the row's tokens are those that ffkv_paged_prefill attends at most, context_lens[b] + seq_len, cut at
 * max_context_len.  key_begin / key_end int32 [batch, seq_len], either or both NULL: documents in one row (begin of the
 * query's document), prefixes that all queries see (end = max(prefix, i + 1)), documents seen both ways (end of the
 * document), queries that see nothing (end 0, padding).  A query's visible keys may lie after it; distances are |i - j|.
 * Unlike in ffkv_paged_prefill, an infinite or NaN V value reaches only the queries that see its key (a workgroup that
 * meets one reruns).  V ranges, types, head dims, workspace and errors as for ffkv_paged_prefill_ws; with_key_end: whether
 * the call has a key_end.
 */
FFKV_API size_t ffkv_prefill_scored_workspace_bytes(int qo_dtype, int cache_dtype, int batch, int seq_len, int num_heads,
                                                    int num_kv_heads, int head_dim, int paged, int max_blocks,
                                                    int max_context_len, int window, int with_key_end);

FFKV_API int ffkv_paged_prefill_scored(const void* q, void* out, int qo_dtype, const void* k_cache, const void* v_cache,
                                       int cache_dtype, const float* k_scale, const float* v_scale,
                                       const int32_t* block_table, const int32_t* context_lens, int batch, int seq_len,
                                       int num_heads, int num_kv_heads, int head_dim, int block_size, int max_blocks,
                                       int num_blocks, int max_context_len, float scale, float score_cap,
                                       const float* slopes, int window, const int32_t* key_begin, const int32_t* key_end,
                                       void* workspace, size_t workspace_bytes, void* stream);

/*
 * The attention weights that the last seq_len tokens of every row give to its cached keys, summed over them and over the
 * query heads of a KV head, under a score rule (see ffkv_paged_prefill_scored, whose q, context_lens, key_begin and key_end
 * these are; the keys must be appended):
 *   weights[b, kvh, j] = decay * prior[b, kvh, j] + sum of softmax(s)_j    j < context_lens[b]
 *   weights[b, kvh, j] = sum of softmax(s)_j                               the seq_len tokens' own keys
 * weights and prior as for ffkv_paged_decode_scored, which gives the same for single tokens beside the attention itself;
 * this call reads no V and writes no output: the prompt's part of what ffkv_evict goes by (the last 16 to 64 tokens of a
 * prompt, a few queries of a chunk).  seq_len 0: the earlier weights' decay alone.  Caches, head dims and GQA groups as for ffkv_paged_decode_scored, any group size.
 * Workspace: ffkv_attention_weights_workspace_bytes, or NULL as for ffkv_paged_decode_scored; calls that share one must not
 * overlap in time.  No counterpart in the reference.
 */
FFKV_API size_t ffkv_attention_weights_workspace_bytes(int batch, int seq_len, int num_heads, int num_kv_heads,
                                                       int head_dim, int max_blocks, int max_context_len);

FFKV_API int ffkv_attention_weights(const void* q, int qo_dtype, const void* k_cache, int cache_dtype, const float* k_scale,
                                    const int32_t* block_table, const int32_t* context_lens, int batch, int seq_len,
                                    int num_heads, int num_kv_heads, int head_dim, int block_size, int max_blocks,
                                    int num_blocks, int max_context_len, float scale, float score_cap,
                                    const float* slopes, int window, const int32_t* key_begin, const int32_t* key_end,
                                    float* weights, const float* prior, float decay, int64_t weight_stride,
                                    void* workspace, size_t workspace_bytes, void* stream);

/*
 * Eviction from the cache by attention weight.  Row b holds context_lens[b] tokens (all appended; clamped to what its
 * block table and weight_stride hold), whose weights per KV head are weights fp32 [batch, num_kv_heads, weight_stride], as
 * ffkv_paged_decode_scored and ffkv_attention_weights leave them.  A row of more than `keep` tokens keeps, per KV head, its
 * first `sinks` and its last `recent` tokens and of those between the keep - sinks - recent with the largest weights (of
 * equal weights the earlier token stays; NaN is the least); a shorter row keeps all.  Then
 *   kept       int32 [batch, num_kv_heads, keep]: the kept tokens' positions in ascending order (entries past the row's
 *              count are left as they were)
 *   kept_lens  int32 [batch]: min(context_lens[b], keep), the row's tokens from now on; not context_lens itself
 *   K and V (and int8 scales) of kept token number j go to position j of the row in dst_table int32 [batch, dst_blocks],
 *              pages of the same pools that no row of the call holds tokens in (pages shared with other rows stay whole;
 *              block_table itself is refused);
 *              dst_table NULL: to position j of the row's own pages, which no other row may hold then
 *   weights_out fp32 [batch, num_kv_heads, out_stride], NULL or weights itself (with its stride) or apart from it: the kept
 *              tokens' weights at their new positions, the rest left as it was
 * Each KV head keeps tokens of its own: position j of a row then holds different tokens in different heads, each with the
 * rotary embedding it was cached with, and the row goes on from position kept_lens[b] (the new tokens' rotary positions
 * go on from the old ones).  A kept token whose source or destination page is absent is not copied.  keep >= 1, sinks
 * and recent >= 0 and together at most keep.  Cache types, head dims and alignment as for ffkv_append.  Workspace:
 * ffkv_evict_workspace_bytes (0 but for few rows over a long bound), or NULL as for ffkv_paged_decode_scored; calls that share
 * one must not overlap in time.  No counterpart in the reference, which evicts whole prefix-cache nodes that no request
 * uses (src/radix_tree.cc).
 */
FFKV_API size_t ffkv_evict_workspace_bytes(int batch, int num_kv_heads, int keep, int64_t weight_stride, int max_blocks);

FFKV_API int ffkv_evict(const float* weights, int64_t weight_stride, const int32_t* context_lens, int keep, int sinks,
                        int recent, void* k_cache, void* v_cache, int cache_dtype, float* k_scale, float* v_scale,
                        const int32_t* block_table, int max_blocks, const int32_t* dst_table, int dst_blocks,
                        int32_t* kept, int32_t* kept_lens, float* weights_out, int64_t out_stride, int batch,
                        int num_kv_heads, int head_dim, int block_size, int num_blocks, void* workspace,
                        size_t workspace_bytes, void* stream);

/* ---- positions on several axes, and attention over selected pages (no counterpart in the reference) ------------------ */

/*
 * Rotary embedding by positions on several axes (time, height and width of image and video tokens).  Pair i of a head (dims
 * i, i + head_dim/2) of token t of row b turns by positions[axis(i)][b][t] * rope_theta^(-2i/head_dim), in ffkv_rope's form;
 * with equal positions on all axes that is ffkv_rope's rotation.  positions int32 [axes, batch, seq_len]; axes 1 to 4; sections
 * (host memory): the pairs of dims of each axis, head_dim/2 together.  interleaved 0: the first sections[0] pairs turn by axis 0,
 * the next sections[1] by axis 1, ..; else pair i turns by axis i % axes while that axis has pairs left (sections[a] of the
 * pairs a, a + axes, ..), all others by axis 0.  The turns are one fp64 product, whose fraction enters cos and sin: good to
 * 2^-22 + |position| * 2^-48 (rope_theta >= 1).  (ffkv_rope rounds its angle to fp32: far positions differ by 2^-24 of the
 * angle.)
 *
 * q [batch, seq_len, num_heads, head_dim] (NULL: none) and k [batch, seq_len, num_kv_heads, head_dim] of one dtype (F32, F16,
 * BF16), head_dim 64, 128 or 256; q_stride etc.: elements from token to token (0: one behind the other; a view into a packed
 * projection has the projection's width), a multiple of 16 bytes; row b's tokens begin batch-contiguously, seq_len * stride
 * behind row b - 1's; batch * seq_len up to 2^29 - 1.  q_out and k_out: q and k themselves (in place, with their strides) or
 * memory that overlaps neither.
 */
FFKV_API int ffkv_rope_axes(const void* q, int64_t q_stride, void* q_out, int64_t q_out_stride, const void* k,
                            int64_t k_stride, void* k_out, int64_t k_out_stride, int dtype, const int32_t* positions,
                            const int* sections, int axes, int interleaved, int batch, int seq_len, int num_heads,
                            int num_kv_heads, int head_dim, float rope_theta, void* stream);

/*
 * ffkv_rope_axes and ffkv_append of the rotated k (as rounded in src_dtype) and v in one pass.  Token t of row b goes to cache
 * position context_lens[b] + t (NULL: t), whatever its positions on the axes are.  k and v are only read: the rotated k is in
 * the pages alone.  The pages are those of ffkv_rope_axes followed by ffkv_append.
 */
FFKV_API int ffkv_rope_append_axes(const void* q, int64_t q_stride, void* q_out, int64_t q_out_stride, const void* k,
                                   int64_t k_stride, const void* v, int64_t v_stride, int src_dtype, void* k_cache,
                                   void* v_cache, int cache_dtype, float* k_scale, float* v_scale,
                                   const int32_t* block_table, const int32_t* context_lens, const int32_t* positions,
                                   const int* sections, int axes, int interleaved, int batch, int seq_len, int num_heads,
                                   int num_kv_heads, int head_dim, int block_size, int max_blocks, int num_blocks,
                                   float rope_theta, void* stream);

/*
 * Key bounds of the pages that the new_tokens tokens from position context_lens[b] on of every row lie on (already appended):
 * for each KV head and dim the smallest and the largest key of the page's tokens of the row, earlier ones included, into
 * bounds [num_blocks, num_kv_heads, 2, head_dim] (lo, then hi).  bounds have the cache's type, or bf16 beside int8 and fp8
 * caches, there rounded outward.  A NaN key gives NaN bounds.  Call it after every append; pages without their row's later
 * tokens (a prefix that rows share, once full) keep their bounds.  Pages on no block-table entry are skipped.
 */
FFKV_API int ffkv_key_bounds(const void* k_cache, int cache_dtype, const float* k_scale, void* bounds,
                             const int32_t* block_table, const int32_t* context_lens, int batch, int new_tokens,
                             int num_kv_heads, int head_dim, int block_size, int max_blocks, int num_blocks, void* stream);

/*
 * Which pages to attend: for every block of query_block query tokens (the last may be shorter) and KV head, `count` logical
 * pages of the row.  Queries q [batch, seq_len, num_heads, head_dim] sit at positions context_lens[b] + t.  Of the pages up to
 * the block's last query's, the first `sinks` and the last `recent` are taken, and of the rest those with the largest
 *     score(page) = sum over the block's queries and the KV head's query heads of sum_d max(q_d lo_d, q_d hi_d)
 * (sums in fp64, rounded once to fp32; of equal scores the lower page; NaN counts as the largest, 0 times an infinite bound as
 * 0; a page on no block-table entry as the lowest).  A row's choice does not depend on the call's other rows.  count up to 2^26,
 * num_blocks at least 1; more lists than one launch takes (4 to 16 million) are refused.  blocks int32 [batch,
 * ceil(seq_len / query_block), num_kv_heads, count]: ascending, -1 behind a row of fewer pages.  `recent` pages count back from the
 * block's last query: with query_block > 1 give at least (query_block + 14) / 16 + 1 for every query to have its own page.
 * bounds_dtype F32, F16 or BF16 (ffkv_key_bounds' type).  max_context_len bounds the rows' tokens, this call's included (0: the
 * table's width); pages past it are not taken.  workspace: NULL or ffkv_select_blocks_workspace_bytes (a captured call needs one
 * where that is not 0).
 */
FFKV_API size_t ffkv_select_blocks_workspace_bytes(int batch, int seq_len, int num_heads, int num_kv_heads, int head_dim,
                                                   int count, int query_block, int max_blocks, int max_context_len);

FFKV_API int ffkv_select_blocks(const void* q, int q_dtype, const void* bounds, int bounds_dtype, const int32_t* block_table,
                                const int32_t* context_lens, int32_t* blocks, int count, int sinks, int recent,
                                int query_block, int batch, int seq_len, int num_heads, int num_kv_heads, int head_dim,
                                int block_size, int max_blocks, int num_blocks, int max_context_len, void* workspace,
                                size_t workspace_bytes, void* stream);

/*
 * Causal attention over listed pages alone: query token t of row b at position context_lens[b] + t attends the tokens up to
 * its own of the pages that blocks[b][t / query_block][kv_head] lists (int32 [batch, ceil(seq_len / query_block), num_kv_heads,
 * count], as ffkv_select_blocks gives them).  Lists may be in any order; entries outside [0, max_blocks), on no block-table
 * entry or past the query count for nothing, and a page listed twice counts twice.  A query without any key gives zeros.  What
 * a query does not attend never reaches it, infinite and NaN values included.  q, out [batch, seq_len, num_heads, head_dim];
 * caches as ffkv_paged_decode takes them (all types; every query_block), count up to 2^26.  The tokens are already appended.
 * workspace: NULL or ffkv_paged_attention_blocks_workspace_bytes (0 but for few lists, which are then split; a captured call
 * without one leaves them whole).
 */
FFKV_API size_t ffkv_paged_attention_blocks_workspace_bytes(int qo_dtype, int cache_dtype, int batch, int seq_len,
                                                            int num_heads, int num_kv_heads, int head_dim, int count,
                                                            int query_block);

FFKV_API int ffkv_paged_attention_blocks(const void* q, void* out, int qo_dtype, const void* k_cache, const void* v_cache,
                                         int cache_dtype, const float* k_scale, const float* v_scale,
                                         const int32_t* block_table, const int32_t* context_lens, const int32_t* blocks,
                                         int count, int query_block, int batch, int seq_len, int num_heads,
                                         int num_kv_heads, int head_dim, int block_size, int max_blocks, int num_blocks,
                                         float scale, void* workspace, size_t workspace_bytes, void* stream);

/* Message describing the last error returned on the calling thread ("" if none). */
FFKV_API const char* ffkv_last_error(void);

/* Library version string. */
FFKV_API const char* ffkv_version(void);

#ifdef __cplusplus
}
#endif

#endif /* FFKV_H_ */
