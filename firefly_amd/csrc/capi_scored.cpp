// capi_scored.cpp - the extern "C" boundary of attention under a score rule, attention weights and cache eviction
// (include/ffkv.h): argument validation, workspaces and error reporting around the HIP launchers.
#include <algorithm>
#include <climits>
#include <cmath>

#include "capi_util.h"

using namespace ffkv::capi;

namespace
{

constexpr float kLog2e = 1.4426950408889634f;

float softmax_scale(float scale, int head_dim)
{
    return scale > 0.0f ? scale : 1.0f / sqrtf(static_cast<float>(head_dim));
}

// The rule's own arguments; FFKV_OK or the error.
int check_rule(float score_cap, const float* slopes, int window, const int32_t* key_begin, const int32_t* key_end)
{
    if (!(score_cap >= 0.0f) || std::isinf(score_cap))
        return fail(FFKV_ERR_INVALID_ARGUMENT, "score_cap must be finite and not negative, got %g",
                    static_cast<double>(score_cap));
    if (window < 0) return fail(FFKV_ERR_INVALID_ARGUMENT, "window must not be negative, got %d", window);
    if (!aligned4(slopes) || !aligned4(key_begin) || !aligned4(key_end))
        return fail(FFKV_ERR_INVALID_ARGUMENT, "slopes, key_begin and key_end must be 4-byte aligned");
    return FFKV_OK;
}

ffkv::ScoreRule make_rule(float score_cap, const float* slopes, int window, const int32_t* key_begin,
                          const int32_t* key_end)
{
    ffkv::ScoreRule r{};
    r.cap = score_cap * kLog2e;  // the kernels' scores are in log2 units
    if (score_cap > 0.0f) r.cap = std::max(r.cap, 1e-30f);  // (its inverse stays far from infinity; below it all scores are as good as 0)
    if (!std::isfinite(r.cap)) r.cap = 0.0f;                // beyond fp32: no score reaches it
    r.inv_cap = r.cap > 0.0f ? 1.0f / r.cap : 0.0f;
    r.window = window;
    r.slopes = slopes;
    r.key_begin = key_begin;
    r.key_end = key_end;
    return r;
}

int check_weights(const float* weights, const float* prior, float decay, int64_t weight_stride, int cap_tokens)
{
    if (prior != nullptr && weights == nullptr) return fail(FFKV_ERR_INVALID_ARGUMENT, "prior without weights");
    if (weights == nullptr) return FFKV_OK;
    if (!(decay >= 0.0f) || std::isinf(decay))
        return fail(FFKV_ERR_INVALID_ARGUMENT, "decay must be finite and not negative, got %g", static_cast<double>(decay));
    if (weight_stride < cap_tokens)
        return fail(FFKV_ERR_INVALID_ARGUMENT, "weight_stride %lld is less than the rows' bound of %d tokens",
                    static_cast<long long>(weight_stride), cap_tokens);
    if (!aligned4(weights) || !aligned4(prior))
        return fail(FFKV_ERR_INVALID_ARGUMENT, "weights and prior must be 4-byte aligned");
    return FFKV_OK;
}

// The matrix-core decode takes it (whatever kernel the plain decode is forced to).
bool scored_mfma(int cache_dtype, int head_dim)
{
    return cache_dtype != FFKV_DTYPE_F32 && (head_dim_mfma(head_dim) || head_dim == 80 || head_dim == 96 || head_dim == 112);
}

// Regions of the weights' pass behind the decode's partials: scores (stride tokens per row and query head) and final states
// [batch, num_heads, 2].
struct ScoreLayout
{
    int64_t stride, scores, final, total;
};

constexpr double kMostBytes = 1e15;

ScoreLayout score_layout(int64_t at, int batch, int num_heads, int cap_tokens)
{
    ScoreLayout l{};
    l.stride = ceil_div(cap_tokens, FFKV_BLOCK_SIZE) * FFKV_BLOCK_SIZE;
    l.scores = align256(at);
    l.final = l.scores + align256(static_cast<int64_t>(batch) * num_heads * l.stride * 4);
    l.total = l.final + align256(static_cast<int64_t>(batch) * num_heads * 8);
    return l;
}

bool score_layout_fits(int batch, int num_heads, int cap_tokens)
{
    return 4.0 * batch * num_heads * (static_cast<double>(cap_tokens) + 16) < kMostBytes;
}

// Most keys that a block of 128 query rows sees: a window's of its tokens, else the row's bound.
int prefill_span(int cap_tokens, int group, int window, bool key_end)
{
    if (window <= 0 || key_end) return cap_tokens;
    return static_cast<int>(std::min<int64_t>(cap_tokens, static_cast<int64_t>(window) + 128 / group + 2 * FFKV_BLOCK_SIZE));
}

// Stream-ordered memory for a call without a workspace; not while the stream is being captured (is_capturing).
int take_memory(void** ws, int64_t bytes, hipStream_t s)
{
    bool capturing = false;
    if (const int rc = is_capturing(s, capturing)) return rc;
    if (capturing)
        return fail(FFKV_ERR_WORKSPACE, "a captured call needs a workspace, of %lld bytes", static_cast<long long>(bytes));
    const hipError_t e = hipMallocAsync(ws, static_cast<size_t>(bytes), s);
    return e == hipSuccess ? FFKV_OK : hip_fail(e, "workspace hipMallocAsync");
}

// What a scored decode launches and holds in its workspace; sizes and types of `a` are set.
struct DecodePlan
{
    bool             mfma, row;
    ffkv::MfmaLayout lay;
    ScoreLayout      scores;
    int64_t          need;
};

DecodePlan plan_decode(ffkv::ScoredDecodeArgs& a, int cap_tokens, int window, bool with_weights)
{
    DecodePlan p{};
    a.group = a.num_heads / a.num_kv_heads;
    p.mfma = scored_mfma(a.cache_dtype, a.head_dim);
    a.chunk = ffkv::decode_chunk(a.batch, a.num_kv_heads, cap_tokens);
    a.max_chunks = static_cast<int>(ceil_div(cap_tokens > 0 ? cap_tokens : 1, a.chunk));
    // Tokens that a row's query sees at most: a window's, which may begin and end inside a page.  The plain decode's rules
    // for the number of work items and for its one-launch form go by these.
    const int span =
        window > 0 ? static_cast<int>(std::min<int64_t>(cap_tokens, static_cast<int64_t>(window) + 2 * FFKV_BLOCK_SIZE))
                   : cap_tokens;
    a.cap_tokens = span;
    p.row = p.mfma && ffkv::decode_use_row(a);
    if (p.mfma) a.items = std::min(ffkv::decode_scored_launch_items(a), ffkv::decode_most_items(a.batch, span));
    a.cap_tokens = cap_tokens;
    if (p.mfma && !p.row)
    {
        p.lay = ffkv::mfma_layout(a.batch, a.num_heads, a.head_dim, 0, a.items);
        p.need = p.lay.total;
    }
    else if (!p.mfma && a.max_chunks > 1)
    {
        const int64_t parts = static_cast<int64_t>(a.batch) * a.num_heads * a.max_chunks;
        p.lay.acc = align256(parts * 2 * 4);
        p.need = p.lay.acc + parts * a.head_dim * 4;
    }
    if (with_weights)
    {
        p.scores = score_layout(p.need, a.batch, a.num_heads, cap_tokens);
        p.need = p.scores.total;
    }
    return p;
}

// The attention weights' workspace: the query rows' states per split of the keys, and folded.
struct WeightLayout
{
    int     splits;
    int64_t part, fin, total;
};

WeightLayout weight_layout(int batch, int seq_len, int num_heads, int num_kv_heads, int head_dim, int cap_tokens)
{
    const int64_t rows = static_cast<int64_t>(batch) * seq_len * num_heads;
    WeightLayout  l{};
    l.splits = ffkv::attention_weights_splits(batch, num_kv_heads, head_dim, cap_tokens);
    l.fin = align256(rows * l.splits * 8);
    l.total = l.fin + align256(rows * 8);
    return l;
}

// The eviction's workspace for long rows (evict.hip); nothing for others.
struct EvictLayout
{
    int     parts;
    int64_t hist0, hist1, state, above, scratch, total;
};

EvictLayout evict_layout(int batch, int num_kv_heads, int keep, int64_t bound)
{
    EvictLayout l{};
    l.parts = ffkv::evict_parts(batch, num_kv_heads, bound);
    if (l.parts == 0) return l;
    const int64_t bh = static_cast<int64_t>(batch) * num_kv_heads;
    l.hist0 = 0;
    l.hist1 = l.hist0 + bh * l.parts * 2048 * 4;
    l.state = l.hist1 + bh * l.parts * 2048 * 4;
    l.above = l.state + align256(bh * 2 * 2 * 4);
    l.scratch = l.above + align256(bh * l.parts * 2 * 4);
    l.total = l.scratch + align256(bh * std::min<int64_t>(keep, bound) * 4);
    return l;
}

}  // namespace

extern "C" {

size_t ffkv_decode_scored_workspace_bytes(int batch, int num_heads, int head_dim, int max_blocks, int max_context_len,
                                          int with_weights)
{
    const size_t plain = ffkv_decode_workspace_bytes(batch, num_heads, head_dim, max_blocks, max_context_len);
    if (plain == 0 || with_weights == 0) return plain;
    const int cap = ffkv::decode_cap_tokens(max_blocks, max_context_len);
    if (!score_layout_fits(batch, num_heads, cap)) return 0;  // refused by the call
    return static_cast<size_t>(score_layout(static_cast<int64_t>(plain), batch, num_heads, cap).total);
}

size_t ffkv_decode_scored_scratch_bytes(int qo_dtype, int cache_dtype, int batch, int num_heads, int num_kv_heads,
                                        int head_dim, int max_blocks, int max_context_len, int window, int with_weights)
{
    // sizes that ffkv_paged_decode_scored refuses need nothing
    if (!is_act(qo_dtype) || !is_cache(cache_dtype) || !head_dim_ok(head_dim) || batch <= 0 || batch > 65535 ||
        num_heads <= 0 || num_heads > 65535 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0 || max_blocks < 0 || window < 0)
        return 0;
    const int cap = ffkv::decode_cap_tokens(max_blocks, max_context_len);
    if (with_weights != 0 && !score_layout_fits(batch, num_heads, cap)) return 0;
    ffkv::ScoredDecodeArgs a{};
    a.qo_dtype = qo_dtype;
    a.cache_dtype = cache_dtype;
    a.batch = batch;
    a.num_heads = num_heads;
    a.num_kv_heads = num_kv_heads;
    a.head_dim = head_dim;
    return static_cast<size_t>(plan_decode(a, cap, window, with_weights != 0).need);
}

int ffkv_paged_decode_scored(const void* q, void* out, int qo_dtype, void* k_cache, void* v_cache, int cache_dtype,
                             float* k_scale, float* v_scale, const int32_t* block_table, const int32_t* context_lens,
                             int batch, int num_heads, int num_kv_heads, int head_dim, int block_size, int max_blocks,
                             int num_blocks, int max_context_len, float scale, float score_cap, const float* slopes,
                             int window, const int32_t* key_begin, const void* k_new, const void* v_new, int src_dtype,
                             float* weights, const float* prior, float decay, int64_t weight_stride, void* workspace,
                             size_t workspace_bytes, void* stream)
{
    if (block_size != FFKV_BLOCK_SIZE) return fail(FFKV_ERR_UNSUPPORTED, "block_size must be 16, got %d", block_size);
    if (!is_act(qo_dtype)) return fail(FFKV_ERR_UNSUPPORTED, "unsupported q/out dtype %d", qo_dtype);
    if (!is_cache(cache_dtype)) return fail(FFKV_ERR_UNSUPPORTED, "unsupported cache dtype %d", cache_dtype);
    if (!head_dim_ok(head_dim))
        return fail(FFKV_ERR_UNSUPPORTED, "head_dim must be a multiple of 8 up to 128, or 256, got %d", head_dim);
    if (batch < 0 || num_heads <= 0 || num_kv_heads <= 0 || max_blocks < 0 || num_blocks < 0)
        return fail(FFKV_ERR_INVALID_ARGUMENT, "bad size (batch %d heads %d kv_heads %d max_blocks %d num_blocks %d)",
                    batch, num_heads, num_kv_heads, max_blocks, num_blocks);
    if (num_heads % num_kv_heads != 0)
        return fail(FFKV_ERR_INVALID_ARGUMENT, "num_heads %d is not a multiple of num_kv_heads %d", num_heads,
                    num_kv_heads);
    const int  group = num_heads / num_kv_heads;
    const bool mfma = scored_mfma(cache_dtype, head_dim);
    if (group > 16 && !mfma)
        return fail(FFKV_ERR_UNSUPPORTED, "GQA group size %d exceeds 16 (fp32 caches, or this head_dim)", group);
    if (batch > 65535 || num_heads > 65535)
        return fail(FFKV_ERR_UNSUPPORTED, "batch and num_heads must be <= 65535");
    if (const int rc = check_rule(score_cap, slopes, window, key_begin, nullptr)) return rc;
    if ((k_new == nullptr) != (v_new == nullptr))
        return fail(FFKV_ERR_INVALID_ARGUMENT, "k_new and v_new come together");
    if (k_new != nullptr && !is_act(src_dtype)) return fail(FFKV_ERR_UNSUPPORTED, "unsupported source dtype %d", src_dtype);
    const int cap = ffkv::decode_cap_tokens(max_blocks, max_context_len);
    if (const int rc = check_weights(weights, prior, decay, weight_stride, cap)) return rc;
    if (batch == 0) return ok();
    if (!q || !out || !k_cache || !v_cache || !block_table || !context_lens)
        return fail(FFKV_ERR_INVALID_ARGUMENT, "null q, out, cache, block_table or context_lens pointer");
    if (quantized(cache_dtype) && (!k_scale || !v_scale))
        return fail(FFKV_ERR_INVALID_ARGUMENT, "quantized cache needs k_scale and v_scale");
    if (!aligned16(q) || !aligned16(out) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(k_new) ||
        !aligned16(v_new))
        return fail(FFKV_ERR_INVALID_ARGUMENT, "q, out, cache, k_new and v_new pointers must be 16-byte aligned");
    if (static_cast<int64_t>(batch) * ceil_div(cap, FFKV_BLOCK_SIZE) > INT32_MAX)
        return fail(FFKV_ERR_UNSUPPORTED, "batch * pages per row exceeds 2^31 - 1 (batch %d, %d tokens per row)",
                    batch, cap);
    if (weights != nullptr && !score_layout_fits(batch, num_heads, cap))
        return fail(FFKV_ERR_UNSUPPORTED, "the scores of %d x %d rows of %d tokens are too many: give max_context_len",
                    batch, num_heads, cap);

    ffkv::ScoredDecodeArgs a{};
    a.q = q;
    a.out = out;
    a.k_cache = k_cache;
    a.v_cache = v_cache;
    a.k_scale = k_scale;
    a.v_scale = v_scale;
    a.block_table = block_table;
    a.context_lens = context_lens;
    a.qo_dtype = qo_dtype;
    a.cache_dtype = cache_dtype;
    a.batch = batch;
    a.num_heads = num_heads;
    a.num_kv_heads = num_kv_heads;
    a.group = group;
    a.head_dim = head_dim;
    a.max_blocks = max_blocks;
    a.num_blocks = num_blocks;
    a.scale_log2 = softmax_scale(scale, head_dim) * kLog2e;
    a.rule = make_rule(score_cap, slopes, window, key_begin, nullptr);

    const DecodePlan       plan = plan_decode(a, cap, window, weights != nullptr);
    const ffkv::MfmaLayout lay = plan.lay;
    const ScoreLayout      sl = plan.scores;
    const bool             row = plan.row;
    const int64_t          need = plan.need;
    hipStream_t s = static_cast<hipStream_t>(stream);
    void*       ws = workspace;
    bool        owned = false;
    if (ws != nullptr && !aligned16(ws)) return fail(FFKV_ERR_INVALID_ARGUMENT, "workspace must be 16-byte aligned");
    if (ws != nullptr && workspace_bytes < static_cast<size_t>(need))
        return fail(FFKV_ERR_WORKSPACE, "workspace of %zu bytes is smaller than the %lld bytes needed", workspace_bytes,
                    static_cast<long long>(need));
    if (ws == nullptr && need > 0)
    {
        if (const int rc = take_memory(&ws, need, s)) return rc;
        owned = true;
    }
    char* wsb = static_cast<char*>(ws);
    if (mfma && !row) a.ws_meta = reinterpret_cast<int32_t*>(wsb + lay.meta);
    if (lay.acc > 0)
    {
        a.ws_ml = reinterpret_cast<float*>(wsb + lay.ml);
        a.ws_acc = reinterpret_cast<float*>(wsb + lay.acc);
    }
    if (weights != nullptr)
    {
        a.ws_scores = reinterpret_cast<float*>(wsb + sl.scores);
        a.ws_final = reinterpret_cast<float*>(wsb + sl.final);
        a.score_stride = sl.stride;
        a.weights = weights;
        a.prior = prior;
        a.decay = decay;
        a.weight_stride = weight_stride;
    }

    hipError_t e = hipSuccess;
    if (k_new != nullptr)
    {
        if (mfma && src_dtype == cache_dtype)  // 16-bit: the decode kernel writes the step's token to its page and attends it
        {
            a.k_new = k_new;
            a.v_new = v_new;
        }
        else
        {
            ffkv::AppendArgs ap{k_new, v_new, k_cache, v_cache, k_scale, v_scale, block_table, context_lens, src_dtype,
                                cache_dtype, batch, 1, num_kv_heads, head_dim, max_blocks, num_blocks};
            e = ffkv::launch_append(ap, s);
        }
    }
    if (e == hipSuccess) e = ffkv::launch_decode_scored(a, mfma, row, s);
    if (owned)
    {
        const hipError_t fe = hipFreeAsync(ws, s);
        if (e == hipSuccess) e = fe;
    }
    if (e != hipSuccess) return hip_fail(e, "scored decode launch");
    return ok();
}

size_t ffkv_prefill_scored_workspace_bytes(int qo_dtype, int cache_dtype, int batch, int seq_len, int num_heads,
                                           int num_kv_heads, int head_dim, int paged, int max_blocks,
                                           int max_context_len, int window, int with_key_end)
{
    // sizes that ffkv_paged_prefill_scored refuses need nothing
    if (!is_act(qo_dtype) || !is_cache(cache_dtype) || cache_dtype == FFKV_DTYPE_F32 || !head_dim_mfma(head_dim) ||
        batch <= 0 || batch > 65535 || seq_len <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_kv_heads > 65535 ||
        num_heads % num_kv_heads != 0 || (paged != 0 && max_blocks < 0) || window < 0)
        return 0;
    ffkv::ScoredPrefillArgs a{};
    a.qo_dtype = qo_dtype;
    a.cache_dtype = cache_dtype;
    a.batch = batch;
    a.seq_len = seq_len;
    a.num_heads = num_heads;
    a.num_kv_heads = num_kv_heads;
    a.group = num_heads / num_kv_heads;
    a.head_dim = head_dim;
    a.paged = paged != 0;
    a.cap_tokens = a.paged ? ffkv::decode_cap_tokens(max_blocks, max_context_len) : seq_len;
    a.span_tokens = prefill_span(a.cap_tokens, a.group, window, with_key_end != 0);
    ffkv::prefill_scored_plan(a);
    return static_cast<size_t>(ffkv::prefill_split_layout(a).total);
}

int ffkv_paged_prefill_scored(const void* q, void* out, int qo_dtype, const void* k_cache, const void* v_cache,
                              int cache_dtype, const float* k_scale, const float* v_scale, const int32_t* block_table,
                              const int32_t* context_lens, int batch, int seq_len, int num_heads, int num_kv_heads,
                              int head_dim, int block_size, int max_blocks, int num_blocks, int max_context_len,
                              float scale, float score_cap, const float* slopes, int window, const int32_t* key_begin,
                              const int32_t* key_end, void* workspace, size_t workspace_bytes, void* stream)
{
    const bool paged = block_table != nullptr;
    if (block_size != FFKV_BLOCK_SIZE) return fail(FFKV_ERR_UNSUPPORTED, "block_size must be 16, got %d", block_size);
    if (!is_act(qo_dtype)) return fail(FFKV_ERR_UNSUPPORTED, "unsupported q/out dtype %d", qo_dtype);
    if (!is_cache(cache_dtype) || cache_dtype == FFKV_DTYPE_F32)
        return fail(FFKV_ERR_UNSUPPORTED, "prefill supports F16, BF16, I8 and FP8_E4M3 caches, got dtype %d",
                    cache_dtype);
    if (!head_dim_mfma(head_dim)) return fail(FFKV_ERR_UNSUPPORTED, "head_dim must be 64, 128 or 256, got %d", head_dim);
    if (batch < 0 || seq_len < 0 || num_heads <= 0 || num_kv_heads <= 0 || (paged && (max_blocks < 0 || num_blocks < 0)))
        return fail(FFKV_ERR_INVALID_ARGUMENT, "bad size (batch %d seq_len %d heads %d kv_heads %d max_blocks %d "
                    "num_blocks %d)", batch, seq_len, num_heads, num_kv_heads, max_blocks, num_blocks);
    if (num_heads % num_kv_heads != 0)
        return fail(FFKV_ERR_INVALID_ARGUMENT, "num_heads %d is not a multiple of num_kv_heads %d", num_heads,
                    num_kv_heads);
    if (batch > 65535 || num_kv_heads > 65535)
        return fail(FFKV_ERR_UNSUPPORTED, "batch and num_kv_heads must be <= 65535");
    if (static_cast<int64_t>(seq_len) * (num_heads / num_kv_heads) > INT32_MAX - 64)
        return fail(FFKV_ERR_UNSUPPORTED, "seq_len * group too large");
    if (static_cast<int64_t>(batch) * num_kv_heads *
            ((static_cast<int64_t>(seq_len) * (num_heads / num_kv_heads) + 127) / 128) > INT32_MAX - 64 * 1024)
        return fail(FFKV_ERR_UNSUPPORTED, "batch * num_kv_heads * ceil(seq_len * group / 128) too large");
    if (const int rc = check_rule(score_cap, slopes, window, key_begin, key_end)) return rc;
    if (batch == 0 || seq_len == 0) return ok();
    if (!q || !out || !k_cache || !v_cache || (paged && !context_lens))
        return fail(FFKV_ERR_INVALID_ARGUMENT, "null q, out, cache or context_lens pointer");
    if (!paged && cache_dtype == FFKV_DTYPE_I8)
        return fail(FFKV_ERR_UNSUPPORTED, "int8 K/V need a block table (their scales are per page slot)");
    if (quantized(cache_dtype) && (!k_scale || !v_scale))
        return fail(FFKV_ERR_INVALID_ARGUMENT, "quantized cache needs k_scale and v_scale");
    if (!aligned16(q) || !aligned16(out) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(workspace))
        return fail(FFKV_ERR_INVALID_ARGUMENT, "q, out, cache and workspace pointers must be 16-byte aligned");

    ffkv::ScoredPrefillArgs a{};
    a.q = q;
    a.out = out;
    a.k_cache = k_cache;
    a.v_cache = v_cache;
    a.k_scale = k_scale;
    a.v_scale = v_scale;
    a.block_table = block_table;
    a.context_lens = context_lens;
    a.qo_dtype = qo_dtype;
    a.cache_dtype = cache_dtype;
    a.batch = batch;
    a.seq_len = seq_len;
    a.num_heads = num_heads;
    a.num_kv_heads = num_kv_heads;
    a.group = num_heads / num_kv_heads;
    a.head_dim = head_dim;
    a.max_blocks = paged ? max_blocks : 0;
    a.num_blocks = paged ? num_blocks : 0;
    a.cap_tokens = paged ? ffkv::decode_cap_tokens(max_blocks, max_context_len) : seq_len;
    a.paged = paged;
    a.scale_log2 = softmax_scale(scale, head_dim) * kLog2e;
    a.rule = make_rule(score_cap, slopes, window, key_begin, key_end);
    a.span_tokens = prefill_span(a.cap_tokens, a.group, window, key_end != nullptr);
    a.n_split = 1;
    if (workspace != nullptr)
    {
        ffkv::prefill_scored_plan(a);
        const ffkv::PrefillSplitLayout lay = ffkv::prefill_split_layout(a);
        if (a.n_split > 1 && workspace_bytes >= static_cast<size_t>(lay.total))
        {
            char* w = static_cast<char*>(workspace);
            a.ws_pieces = reinterpret_cast<int32_t*>(w + lay.pieces);
            a.ws_ml = reinterpret_cast<float*>(w + lay.ml);
            a.ws_acc = reinterpret_cast<float*>(w + lay.acc);
        }
        else
        {
            a.n_split = 1;
        }
    }
    const hipError_t e = ffkv::launch_prefill_scored(a, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return hip_fail(e, "scored prefill launch");
    return ok();
}

size_t ffkv_attention_weights_workspace_bytes(int batch, int seq_len, int num_heads, int num_kv_heads, int head_dim,
                                              int max_blocks, int max_context_len)
{
    if (batch <= 0 || seq_len <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0 || head_dim <= 0)
        return 0;
    const int cap = ffkv::decode_cap_tokens(max_blocks, max_context_len);
    const WeightLayout l = weight_layout(batch, seq_len, num_heads, num_kv_heads, head_dim, cap);
    return static_cast<size_t>(l.total);
}

int ffkv_attention_weights(const void* q, int qo_dtype, const void* k_cache, int cache_dtype, const float* k_scale,
                           const int32_t* block_table, const int32_t* context_lens, int batch, int seq_len, int num_heads,
                           int num_kv_heads, int head_dim, int block_size, int max_blocks, int num_blocks,
                           int max_context_len, float scale, float score_cap, const float* slopes, int window,
                           const int32_t* key_begin, const int32_t* key_end, float* weights, const float* prior,
                           float decay, int64_t weight_stride, void* workspace, size_t workspace_bytes, void* stream)
{
    if (block_size != FFKV_BLOCK_SIZE) return fail(FFKV_ERR_UNSUPPORTED, "block_size must be 16, got %d", block_size);
    if (!is_act(qo_dtype)) return fail(FFKV_ERR_UNSUPPORTED, "unsupported q dtype %d", qo_dtype);
    if (!is_cache(cache_dtype)) return fail(FFKV_ERR_UNSUPPORTED, "unsupported cache dtype %d", cache_dtype);
    if (!head_dim_ok(head_dim))
        return fail(FFKV_ERR_UNSUPPORTED, "head_dim must be a multiple of 8 up to 128, or 256, got %d", head_dim);
    if (batch < 0 || seq_len < 0 || num_heads <= 0 || num_kv_heads <= 0 || max_blocks < 0 || num_blocks < 0)
        return fail(FFKV_ERR_INVALID_ARGUMENT, "bad size (batch %d seq_len %d heads %d kv_heads %d max_blocks %d "
                    "num_blocks %d)", batch, seq_len, num_heads, num_kv_heads, max_blocks, num_blocks);
    if (num_heads % num_kv_heads != 0)
        return fail(FFKV_ERR_INVALID_ARGUMENT, "num_heads %d is not a multiple of num_kv_heads %d", num_heads,
                    num_kv_heads);
    if (batch > 65535 || num_heads > 65535) return fail(FFKV_ERR_UNSUPPORTED, "batch and num_heads must be <= 65535");
    const int group = num_heads / num_kv_heads;
    if (static_cast<int64_t>(seq_len) * group > (1 << 20))  // 65536 blocks of 16 query rows
        return fail(FFKV_ERR_UNSUPPORTED, "seq_len * group must be <= 2^20");
    if (const int rc = check_rule(score_cap, slopes, window, key_begin, key_end)) return rc;
    const int cap = ffkv::decode_cap_tokens(max_blocks, max_context_len);
    if (batch == 0) return ok();
    if ((seq_len > 0 && !q) || !k_cache || !block_table || !context_lens || !weights)
        return fail(FFKV_ERR_INVALID_ARGUMENT, "null q, cache, block_table, context_lens or weights pointer");
    if (const int rc = check_weights(weights, prior, decay, weight_stride, cap)) return rc;
    if (quantized(cache_dtype) && !k_scale) return fail(FFKV_ERR_INVALID_ARGUMENT, "quantized cache needs k_scale");
    if (!aligned16(q) || !aligned16(k_cache) || !aligned16(workspace))
        return fail(FFKV_ERR_INVALID_ARGUMENT, "q, cache and workspace pointers must be 16-byte aligned");
    if (static_cast<int64_t>(batch) * num_kv_heads * ceil_div(static_cast<int64_t>(seq_len) * group, 16) > INT32_MAX)
        return fail(FFKV_ERR_UNSUPPORTED, "batch * seq_len * num_heads too large");

    const WeightLayout lay = weight_layout(batch, seq_len, num_heads, num_kv_heads, head_dim, cap);
    hipStream_t        s = static_cast<hipStream_t>(stream);
    void*              ws = workspace;
    if (ws != nullptr && workspace_bytes < static_cast<size_t>(lay.total))
        return fail(FFKV_ERR_WORKSPACE, "workspace of %zu bytes is smaller than the %lld bytes needed", workspace_bytes,
                    static_cast<long long>(lay.total));
    if (ws == nullptr && lay.total > 0)
        if (const int rc = take_memory(&ws, lay.total, s)) return rc;
    ffkv::WeightArgs a{};
    a.q = q;
    a.k_cache = k_cache;
    a.k_scale = k_scale;
    a.block_table = block_table;
    a.context_lens = context_lens;
    a.qo_dtype = qo_dtype;
    a.cache_dtype = cache_dtype;
    a.batch = batch;
    a.seq_len = seq_len;
    a.num_heads = num_heads;
    a.num_kv_heads = num_kv_heads;
    a.group = group;
    a.head_dim = head_dim;
    a.max_blocks = max_blocks;
    a.num_blocks = num_blocks;
    a.cap_tokens = cap;
    a.scale_log2 = softmax_scale(scale, head_dim) * kLog2e;
    a.rule = make_rule(score_cap, slopes, window, key_begin, key_end);
    a.splits = lay.splits;
    a.part = reinterpret_cast<float2*>(static_cast<char*>(ws) + lay.part);
    a.fin = reinterpret_cast<float2*>(static_cast<char*>(ws) + lay.fin);
    a.weights = weights;
    a.prior = prior;
    a.decay = decay;
    a.weight_stride = weight_stride;
    hipError_t e = ffkv::launch_attention_weights(a, scored_mfma(cache_dtype, head_dim), s);
    if (workspace == nullptr && ws != nullptr)
    {
        const hipError_t fe = hipFreeAsync(ws, s);
        if (e == hipSuccess) e = fe;
    }
    if (e != hipSuccess) return hip_fail(e, "attention weights launch");
    return ok();
}

size_t ffkv_evict_workspace_bytes(int batch, int num_kv_heads, int keep, int64_t weight_stride, int max_blocks)
{
    if (batch <= 0 || num_kv_heads <= 0 || keep <= 0 || weight_stride <= 0 || max_blocks <= 0) return 0;
    const int64_t bound = std::min<int64_t>(weight_stride, static_cast<int64_t>(max_blocks) * FFKV_BLOCK_SIZE);
    return bound > INT32_MAX - 64 * 1024 ? 0 : static_cast<size_t>(evict_layout(batch, num_kv_heads, keep, bound).total);
}

int ffkv_evict(const float* weights, int64_t weight_stride, const int32_t* context_lens, int keep, int sinks, int recent,
               void* k_cache, void* v_cache, int cache_dtype, float* k_scale, float* v_scale, const int32_t* block_table,
               int max_blocks, const int32_t* dst_table, int dst_blocks, int32_t* kept, int32_t* kept_lens,
               float* weights_out, int64_t out_stride, int batch, int num_kv_heads, int head_dim, int block_size,
               int num_blocks, void* workspace, size_t workspace_bytes, void* stream)
{
    if (block_size != FFKV_BLOCK_SIZE) return fail(FFKV_ERR_UNSUPPORTED, "block_size must be 16, got %d", block_size);
    if (!is_cache(cache_dtype)) return fail(FFKV_ERR_UNSUPPORTED, "unsupported cache dtype %d", cache_dtype);
    if (!head_dim_ok(head_dim))
        return fail(FFKV_ERR_UNSUPPORTED, "head_dim must be a multiple of 8 up to 128, or 256, got %d", head_dim);
    if (batch < 0 || num_kv_heads <= 0 || max_blocks < 0 || num_blocks < 0 || dst_blocks < 0 || weight_stride < 0 ||
        out_stride < 0)
        return fail(FFKV_ERR_INVALID_ARGUMENT, "bad size (batch %d kv_heads %d max_blocks %d dst_blocks %d num_blocks %d)",
                    batch, num_kv_heads, max_blocks, dst_blocks, num_blocks);
    if (batch > 65535 || num_kv_heads > 65535)
        return fail(FFKV_ERR_UNSUPPORTED, "batch and num_kv_heads must be <= 65535");
    if (keep < 1 || sinks < 0 || recent < 0 || static_cast<int64_t>(sinks) + recent > keep)
        return fail(FFKV_ERR_INVALID_ARGUMENT, "keep %d must be at least 1 and hold sinks %d and recent %d", keep, sinks,
                    recent);
    const int64_t bound = std::min<int64_t>(weight_stride, static_cast<int64_t>(max_blocks) * FFKV_BLOCK_SIZE);
    if (bound > INT32_MAX - 64 * 1024) return fail(FFKV_ERR_UNSUPPORTED, "rows of 2^31 tokens");
    if (weights_out != nullptr && out_stride < std::min<int64_t>(keep, bound))
        return fail(FFKV_ERR_INVALID_ARGUMENT, "out_stride %lld is less than the kept tokens",
                    static_cast<long long>(out_stride));
    if (weights_out != nullptr && weights_out == weights && out_stride != weight_stride)
        return fail(FFKV_ERR_INVALID_ARGUMENT, "weights_out in place needs the weights' own stride");
    if (batch == 0) return ok();
    if (!weights || !context_lens || !k_cache || !v_cache || !block_table || !kept || !kept_lens)
        return fail(FFKV_ERR_INVALID_ARGUMENT, "null weights, context_lens, cache, block_table, kept or kept_lens pointer");
    if (kept_lens == context_lens)
        return fail(FFKV_ERR_INVALID_ARGUMENT, "kept_lens must not be context_lens");
    if (dst_table == block_table)
        return fail(FFKV_ERR_INVALID_ARGUMENT, "dst_table must not be block_table: NULL moves within the rows' own pages");
    if (cache_dtype == FFKV_DTYPE_I8 && (!k_scale || !v_scale))
        return fail(FFKV_ERR_INVALID_ARGUMENT, "int8 cache needs k_scale and v_scale");
    if (!aligned16(k_cache) || !aligned16(v_cache) || !aligned16(workspace))
        return fail(FFKV_ERR_INVALID_ARGUMENT, "cache and workspace pointers must be 16-byte aligned");
    if (!aligned4(weights) || !aligned4(weights_out) || !aligned4(kept) || !aligned4(kept_lens))
        return fail(FFKV_ERR_INVALID_ARGUMENT, "weights, kept and kept_lens must be 4-byte aligned");

    ffkv::EvictArgs a{};
    a.weights = weights;
    a.weight_stride = weight_stride;
    a.context_lens = context_lens;
    a.keep = keep;
    a.sinks = sinks;
    a.recent = recent;
    a.k_cache = k_cache;
    a.v_cache = v_cache;
    a.k_scale = k_scale;
    a.v_scale = v_scale;
    a.cache_dtype = cache_dtype;
    a.block_table = block_table;
    a.max_blocks = max_blocks;
    a.dst_table = dst_table;
    a.dst_blocks = dst_blocks;
    a.kept = kept;
    a.kept_lens = kept_lens;
    a.weights_out = weights_out;
    a.out_stride = out_stride;
    a.batch = batch;
    a.num_kv_heads = num_kv_heads;
    a.head_dim = head_dim;
    a.num_blocks = num_blocks;
    const EvictLayout lay = evict_layout(batch, num_kv_heads, keep, bound);
    hipStream_t       s = static_cast<hipStream_t>(stream);
    void*             ws = workspace;
    if (ws != nullptr && workspace_bytes < static_cast<size_t>(lay.total))
        return fail(FFKV_ERR_WORKSPACE, "workspace of %zu bytes is smaller than the %lld bytes needed", workspace_bytes,
                    static_cast<long long>(lay.total));
    if (ws == nullptr && lay.total > 0)
        if (const int rc = take_memory(&ws, lay.total, s)) return rc;
    a.parts = lay.parts;
    if (a.parts > 0)
    {
        char* w = static_cast<char*>(ws);
        a.hist0 = reinterpret_cast<int*>(w + lay.hist0);
        a.hist1 = reinterpret_cast<int*>(w + lay.hist1);
        a.state = reinterpret_cast<uint32_t*>(w + lay.state);
        a.above = reinterpret_cast<int*>(w + lay.above);
        a.scratch = weights_out == weights ? reinterpret_cast<float*>(w + lay.scratch) : nullptr;
    }
    hipError_t e = ffkv::launch_evict(a, s);
    if (workspace == nullptr && ws != nullptr)
    {
        const hipError_t fe = hipFreeAsync(ws, s);
        if (e == hipSuccess) e = fe;
    }
    if (e != hipSuccess) return hip_fail(e, "evict launch");
    return ok();
}

}  // extern "C"
