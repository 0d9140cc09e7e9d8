// capi_blocks.cpp - the extern "C" boundary of rotary positions on several axes, the pages' key bounds, the choice of pages
// and the attention over chosen pages (include/ffkv.h): argument validation, workspaces and error reporting around the HIP
// launchers.
#include <algorithm>
#include <climits>
#include <cmath>

#include "blocks.h"
#include "capi_util.h"

using namespace ffkv::capi;

namespace
{

constexpr float kLog2e = 1.4426950408889634f;

int64_t element_bytes(int dt) { return dt == FFKV_DTYPE_F32 ? 4 : (quantized(dt) ? 1 : 2); }

// A token stride (elements; 0: the tokens lie one behind the other) of `heads` heads; FFKV_OK or the error.
int check_stride(const char* name, int64_t& stride, int heads, int head_dim, int dtype)
{
    const int64_t row = static_cast<int64_t>(heads) * head_dim;
    if (stride == 0) stride = row;
    if (stride < row || stride * element_bytes(dtype) % 16 != 0)
        return fail(FFKV_ERR_INVALID_ARGUMENT, "%s of %lld elements must be at least %lld and a multiple of 16 bytes", name,
                    static_cast<long long>(stride), static_cast<long long>(row));
    return FFKV_OK;
}

// The axes' sections into `a`; FFKV_OK or the error.
int set_sections(ffkv::RopeAxesArgs& a, const int* sections, int axes, int interleaved)
{
    if (axes < 1 || axes > ffkv::kMaxAxes)
        return fail(FFKV_ERR_INVALID_ARGUMENT, "axes must be 1 to %d, got %d", ffkv::kMaxAxes, axes);
    if (sections == nullptr) return fail(FFKV_ERR_INVALID_ARGUMENT, "null sections pointer");
    const int half = a.head_dim / 2;
    int64_t   sum = 0;
    for (int i = 0; i < axes; ++i)
    {
        if (sections[i] < 0) return fail(FFKV_ERR_INVALID_ARGUMENT, "a section has %d pairs", sections[i]);
        sum += sections[i];
    }
    if (sum != half)
        return fail(FFKV_ERR_INVALID_ARGUMENT, "the sections have %lld pairs of dims, not head_dim / 2 = %d",
                    static_cast<long long>(sum), half);
    a.axes = axes;
    a.interleaved = interleaved != 0;
    for (int i = 0, end = 0; i < ffkv::kMaxAxes; ++i)
    {
        const int n = i < axes ? sections[i] : 0;
        if (interleaved != 0 && i > 0 && n > 0 && static_cast<int64_t>(n - 1) * axes + i >= half)
            return fail(FFKV_ERR_INVALID_ARGUMENT, "axis %d has %d interleaved pairs, more than fit head_dim / 2 = %d", i, n, half);
        end += n;
        a.section_end[i] = interleaved != 0 ? n : (i < axes ? end : half);
    }
    return FFKV_OK;
}

// Both forms of the rotation: with k_cache the append, else k_out.
int rope_axes(ffkv::RopeAxesArgs a, const int* sections, int axes, int interleaved, int block_size, float rope_theta,
              void* stream)
{
    const bool append = a.k_cache != nullptr || a.v_cache != nullptr;
    if (block_size != FFKV_BLOCK_SIZE) return fail(FFKV_ERR_UNSUPPORTED, "block_size must be 16, got %d", block_size);
    if (!is_act(a.src_dtype)) return fail(FFKV_ERR_UNSUPPORTED, "unsupported q/k/v dtype %d", a.src_dtype);
    if (append && !is_cache(a.cache_dtype)) return fail(FFKV_ERR_UNSUPPORTED, "unsupported cache dtype %d", a.cache_dtype);
    if (!head_dim_mfma(a.head_dim))
        return fail(FFKV_ERR_UNSUPPORTED, "head_dim must be 64, 128 or 256, got %d", a.head_dim);
    if (a.q == nullptr) a.num_heads = 0;
    if (a.batch < 0 || a.seq_len < 0 || a.num_heads < 0 || a.num_kv_heads <= 0 || a.max_blocks < 0 || a.num_blocks < 0)
        return fail(FFKV_ERR_INVALID_ARGUMENT, "bad size (batch %d seq_len %d heads %d kv_heads %d max_blocks %d "
                    "num_blocks %d)", a.batch, a.seq_len, a.num_heads, a.num_kv_heads, a.max_blocks, a.num_blocks);
    if (a.num_heads > 65535 || a.num_kv_heads > 65535)
        return fail(FFKV_ERR_UNSUPPORTED, "num_heads and num_kv_heads must be <= 65535");
    if (static_cast<int64_t>(a.batch) * a.seq_len > INT32_MAX / 4)
        return fail(FFKV_ERR_UNSUPPORTED, "batch * seq_len must be <= 2^29 - 1");
    if (!(rope_theta > 0.0f) || std::isinf(rope_theta))
        return fail(FFKV_ERR_INVALID_ARGUMENT, "rope_theta must be positive and finite, got %g", static_cast<double>(rope_theta));
    if (const int rc = set_sections(a, sections, axes, interleaved)) return rc;
    if (const int rc = check_stride("q_stride", a.q_stride, a.num_heads, a.head_dim, a.src_dtype)) return rc;
    if (const int rc = check_stride("q_out_stride", a.q_out_stride, a.num_heads, a.head_dim, a.src_dtype)) return rc;
    if (const int rc = check_stride("k_stride", a.k_stride, a.num_kv_heads, a.head_dim, a.src_dtype)) return rc;
    if (const int rc = check_stride(append ? "v_stride" : "k_out_stride", append ? a.v_stride : a.k_out_stride, a.num_kv_heads,
                                    a.head_dim, a.src_dtype))
        return rc;
    if (a.batch == 0 || a.seq_len == 0) return ok();
    if (!a.k || !a.positions || (a.q && !a.q_out) || (!append && !a.k_out))
        return fail(FFKV_ERR_INVALID_ARGUMENT, "null k, positions or output pointer");
    if ((a.q && a.q_out == a.q && a.q_out_stride != a.q_stride) || (!append && a.k_out == a.k && a.k_out_stride != a.k_stride))
        return fail(FFKV_ERR_INVALID_ARGUMENT, "in place needs the input's own stride");
    if (append && (!a.v || !a.k_cache || !a.v_cache || !a.block_table))
        return fail(FFKV_ERR_INVALID_ARGUMENT, "null v, cache or block_table pointer");
    if (append && quantized(a.cache_dtype) && (!a.k_scale || !a.v_scale))
        return fail(FFKV_ERR_INVALID_ARGUMENT, "quantized cache needs k_scale and v_scale");
    if (!aligned16(a.q) || !aligned16(a.q_out) || !aligned16(a.k) || !aligned16(a.k_out) || !aligned16(a.v) ||
        !aligned16(a.k_cache) || !aligned16(a.v_cache))
        return fail(FFKV_ERR_INVALID_ARGUMENT, "q, k, v, output and cache pointers must be 16-byte aligned");
    if (!aligned4(a.positions)) return fail(FFKV_ERR_INVALID_ARGUMENT, "positions must be 4-byte aligned");
    a.rate_log2 = -2.0 * std::log2(static_cast<double>(rope_theta)) / a.head_dim;
    const hipError_t e = ffkv::launch_rope_axes(a, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? ok() : hip_fail(e, "rope axes launch");
}

// Stream-ordered memory for a call without a workspace.
int take_memory(void** ws, int64_t bytes, hipStream_t s)
{
    const hipError_t e = hipMallocAsync(ws, static_cast<size_t>(bytes), s);
    return e == hipSuccess ? FFKV_OK : hip_fail(e, "workspace hipMallocAsync");
}

int lists_of(int seq_len, int query_block) { return static_cast<int>(ceil_div(seq_len, query_block)); }

// Pages of a row at most.
int most_pages(int max_blocks, int max_context_len)
{
    return static_cast<int>(ceil_div(ffkv::decode_cap_tokens(max_blocks, max_context_len), FFKV_BLOCK_SIZE));
}

constexpr double kMostBytes = 1e15;

constexpr int kMostListed = 1 << 26;  // pages of a list: their tokens count in 32 bits

// A choice's workspace: the scores, one per block of queries, KV head and page, and the queries' sums.
struct SelectLayout
{
    int64_t stride, sums, total;  // total -1: beyond all memory, or a launch's threads
};

SelectLayout select_layout(int batch, int seq_len, int num_heads, int num_kv_heads, int head_dim, int pages, int count,
                           int query_block)
{
    if (pages <= count) return SelectLayout{};  // nothing is left out
    const int        lists = lists_of(seq_len, query_block);
    ffkv::SelectArgs a{};
    a.batch = batch;
    a.seq_len = seq_len;
    a.num_kv_heads = num_kv_heads;
    a.group = num_heads / num_kv_heads;
    a.head_dim = head_dim;
    a.most_pages = pages;
    a.query_block = query_block;
    a.lists = lists;
    a.count = count;
    if (ffkv::select_in_one(a)) return SelectLayout{};
    if (ffkv::select_threads(a) > ffkv::kMostThreads) return SelectLayout{0, 0, -1};
    const double  each = 4.0 * pages + 16.0 * head_dim + 256.0;
    if (each * batch * lists * num_kv_heads > kMostBytes) return SelectLayout{0, 0, -1};
    const int64_t all = static_cast<int64_t>(batch) * lists * num_kv_heads;
    SelectLayout  l{};
    l.stride = ceil_div(pages, 4) * 4;  // whole 16-byte words
    l.sums = align256(all * l.stride * 4);
    l.total = l.sums + (ffkv::select_by_lists(seq_len, lists, num_heads / num_kv_heads) ? all * head_dim * 16 : 0);
    return l;
}

}  // namespace

extern "C" {

int ffkv_rope_axes(const void* q, int64_t q_stride, void* q_out, int64_t q_out_stride, const void* k, int64_t k_stride,
                   void* k_out, int64_t k_out_stride, int dtype, const int32_t* positions, const int* sections, int axes,
                   int interleaved, int batch, int seq_len, int num_heads, int num_kv_heads, int head_dim, float rope_theta,
                   void* stream)
{
    ffkv::RopeAxesArgs a{};
    a.q = q;
    a.k = k;
    a.q_out = q_out;
    a.k_out = k_out;
    a.positions = positions;
    a.q_stride = q_stride;
    a.k_stride = k_stride;
    a.q_out_stride = q_out_stride;
    a.k_out_stride = k_out_stride;
    a.src_dtype = dtype;
    a.cache_dtype = dtype;
    a.batch = batch;
    a.seq_len = seq_len;
    a.num_heads = num_heads;
    a.num_kv_heads = num_kv_heads;
    a.head_dim = head_dim;
    return rope_axes(a, sections, axes, interleaved, FFKV_BLOCK_SIZE, rope_theta, stream);
}

int ffkv_rope_append_axes(const void* q, int64_t q_stride, void* q_out, int64_t q_out_stride, const void* k, int64_t k_stride,
                          const void* v, int64_t v_stride, int src_dtype, void* k_cache, void* v_cache, int cache_dtype,
                          float* k_scale, float* v_scale, const int32_t* block_table, const int32_t* context_lens,
                          const int32_t* positions, const int* sections, int axes, int interleaved, int batch, int seq_len,
                          int num_heads, int num_kv_heads, int head_dim, int block_size, int max_blocks, int num_blocks,
                          float rope_theta, void* stream)
{
    if (k_cache == nullptr && v_cache == nullptr && batch > 0 && seq_len > 0)
        return fail(FFKV_ERR_INVALID_ARGUMENT, "null cache pointer");
    ffkv::RopeAxesArgs a{};
    a.q = q;
    a.k = k;
    a.v = v;
    a.q_out = q_out;
    a.k_cache = k_cache;
    a.v_cache = v_cache;
    a.k_scale = k_scale;
    a.v_scale = v_scale;
    a.block_table = block_table;
    a.context_lens = context_lens;
    a.positions = positions;
    a.q_stride = q_stride;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.q_out_stride = q_out_stride;
    a.src_dtype = src_dtype;
    a.cache_dtype = cache_dtype;
    a.batch = batch;
    a.seq_len = seq_len;
    a.num_heads = num_heads;
    a.num_kv_heads = num_kv_heads;
    a.head_dim = head_dim;
    a.max_blocks = max_blocks;
    a.num_blocks = num_blocks;
    return rope_axes(a, sections, axes, interleaved, block_size, rope_theta, stream);
}

int ffkv_key_bounds(const void* k_cache, int cache_dtype, const float* k_scale, void* bounds, const int32_t* block_table,
                    const int32_t* context_lens, int batch, int new_tokens, int num_kv_heads, int head_dim, int block_size,
                    int max_blocks, int num_blocks, void* stream)
{
    if (block_size != FFKV_BLOCK_SIZE) return fail(FFKV_ERR_UNSUPPORTED, "block_size must be 16, got %d", block_size);
    if (!is_cache(cache_dtype)) return fail(FFKV_ERR_UNSUPPORTED, "unsupported cache dtype %d", cache_dtype);
    if (!head_dim_ok(head_dim))
        return fail(FFKV_ERR_UNSUPPORTED, "head_dim must be a multiple of 8 up to 128, or 256, got %d", head_dim);
    if (batch < 0 || new_tokens < 0 || num_kv_heads <= 0 || max_blocks < 0 || num_blocks < 0)
        return fail(FFKV_ERR_INVALID_ARGUMENT, "bad size (batch %d new_tokens %d kv_heads %d max_blocks %d num_blocks %d)", batch,
                    new_tokens, num_kv_heads, max_blocks, num_blocks);
    if (batch > 65535 || num_kv_heads > 65535)
        return fail(FFKV_ERR_UNSUPPORTED, "batch and num_kv_heads must be <= 65535");
    if (batch == 0 || new_tokens == 0) return ok();
    if (!k_cache || !bounds || !block_table || !context_lens)
        return fail(FFKV_ERR_INVALID_ARGUMENT, "null cache, bounds, block_table or context_lens pointer");
    if (quantized(cache_dtype) && !k_scale) return fail(FFKV_ERR_INVALID_ARGUMENT, "quantized cache needs k_scale");
    if (!aligned16(k_cache) || !aligned16(bounds))
        return fail(FFKV_ERR_INVALID_ARGUMENT, "cache and bounds pointers must be 16-byte aligned");
    ffkv::KeyBoundsArgs a{};
    a.k_cache = k_cache;
    a.k_scale = k_scale;
    a.bounds = bounds;
    a.block_table = block_table;
    a.context_lens = context_lens;
    a.cache_dtype = cache_dtype;
    a.batch = batch;
    a.new_tokens = new_tokens;
    a.num_kv_heads = num_kv_heads;
    a.head_dim = head_dim;
    a.max_blocks = max_blocks;
    a.num_blocks = num_blocks;
    if (ffkv::key_bounds_threads(a) > ffkv::kMostThreads)
        return fail(FFKV_ERR_UNSUPPORTED, "the pages of %d new tokens are too many for one call", new_tokens);
    const hipError_t e = ffkv::launch_key_bounds(a, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? ok() : hip_fail(e, "key bounds launch");
}

size_t ffkv_select_blocks_workspace_bytes(int batch, int seq_len, int num_heads, int num_kv_heads, int head_dim, int count,
                                          int query_block, int max_blocks, int max_context_len)
{
    // sizes that ffkv_select_blocks refuses need nothing
    if (batch <= 0 || batch > 65535 || seq_len <= 0 || num_heads <= 0 || num_heads > 65535 || num_kv_heads <= 0 ||
        num_heads % num_kv_heads != 0 || !head_dim_ok(head_dim) || count <= 0 || count > kMostListed || query_block <= 0 ||
        max_blocks <= 0)
        return 0;
    const int64_t n = select_layout(batch, seq_len, num_heads, num_kv_heads, head_dim, most_pages(max_blocks, max_context_len),
                                    count, query_block).total;
    return n > 0 ? static_cast<size_t>(n) : 0;
}

int ffkv_select_blocks(const void* q, int q_dtype, const void* bounds, int bounds_dtype, const int32_t* block_table,
                       const int32_t* context_lens, int32_t* blocks, int count, int sinks, int recent, int query_block,
                       int batch, int seq_len, int num_heads, int num_kv_heads, int head_dim, int block_size, int max_blocks,
                       int num_blocks, int max_context_len, void* workspace, size_t workspace_bytes, void* stream)
{
    if (block_size != FFKV_BLOCK_SIZE) return fail(FFKV_ERR_UNSUPPORTED, "block_size must be 16, got %d", block_size);
    if (!is_act(q_dtype)) return fail(FFKV_ERR_UNSUPPORTED, "unsupported q dtype %d", q_dtype);
    if (!is_act(bounds_dtype)) return fail(FFKV_ERR_UNSUPPORTED, "unsupported bounds dtype %d", bounds_dtype);
    if (!head_dim_ok(head_dim))
        return fail(FFKV_ERR_UNSUPPORTED, "head_dim must be a multiple of 8 up to 128, or 256, got %d", head_dim);
    if (batch < 0 || seq_len < 0 || num_heads <= 0 || num_kv_heads <= 0 || max_blocks < 0 || num_blocks < 0)
        return fail(FFKV_ERR_INVALID_ARGUMENT, "bad size (batch %d seq_len %d heads %d kv_heads %d max_blocks %d "
                    "num_blocks %d)", batch, seq_len, num_heads, num_kv_heads, max_blocks, num_blocks);
    if (num_heads % num_kv_heads != 0)
        return fail(FFKV_ERR_INVALID_ARGUMENT, "num_heads %d is not a multiple of num_kv_heads %d", num_heads, num_kv_heads);
    if (batch > 65535 || num_heads > 65535) return fail(FFKV_ERR_UNSUPPORTED, "batch and num_heads must be <= 65535");
    if (query_block < 1) return fail(FFKV_ERR_INVALID_ARGUMENT, "query_block must be at least 1, got %d", query_block);
    if (num_blocks < 1 && batch > 0) return fail(FFKV_ERR_INVALID_ARGUMENT, "bounds of no page");
    if (count < 1 || sinks < 0 || recent < 0 || static_cast<int64_t>(sinks) + recent > count)
        return fail(FFKV_ERR_INVALID_ARGUMENT, "count %d must be at least 1 and hold sinks %d and recent %d", count, sinks, recent);
    if (count > kMostListed) return fail(FFKV_ERR_UNSUPPORTED, "count must be <= 2^26, got %d", count);
    if (batch == 0 || seq_len == 0) return ok();
    if (!q || !bounds || !block_table || !context_lens || !blocks)
        return fail(FFKV_ERR_INVALID_ARGUMENT, "null q, bounds, block_table, context_lens or blocks pointer");
    if (!aligned16(q) || !aligned16(bounds) || !aligned16(workspace))
        return fail(FFKV_ERR_INVALID_ARGUMENT, "q, bounds and workspace pointers must be 16-byte aligned");
    if (!aligned4(blocks)) return fail(FFKV_ERR_INVALID_ARGUMENT, "blocks must be 4-byte aligned");
    const int     lists = lists_of(seq_len, query_block);
    const int     group = num_heads / num_kv_heads;
    const int     pages = most_pages(max_blocks, max_context_len);
    const SelectLayout lay = select_layout(batch, seq_len, num_heads, num_kv_heads, head_dim, pages, count, query_block);
    const int64_t need = lay.total;
    if (static_cast<int64_t>(batch) * lists * num_kv_heads > INT32_MAX)
        return fail(FFKV_ERR_UNSUPPORTED, "batch * blocks of queries * num_kv_heads too large");
    if (static_cast<int64_t>(std::min(query_block, seq_len)) * group > INT32_MAX / 2)
        return fail(FFKV_ERR_UNSUPPORTED, "query_block * group too large");
    if (need < 0 || static_cast<int64_t>(batch) * lists * num_kv_heads * ceil_div(pages, 32) > INT32_MAX)
        return fail(FFKV_ERR_UNSUPPORTED, "the scores of %d x %d lists of %d KV heads over %d pages are too many: give "
                    "max_context_len, or fewer in a call", batch, lists, num_kv_heads, pages);
    ffkv::SelectArgs a{};
    a.q = q;
    a.bounds = bounds;
    a.block_table = block_table;
    a.context_lens = context_lens;
    a.blocks = blocks;
    a.stride = lay.stride;
    a.q_dtype = q_dtype;
    a.bounds_dtype = bounds_dtype;
    a.batch = batch;
    a.seq_len = seq_len;
    a.num_heads = num_heads;
    a.num_kv_heads = num_kv_heads;
    a.group = group;
    a.head_dim = head_dim;
    a.max_blocks = max_blocks;
    a.num_blocks = num_blocks;
    a.most_pages = pages;
    a.query_block = query_block;
    a.lists = lists;
    a.count = count;
    a.sinks = sinks;
    a.recent = recent;
    if (ffkv::select_threads(a) > ffkv::kMostThreads)
        return fail(FFKV_ERR_UNSUPPORTED, "%d x %d lists of %d KV heads are too many for one call", batch, lists, num_kv_heads);
    hipStream_t s = static_cast<hipStream_t>(stream);
    void*       ws = workspace;
    if (ws != nullptr && workspace_bytes < static_cast<size_t>(need))
        return fail(FFKV_ERR_WORKSPACE, "workspace of %zu bytes is smaller than the %lld bytes needed", workspace_bytes,
                    static_cast<long long>(need));
    if (ws == nullptr && need > 0)
    {
        bool capturing = false;
        if (const int rc = is_capturing(s, capturing)) return rc;
        if (capturing)
            return fail(FFKV_ERR_WORKSPACE, "a captured call needs a workspace, of %lld bytes", static_cast<long long>(need));
        if (const int rc = take_memory(&ws, need, s)) return rc;
    }
    a.scores = static_cast<float*>(ws);
    a.query_sums = need > 0 ? reinterpret_cast<double*>(static_cast<char*>(ws) + lay.sums) : nullptr;
    hipError_t e = ffkv::launch_select(a, s);
    if (workspace == nullptr && ws != nullptr)
    {
        const hipError_t fe = hipFreeAsync(ws, s);
        if (e == hipSuccess) e = fe;
    }
    return e == hipSuccess ? ok() : hip_fail(e, "select blocks launch");
}

size_t ffkv_paged_attention_blocks_workspace_bytes(int qo_dtype, int cache_dtype, int batch, int seq_len, int num_heads,
                                                   int num_kv_heads, int head_dim, int count, int query_block)
{
    // sizes that ffkv_paged_attention_blocks refuses need nothing
    if (!is_act(qo_dtype) || !is_cache(cache_dtype) || !head_dim_ok(head_dim) || batch <= 0 || batch > 65535 || seq_len <= 0 ||
        num_heads <= 0 || num_heads > 65535 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0 || count <= 0 ||
        count > kMostListed || query_block <= 0)
        return 0;
    ffkv::BlocksArgs a{};
    a.qo_dtype = qo_dtype;
    a.cache_dtype = cache_dtype;
    a.batch = batch;
    a.seq_len = seq_len;
    a.num_heads = num_heads;
    a.num_kv_heads = num_kv_heads;
    a.group = num_heads / num_kv_heads;
    a.head_dim = head_dim;
    a.count = count;
    a.max_blocks = INT_MAX;
    a.query_block = std::min(query_block, seq_len);  // as the call has it
    a.lists = lists_of(seq_len, a.query_block);
    if (static_cast<int64_t>(batch) * seq_len * num_heads > INT32_MAX) return 0;
    return static_cast<size_t>(ffkv::plan_blocks(a).total);
}

int ffkv_paged_attention_blocks(const void* q, void* out, int qo_dtype, const void* k_cache, const void* v_cache,
                                int cache_dtype, const float* k_scale, const float* v_scale, const int32_t* block_table,
                                const int32_t* context_lens, const int32_t* blocks, int count, int query_block, int batch,
                                int seq_len, int num_heads, int num_kv_heads, int head_dim, int block_size, int max_blocks,
                                int num_blocks, float scale, void* workspace, size_t workspace_bytes, void* stream)
{
    if (block_size != FFKV_BLOCK_SIZE) return fail(FFKV_ERR_UNSUPPORTED, "block_size must be 16, got %d", block_size);
    if (!is_act(qo_dtype)) return fail(FFKV_ERR_UNSUPPORTED, "unsupported q/out dtype %d", qo_dtype);
    if (!is_cache(cache_dtype)) return fail(FFKV_ERR_UNSUPPORTED, "unsupported cache dtype %d", cache_dtype);
    if (!head_dim_ok(head_dim))
        return fail(FFKV_ERR_UNSUPPORTED, "head_dim must be a multiple of 8 up to 128, or 256, got %d", head_dim);
    if (batch < 0 || seq_len < 0 || num_heads <= 0 || num_kv_heads <= 0 || max_blocks < 0 || num_blocks < 0)
        return fail(FFKV_ERR_INVALID_ARGUMENT, "bad size (batch %d seq_len %d heads %d kv_heads %d max_blocks %d "
                    "num_blocks %d)", batch, seq_len, num_heads, num_kv_heads, max_blocks, num_blocks);
    if (num_heads % num_kv_heads != 0)
        return fail(FFKV_ERR_INVALID_ARGUMENT, "num_heads %d is not a multiple of num_kv_heads %d", num_heads, num_kv_heads);
    if (batch > 65535 || num_heads > 65535) return fail(FFKV_ERR_UNSUPPORTED, "batch and num_heads must be <= 65535");
    if (count < 1) return fail(FFKV_ERR_INVALID_ARGUMENT, "count must be at least 1, got %d", count);
    if (count > kMostListed) return fail(FFKV_ERR_UNSUPPORTED, "count must be <= 2^26, got %d", count);
    if (query_block < 1) return fail(FFKV_ERR_INVALID_ARGUMENT, "query_block must be at least 1, got %d", query_block);
    if (batch == 0 || seq_len == 0) return ok();
    if (!q || !out || !k_cache || !v_cache || !block_table || !context_lens || !blocks)
        return fail(FFKV_ERR_INVALID_ARGUMENT, "null q, out, cache, block_table, context_lens or blocks pointer");
    if (quantized(cache_dtype) && (!k_scale || !v_scale))
        return fail(FFKV_ERR_INVALID_ARGUMENT, "quantized cache needs k_scale and v_scale");
    if (!aligned16(q) || !aligned16(out) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(workspace))
        return fail(FFKV_ERR_INVALID_ARGUMENT, "q, out, cache and workspace pointers must be 16-byte aligned");
    if (!aligned4(blocks)) return fail(FFKV_ERR_INVALID_ARGUMENT, "blocks must be 4-byte aligned");
    if (static_cast<int64_t>(batch) * seq_len * num_heads > INT32_MAX)
        return fail(FFKV_ERR_UNSUPPORTED, "batch * seq_len * num_heads too large");
    query_block = std::min(query_block, seq_len);  // (one list either way)

    ffkv::BlocksArgs a{};
    a.q = q;
    a.out = out;
    a.k_cache = k_cache;
    a.v_cache = v_cache;
    a.k_scale = k_scale;
    a.v_scale = v_scale;
    a.block_table = block_table;
    a.context_lens = context_lens;
    a.blocks = blocks;
    a.qo_dtype = qo_dtype;
    a.cache_dtype = cache_dtype;
    a.batch = batch;
    a.seq_len = seq_len;
    a.num_heads = num_heads;
    a.num_kv_heads = num_kv_heads;
    a.group = num_heads / num_kv_heads;
    a.head_dim = head_dim;
    a.max_blocks = max_blocks;
    a.num_blocks = num_blocks;
    a.query_block = query_block;
    a.lists = lists_of(seq_len, query_block);
    a.count = count;
    a.scale_log2 = (scale > 0.0f ? scale : 1.0f / sqrtf(static_cast<float>(head_dim))) * kLog2e;
    if (ffkv::blocks_threads(a) > ffkv::kMostThreads)
        return fail(FFKV_ERR_UNSUPPORTED, "%d x %d tokens of %d KV heads are too many for one call", batch, seq_len, num_kv_heads);
    const ffkv::BlocksLayout lay = ffkv::plan_blocks(a);
    hipStream_t s = static_cast<hipStream_t>(stream);
    void*       ws = workspace;
    if (ws != nullptr && workspace_bytes < static_cast<size_t>(lay.total))
        return fail(FFKV_ERR_WORKSPACE, "workspace of %zu bytes is smaller than the %lld bytes needed", workspace_bytes,
                    static_cast<long long>(lay.total));
    if (ws == nullptr && lay.total > 0)
    {
        bool capturing = false;
        if (const int rc = is_capturing(s, capturing)) return rc;
        if (capturing)  // whole lists need no workspace
        {
            a.splits = 1;
            a.pair = ffkv::blocks_pairable(a);
        }
        else if (const int rc = take_memory(&ws, lay.total, s))
            return rc;
    }
    if (a.splits > 1) ffkv::set_blocks_workspace(a, lay, ws);
    hipError_t e = ffkv::launch_blocks(a, s);
    if (workspace == nullptr && ws != nullptr)
    {
        const hipError_t fe = hipFreeAsync(ws, s);
        if (e == hipSuccess) e = fe;
    }
    return e == hipSuccess ? ok() : hip_fail(e, "blocks attention launch");
}

}  // extern "C"
