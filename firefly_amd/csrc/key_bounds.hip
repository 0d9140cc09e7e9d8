// key_bounds.hip - the smallest and largest key of a page, per KV head and dim: what the choice of pages to attend goes by.
//
// For every page that the last new_tokens tokens of a row lie on: lo[d] = min, hi[d] = max over the page's tokens of the
// row of k[d] (code times scale on quantized caches).  NaN keys give NaN bounds.  They are kept in the cache's type, or in
// bf16 beside 8-bit caches, there rounded outward (lo down, hi up), so that they still bound every key.  A page's bounds are
// computed from the page alone, whatever they were: a step that is taken back and run again leaves no trace of the tokens
// that went.
//
// Bound by HBM: every touched page's K is read once, an eighth of it written (8 int8 prompts of 4001 tokens, 8 heads of 128, 42 MB:
// 8.5 us a call = 5.0 TB/s; a copy of 42 MB 9.9); a step, whose 64 pages are 2 MB, by its launch and the chain of length, table
// and page (3.8 us).
#include "blocks.h"
#include "ffkv_device.h"

#include <algorithm>

namespace ffkv
{

namespace
{

constexpr int kBoundsThreads = 256;

// x as the bf16 next to it toward -inf (DOWN) or +inf.
template <bool DOWN>
__device__ __forceinline__ uint32_t bf16_toward(float x)
{
    uint32_t u = f2u(x);
    if (x == x && ((u >> 31) != 0) == DOWN) u += 0xffffu;  // away from zero
    return u >> 16;
}

template <int CT, bool DOWN>
__device__ __forceinline__ void store_bound8(void* bounds, size_t at, const float* x)
{
    Raw8 r;
    if constexpr (CT == I8 || CT == FP8)
    {
#pragma unroll
        for (int i = 0; i < 4; ++i) r.w[i] = bf16_toward<DOWN>(x[2 * i]) | (bf16_toward<DOWN>(x[2 * i + 1]) << 16);
        store_raw8<BF16>(bounds, at, r);
    }
    else
    {
        pack8<CT>(x, r);
        store_raw8<CT>(bounds, at, r);
    }
}

}  // namespace

// A thread takes 8 dims of one head of one page, with the loads of its tokens in flight together; neighbouring threads take
// neighbouring chunks of the token's row of all heads.
template <int CT>
__global__ __launch_bounds__(kBoundsThreads) void key_bounds_kernel(KeyBoundsArgs a, int pages, int chunks)
{
    const int     b = static_cast<int>(blockIdx.y);
    const int64_t ctx = a.context_lens[b];
    const int64_t end = min(ctx + a.new_tokens, static_cast<int64_t>(a.max_blocks) * kBlockSize);
    const int64_t first = ctx > 0 ? ctx >> 4 : 0;
    const int64_t idx = static_cast<int64_t>(blockIdx.x) * kBoundsThreads + threadIdx.x;
    const int64_t j = idx / chunks;
    const int     c = static_cast<int>(idx - j * chunks);
    const int64_t page = first + j;
    if (j >= pages || page * kBlockSize >= end) return;
    const int phys = a.block_table[static_cast<int64_t>(b) * a.max_blocks + page];
    if (phys < 0 || phys >= a.num_blocks) return;
    const int    live = static_cast<int>(min(end - page * kBlockSize, static_cast<int64_t>(kBlockSize)));
    const int    per_head = a.head_dim / 8;
    const int    h = c / per_head;
    const int    row = a.num_kv_heads * a.head_dim;  // elements of a token
    const size_t base = static_cast<size_t>(phys) * kBlockSize * row + static_cast<size_t>(c) * 8;
    Raw8  raw[kBlockSize];
    float scale[kBlockSize];
#pragma unroll
    for (int t = 0; t < kBlockSize; ++t)
    {
        const int s = t < live ? t : 0;  // (a slot past the row's end reads the first again)
        load_raw8<CT>(a.k_cache, base + static_cast<size_t>(s) * row, raw[t]);
        if constexpr (CT == I8) scale[t] = a.k_scale[(static_cast<size_t>(phys) * kBlockSize + s) * a.num_kv_heads + h];
    }
    float lo[8], hi[8];
#pragma unroll
    for (int t = 0; t < kBlockSize; ++t)
    {
        float x[8];
        unpack8<CT>(raw[t], x);
#pragma unroll
        for (int e = 0; e < 8; ++e)
        {
            if constexpr (CT == I8) x[e] *= scale[t];
            if constexpr (CT == FP8) x[e] *= a.k_scale[h];
            lo[e] = t == 0 ? x[e] : __builtin_elementwise_minimum(lo[e], x[e]);
            hi[e] = t == 0 ? x[e] : __builtin_elementwise_maximum(hi[e], x[e]);
        }
    }
    const size_t at = (static_cast<size_t>(phys) * a.num_kv_heads + h) * 2 * a.head_dim + (c - h * per_head) * 8;
    store_bound8<CT, true>(a.bounds, at, lo);
    store_bound8<CT, false>(a.bounds, at + a.head_dim, hi);
}

namespace
{

// Pages of a row that its new tokens lie on, at most.
int64_t new_pages(const KeyBoundsArgs& a)
{
    return std::min<int64_t>((static_cast<int64_t>(a.new_tokens) + kBlockSize - 2) / kBlockSize + 1, a.max_blocks);
}

}  // namespace

// (of a row: the rows are the grid's second dimension)
int64_t key_bounds_threads(const KeyBoundsArgs& a)
{
    const int64_t chunks = static_cast<int64_t>(a.num_kv_heads) * a.head_dim / 8;
    return (new_pages(a) * chunks + kBoundsThreads - 1) / kBoundsThreads * kBoundsThreads;
}

hipError_t launch_key_bounds(const KeyBoundsArgs& a, hipStream_t stream)
{
    if (key_bounds_threads(a) > kMostThreads) return hipErrorInvalidConfiguration;
    const int     chunks = a.num_kv_heads * a.head_dim / 8;
    const int64_t pages = new_pages(a);
    const int64_t wgs = key_bounds_threads(a) / kBoundsThreads;
    if (wgs <= 0) return hipSuccess;
    const dim3 grid(static_cast<unsigned>(wgs), static_cast<unsigned>(a.batch));
    auto go = [&]<int CT>()
    {
        hipLaunchKernelGGL((key_bounds_kernel<CT>), grid, dim3(kBoundsThreads), 0, stream, a, static_cast<int>(pages), chunks);
        return hipGetLastError();
    };
    switch (a.cache_dtype)
    {
        case F32:
            return go.template operator()<F32>();
        case F16:
            return go.template operator()<F16>();
        case BF16:
            return go.template operator()<BF16>();
        case I8:
            return go.template operator()<I8>();
        default:
            return go.template operator()<FP8>();
    }
}

}  // namespace ffkv
