// evict.hip - eviction from the paged cache by attention weight: which tokens of a row stay, and their move.
//
// Row b holds n tokens, KV head h their weights w_0 .. w_{n-1}.  Where n > keep, the head keeps its first `sinks` and last
// `recent` tokens and, of those between, the keep - sinks - recent with the largest weights (of equal ones the earlier, NaN
// least of all), in the order of their positions; where n <= keep, all.  The kept tokens' K, V and scales go to slots 0, 1,
// .. of the row's destination pages, each head's by itself, and their weights to the front of the row of weights.
#include "mfma_common.h"

namespace ffkv
{

namespace
{

constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / 64;
constexpr int kSelPer = 32;                       // weights a thread holds: a tile is 32768 of a row's weights
constexpr int kSelTile = kSelThreads * kSelPer;
constexpr int kSelBins = 2048;                    // 11 bits of the key a pass

// Keys order as the weights do: larger is larger, -0 equals 0, NaN is 0 (below -inf).
__device__ __forceinline__ uint32_t weight_key(float w)
{
    const uint32_t u = f2u(w + 0.0f);
    return w != w ? 0u : u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}

}  // namespace

// One workgroup per (row, KV head).  The key of the last token to stay is found by three passes over the keys' bits, 11, 11
// and 10 of them, each a histogram in LDS of the keys that agree in the bits above and a search from its top; then every
// wave counts its stretches' tokens above that key and equal to it, a scan gives each its first place, and the kept
// tokens are written in order.  A row of up to 32768 tokens is read once and held in registers.
__global__ __launch_bounds__(kSelThreads) void evict_select(EvictArgs a)
{
    __shared__ int s_hist[kSelBins];
    __shared__ int s_tot[kSelWaves];
    __shared__ int s_found[2];
    __shared__ int s_cnt[kSelPer * kSelWaves];  // tokens above the key and equal to it (<< 16) per 64 of a tile
    __shared__ int s_base[2][kSelPer * kSelWaves];
    const int h = static_cast<int>(blockIdx.x);
    const int b = static_cast<int>(blockIdx.y);
    const int tid = static_cast<int>(threadIdx.x);
    const int lane = tid & 63;
    const int wave = tid >> 6;
    const int64_t bound = min(a.weight_stride, static_cast<int64_t>(a.max_blocks) * kBlockSize);
    const int     n = static_cast<int>(min(max(static_cast<int64_t>(a.context_lens[b]), int64_t{0}), bound));
    const int     count = min(n, a.keep);
    const int64_t bh = static_cast<int64_t>(b) * a.num_kv_heads + h;
    const float*  w = a.weights + bh * a.weight_stride;
    int32_t*      kept = a.kept + bh * a.keep;
    float*        out = a.weights_out != nullptr ? a.weights_out + bh * a.out_stride : nullptr;
    if (h == 0 && tid == 0) a.kept_lens[b] = count;
    if (n <= a.keep)
    {
        for (int i = tid; i < n; i += kSelThreads)
        {
            kept[i] = i;
            if (out != nullptr) out[i] = w[i];  // (in place: the same value)
        }
        return;
    }

    const int lo = a.sinks, hi = n - a.recent;  // the tokens between: more than are kept of them
    const int most = a.keep - a.sinks - a.recent;
    float     x[kSelPer];
    auto load = [&](int t0)
    {
#pragma unroll
        for (int k = 0; k < kSelPer; ++k)
        {
            const int i = t0 + k * kSelThreads + tid;
            x[k] = i < n ? w[i] : 0.0f;
        }
    };
    const bool one = n <= kSelTile;
    if (one) load(0);

    // The key of the most-th largest of the tokens between, and how many of those equal to it stay.
    uint32_t key = 0;
    int      need = most;
    if (most > 0)
    {
        for (int pass = 0; pass < 3; ++pass)
        {
            const int      shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0);
            const uint32_t bins = pass == 2 ? 1024u : 2048u;
            const uint32_t above = pass == 0 ? 0u : ~uint32_t{0} << (pass == 1 ? 21 : 10);  // bits found so far
            for (int i = tid; i < kSelBins; i += kSelThreads) s_hist[i] = 0;
            __syncthreads();
            for (int t0 = 0; t0 < n; t0 += kSelTile)
            {
                if (!one) load(t0);
#pragma unroll
                for (int k = 0; k < kSelPer; ++k)
                {
                    const int i = t0 + k * kSelThreads + tid;
                    if (i >= lo && i < hi)
                    {
                        const uint32_t u = weight_key(x[k]);
                        if ((u & above) == key) atomicAdd(&s_hist[(u >> shift) & (bins - 1)], 1);
                    }
                }
            }
            __syncthreads();
            const int top = kSelBins - 1 - 2 * tid;
            const int c0 = s_hist[top], c1 = s_hist[top - 1];
            const int incl = wave_scan(c0 + c1);
            if (lane == 63) s_tot[wave] = incl;
            __syncthreads();
            int before = incl - c0 - c1;
            for (int v = 0; v < wave; ++v) before += s_tot[v];
            if (before < need && need <= before + c0 + c1)
            {
                const bool first = need <= before + c0;
                s_found[0] = first ? top : top - 1;
                s_found[1] = need - before - (first ? 0 : c0);
            }
            __syncthreads();
            key |= static_cast<uint32_t>(s_found[0]) << shift;
            need = s_found[1];
        }
    }

    // The kept tokens in order: token i's place is the number of tokens before it that stay for sure, and of those equal to
    // the key, the first `need`.
    int base_sure = 0, base_equal = 0;
    for (int t0 = 0; t0 < n; t0 += kSelTile)
    {
        if (!one) load(t0);
        uint32_t sure = 0, equal = 0;  // bit k: of token k
#pragma unroll
        for (int k = 0; k < kSelPer; ++k)
        {
            const int      i = t0 + k * kSelThreads + tid;
            const uint32_t u = weight_key(x[k]);
            const bool     ends = i < lo || (i >= hi && i < n);
            const bool     between = i >= lo && i < hi && most > 0;
            const bool     s = ends || (between && u > key), e = between && u == key;
            sure |= static_cast<uint32_t>(s) << k;
            equal |= static_cast<uint32_t>(e) << k;
            const uint64_t bs = __ballot(s), be = __ballot(e);
            if (lane == 0) s_cnt[k * kSelWaves + wave] = __popcll(bs) | (__popcll(be) << 16);
        }
        __syncthreads();
        // exclusive sums over the 512 stretches in order, 8 per lane of the first wave
        if (wave == 0)
        {
            int cs[8], ce[8], ts = 0, te = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j)
            {
                const int v = s_cnt[8 * lane + j];
                cs[j] = ts, ce[j] = te;
                ts += v & 0xffff, te += v >> 16;
            }
            const int xs = wave_scan(ts) - ts, xe = wave_scan(te) - te;
#pragma unroll
            for (int j = 0; j < 8; ++j)
            {
                s_base[0][8 * lane + j] = xs + cs[j];
                s_base[1][8 * lane + j] = xe + ce[j];
            }
            if (lane == 63) s_found[0] = xs + ts, s_found[1] = xe + te;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kSelPer; ++k)
        {
            if (t0 + k * kSelThreads >= n) break;  // uniform
            const bool     s = sure >> k & 1, e = equal >> k & 1;
            const uint64_t bs = __ballot(s), be = __ballot(e);
            const uint64_t below = (uint64_t{1} << lane) - 1;
            const int      es = base_equal + s_base[1][k * kSelWaves + wave] + __popcll(be & below);
            if (s || (e && es < need))
            {
                const int at = base_sure + s_base[0][k * kSelWaves + wave] + __popcll(bs & below) + min(es, need);
                kept[at] = t0 + k * kSelThreads + tid;
                if (out != nullptr) out[at] = x[k];  // in place too: every token moves to its own place or before it
            }
        }
        base_sure += s_found[0];
        base_equal += s_found[1];
        __syncthreads();
    }
}

namespace
{

constexpr int kCopyThreads = 256;
constexpr int kCopyTokens = 32;  // tokens of a workgroup's share

// Slot (page * 16 + offset) of token t of a row in a pool of num_blocks pages, or -1 where it is on no page.
__device__ __forceinline__ int64_t slot_of(const int32_t* table, int max_blocks, int num_blocks, int t)
{
    if (t < 0 || (t >> 4) >= max_blocks) return -1;
    const int page = table[t >> 4];
    return page < 0 || page >= num_blocks ? -1 : static_cast<int64_t>(page) * kBlockSize + (t & 15);
}

}  // namespace

// The kept tokens' rows of one KV head to their new slots, other pages than those they come from: a workgroup takes 32
// tokens, K and V (and their scales), in pieces of U (16 or 8 bytes) of which a row has `units`.
template <typename U>
__global__ __launch_bounds__(kCopyThreads) void evict_copy(EvictArgs a, int units)
{
    __shared__ int64_t s_src[kCopyTokens], s_dst[kCopyTokens];
    const int h = static_cast<int>(blockIdx.y);
    const int b = static_cast<int>(blockIdx.z);
    const int tid = static_cast<int>(threadIdx.x);
    const int j0 = static_cast<int>(blockIdx.x) * kCopyTokens;
    const int count = min(a.kept_lens[b], a.keep);
    const int m = min(kCopyTokens, count - j0);
    if (m <= 0) return;
    if (tid < m)
    {
        const int t = a.kept[(static_cast<int64_t>(b) * a.num_kv_heads + h) * a.keep + j0 + tid];
        const int64_t src = slot_of(a.block_table + static_cast<int64_t>(b) * a.max_blocks, a.max_blocks, a.num_blocks, t);
        const int64_t dst = slot_of(a.dst_table + static_cast<int64_t>(b) * a.dst_blocks, a.dst_blocks, a.num_blocks, j0 + tid);
        s_src[tid] = dst < 0 || src < 0 ? -1 : src * a.num_kv_heads + h;
        s_dst[tid] = dst * a.num_kv_heads + h;
        if (a.cache_dtype == I8 && s_src[tid] >= 0)
        {
            a.k_scale[s_dst[tid]] = a.k_scale[s_src[tid]];
            a.v_scale[s_dst[tid]] = a.v_scale[s_src[tid]];
        }
    }
    __syncthreads();
    const U* ks = static_cast<const U*>(a.k_cache);
    const U* vs = static_cast<const U*>(a.v_cache);
    U*       kd = static_cast<U*>(a.k_cache);
    U*       vd = static_cast<U*>(a.v_cache);
    const int total = m * units;
    constexpr int UN = 4;
    for (int i0 = tid; i0 < total; i0 += kCopyThreads * UN)
    {
        U       k[UN], v[UN];
        int64_t to[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u)
        {
            const int i = i0 + u * kCopyThreads;
            to[u] = -1;
            if (i < total)
            {
                const int j = i / units, c = i - j * units;
                if (s_src[j] >= 0)
                {
                    k[u] = ks[s_src[j] * units + c];
                    v[u] = vs[s_src[j] * units + c];
                    to[u] = s_dst[j] * units + c;
                }
            }
        }
#pragma unroll
        for (int u = 0; u < UN; ++u)
            if (to[u] >= 0)
            {
                kd[to[u]] = k[u];
                vd[to[u]] = v[u];
            }
    }
}

// The same within the row's own pages: a workgroup takes all of a head's K (blockIdx.x 0) or V (1), so that what is
// read can be ordered before what is written over it.  A token moves to its own place or before it and the kept tokens
// are in order, so a stretch of them is read before it is written, and the writes reach no token of a later stretch.
template <typename U>
__global__ __launch_bounds__(1024) void evict_move(EvictArgs a, int units)
{
    constexpr int TOK = 1024;  // table lookups of a round, one a thread
    constexpr int UN = 8;
    __shared__ int64_t s_src[TOK], s_dst[TOK];
    const int h = static_cast<int>(blockIdx.y);
    const int b = static_cast<int>(blockIdx.z);
    const int tid = static_cast<int>(threadIdx.x);
    const int count = min(a.kept_lens[b], a.keep);
    U*        pool = static_cast<U*>(blockIdx.x == 0 ? a.k_cache : a.v_cache);
    float*    scale = blockIdx.x == 0 ? a.k_scale : a.v_scale;
    const int32_t* table = a.block_table + static_cast<int64_t>(b) * a.max_blocks;
    const int32_t* kept = a.kept + (static_cast<int64_t>(b) * a.num_kv_heads + h) * a.keep;
    for (int j0 = 0; j0 < count; j0 += TOK)
    {
        const int m = min(TOK, count - j0);
        float     sc = 0.0f;
        int64_t   src = -1, dst = -1;
        if (tid < m)
        {
            const int t = kept[j0 + tid];
            src = slot_of(table, a.max_blocks, a.num_blocks, t);
            dst = slot_of(table, a.max_blocks, a.num_blocks, j0 + tid);
            src = src < 0 || dst < 0 || src == dst ? -1 : src * a.num_kv_heads + h;
            dst = dst * a.num_kv_heads + h;
            if (a.cache_dtype == I8 && src >= 0) sc = scale[src];
            s_src[tid] = src;
            s_dst[tid] = dst;
        }
        const bool any = __syncthreads_or(src >= 0) != 0;
        if (!any) continue;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // every scale of the round is read
        __syncthreads();
        if (a.cache_dtype == I8 && src >= 0) scale[dst] = sc;
        const int total = m * units;
        for (int i0 = tid; i0 - tid < total; i0 += 1024 * UN)
        {
            U       x[UN];
            int64_t to[UN];
#pragma unroll
            for (int u = 0; u < UN; ++u)
            {
                const int i = i0 + u * 1024;
                to[u] = -1;
                if (i < total)
                {
                    const int j = i / units, c = i - j * units;
                    if (s_src[j] >= 0)
                    {
                        x[u] = pool[s_src[j] * units + c];
                        to[u] = s_dst[j] * units + c;
                    }
                }
            }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the stretch is read before any of it is written
            __syncthreads();
#pragma unroll
            for (int u = 0; u < UN; ++u)
                if (to[u] >= 0) pool[to[u]] = x[u];
        }
        __syncthreads();  // s_src and s_dst are read
    }
}

hipError_t launch_evict(const EvictArgs& a, hipStream_t stream)
{
    const unsigned heads = static_cast<unsigned>(a.num_kv_heads), rows = static_cast<unsigned>(a.batch);
    hipLaunchKernelGGL(evict_select, dim3(heads, rows), dim3(kSelThreads), 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int es = a.cache_dtype == F32 ? 4 : (a.cache_dtype == I8 || a.cache_dtype == FP8 ? 1 : 2);
    const int row = a.head_dim * es;  // a multiple of 8 bytes
    if (a.dst_table == nullptr)
    {
        if (row % 16 == 0)
            hipLaunchKernelGGL((evict_move<u32x4>), dim3(2, heads, rows), dim3(1024), 0, stream, a, row / 16);
        else
            hipLaunchKernelGGL((evict_move<u32x2>), dim3(2, heads, rows), dim3(1024), 0, stream, a, row / 8);
        return hipGetLastError();
    }
    const dim3 grid(static_cast<unsigned>((a.keep + kCopyTokens - 1) / kCopyTokens), heads, rows);
    if (row % 16 == 0)
        hipLaunchKernelGGL((evict_copy<u32x4>), grid, dim3(kCopyThreads), 0, stream, a, row / 16);
    else
        hipLaunchKernelGGL((evict_copy<u32x2>), grid, dim3(kCopyThreads), 0, stream, a, row / 8);
    return hipGetLastError();
}

}  // namespace ffkv
