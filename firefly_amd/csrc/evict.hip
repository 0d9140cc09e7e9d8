// evict.hip - eviction from the paged cache by attention weight: which tokens of a row stay, and their move.
//
// Row b holds n tokens, KV head h their weights w_0 .. w_{n-1}.  Where n > keep, the head keeps its first `sinks` and last
// `recent` tokens and, of those between, the keep - sinks - recent with the largest weights (of equal ones the earlier, NaN
// least of all), in the order of their positions; where n <= keep, all.  The kept tokens' K, V and scales go to slots 0, 1,
// .. of the row's destination pages, each head's by itself, and their weights to the front of the row of weights.
//
// Bound by HBM in the copy and by latency in the choice.  Measured (8 KV heads of 128 dims): 64 int8 rows of 900 to 8000 tokens
// cut to 1000 87 us (choice 17, copy 62: 4.6 TB/s); one bf16 row of 131k cut to 16k 65 us (choice in parts 30, copy 26:
// 5.1 TB/s); 4 fp32 rows of 200 to 1000 cut to 256 12.6 us (two launches of 6).  In place 82, 207 and 14.5 us: one long row has
// two workgroups per KV head there (evict_move).
#include "mfma_common.h"

#include <algorithm>

namespace ffkv
{

namespace
{

constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / 64;
constexpr int kSelBins = 2048;                    // 11 bits of the key a pass
constexpr int kSelPartPer = 8;                    // weights a thread holds of a part of a long row
constexpr int kSelPart = kSelThreads * kSelPartPer;

// Keys order as the weights do: larger is larger, -0 equals 0, NaN is 0 (below -inf).
__device__ __forceinline__ uint32_t weight_key(float w)
{
    const uint32_t u = f2u(w + 0.0f);
    return w != w ? 0u : u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}

// Writes the kept tokens of a tile, token t0 + 1024 k + thread in x[k], in order: token i's place is the number of tokens
// before it that stay for sure (`base_sure` before the tile) and, of those between the ends that equal the key, as many as
// `need`.  s_found: the tile's two counts.
template <int PER>
__device__ __forceinline__ void write_kept(const float (&x)[PER], int t0, int n, int lo, int hi, int most, uint32_t key,
                                           int need, int base_sure, int base_equal, int32_t* kept, float* out, int* s_cnt,
                                           int (*s_base)[PER * kSelWaves], int* s_found)
{
    constexpr int kSelPer = PER;
    constexpr int kPerLane = PER * kSelWaves / 64;
    static_assert(PER * kSelWaves % 64 == 0, "a wave scans the stretches");
    const int tid = static_cast<int>(threadIdx.x);
    const int lane = tid & 63;
    const int wave = tid >> 6;
    uint32_t sure = 0, equal = 0;  // bit k: of token k
#pragma unroll
    for (int k = 0; k < kSelPer; ++k)
    {
        if (t0 + k * kSelThreads >= n)  // uniform
        {
            if (lane == 0) s_cnt[k * kSelWaves + wave] = 0;
            continue;
        }
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
    // Weights in place: every wave has its tokens' before any wave writes over them.  (A barrier waits for LDS alone, and the
    // weights of a wave at the row's ends, which no comparison has needed, may still be on their way.)
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    // exclusive sums over the stretches in order, kPerLane per lane of the first wave
    if (wave == 0)
    {
        int cs[kPerLane], ce[kPerLane], ts = 0, te = 0;
#pragma unroll
        for (int j = 0; j < kPerLane; ++j)
        {
            const int v = s_cnt[kPerLane * lane + j];
            cs[j] = ts, ce[j] = te;
            ts += v & 0xffff, te += v >> 16;
        }
        const int xs = wave_scan(ts) - ts, xe = wave_scan(te) - te;
#pragma unroll
        for (int j = 0; j < kPerLane; ++j)
        {
            s_base[0][kPerLane * lane + j] = xs + cs[j];
            s_base[1][kPerLane * lane + j] = xe + ce[j];
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
}

}  // namespace

// One workgroup per (row, KV head).  The key of the last token to stay is found by three passes over the keys' bits, 11, 11
// and 10 of them, each a histogram in LDS of the keys that agree in the bits above and a search from its top; then every
// wave counts its stretches' tokens above that key and equal to it, a scan gives each its first place, and the kept
// tokens are written in order.  A row of up to 1024 * PER tokens is read once and held in registers.
template <int PER>
__global__ __launch_bounds__(kSelThreads) void evict_select(EvictArgs a)
{
    constexpr int kSelPer = PER;
    constexpr int kSelTile = kSelThreads * PER;
    constexpr int kStretches = PER * kSelWaves;  // of 64 tokens, in a tile
    __shared__ int s_hist[kSelBins];
    __shared__ int s_tot[kSelWaves];
    __shared__ int s_found[2];
    __shared__ int s_cnt[kStretches];  // tokens above the key and equal to it (<< 16) per 64 of a tile
    __shared__ int s_base[2][kStretches];
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
            x[k] = 0.0f;
            if (t0 + k * kSelThreads < n) x[k] = i < n ? w[i] : 0.0f;  // (the outer test is uniform)
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
                    if (t0 + k * kSelThreads >= n) break;  // uniform
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
            const int tot = lane < kSelWaves ? s_tot[lane] : 0;
            const int before = incl - c0 - c1 + __shfl(wave_scan(tot) - tot, wave, 64);
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
        write_kept<PER>(x, t0, n, lo, hi, most, key, need, base_sure, base_equal, kept, out, s_cnt, s_base, s_found);
        base_sure += s_found[0];
        base_equal += s_found[1];
        __syncthreads();
    }
}

// The same for few long rows, which one workgroup each would hold up (a CU reads about 50 GB/s): a row's weights in parts of
// 8192, a workgroup per part, and a launch per pass.  Level 0 to 2 are the histograms of the parts, each of which first finds
// the key's bits of the level before from all parts' histograms; level 3 writes the kept tokens.  Every workgroup of a row
// does the searches for itself, so nothing waits but for the launch before, and no order of atomics is seen in the results.
// hist0 and hist1 [batch * heads, parts, 2048] take the levels in turn, state [batch * heads, 2] the key and how many equal
// to it stay, above [2, batch * heads, parts] the parts' tokens above the bits found at levels 1 and 2.
// One row of 131k tokens at 8 KV heads: 128 us in one workgroup per head, 30 us so.
namespace
{

// Sum of x over the workgroup's threads, in every thread.
__device__ __forceinline__ int block_sum(int x, int* s_tmp)
{
    const int wave = static_cast<int>(threadIdx.x) >> 6, lane = static_cast<int>(threadIdx.x) & 63;
    x = __builtin_amdgcn_readlane(wave_scan(x), 63);
    __syncthreads();
    if (lane == 0) s_tmp[wave] = x;
    __syncthreads();
    return __builtin_amdgcn_readlane(wave_scan(lane < kSelWaves ? s_tmp[lane] : 0), 63);
}

}  // namespace

template <int LEVEL>
__global__ __launch_bounds__(kSelThreads) void evict_select_part(EvictArgs a)
{
    constexpr int PER = kSelPartPer;
    constexpr int kStretches = PER * kSelWaves;
    __shared__ int s_hist[LEVEL < 3 ? kSelBins : 1];
    __shared__ int s_tot[kSelWaves];
    __shared__ int s_found[2];
    __shared__ int s_cnt[kStretches], s_base[2][kStretches];
    const int part = static_cast<int>(blockIdx.x);
    const int h = static_cast<int>(blockIdx.y);
    const int b = static_cast<int>(blockIdx.z);
    const int tid = static_cast<int>(threadIdx.x);
    const int lane = tid & 63;
    const int wave = tid >> 6;
    const int64_t bound = min(a.weight_stride, static_cast<int64_t>(a.max_blocks) * kBlockSize);
    const int     n = static_cast<int>(min(max(static_cast<int64_t>(a.context_lens[b]), int64_t{0}), bound));
    const int     t0 = part * kSelPart;
    const int64_t bh = static_cast<int64_t>(b) * a.num_kv_heads + h;
    const int64_t all = static_cast<int64_t>(a.batch) * a.num_kv_heads;
    const float*  w = a.weights + bh * a.weight_stride;
    if (LEVEL == 3 && part == 0 && h == 0 && tid == 0) a.kept_lens[b] = min(n, a.keep);
    if (t0 >= n) return;
    int32_t* kept = a.kept + bh * a.keep;
    // (weights in place go through a copy: another part may not have read its own yet)
    float* out = a.weights_out != nullptr ? a.weights_out + bh * a.out_stride : nullptr;
    if (a.scratch != nullptr) out = a.scratch + bh * min(bound, static_cast<int64_t>(a.keep));
    if (n <= a.keep)
    {
        if (LEVEL == 3)
            for (int i = t0 + tid; i < min(n, t0 + kSelPart); i += kSelThreads)
            {
                kept[i] = i;
                if (out != nullptr) out[i] = w[i];
            }
        return;
    }
    const int parts = (n + kSelPart - 1) / kSelPart;  // of this row
    const int lo = a.sinks, hi = n - a.recent;
    const int most = a.keep - a.sinks - a.recent;
    if (LEVEL < 3 && most == 0) return;

    float x[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k)
    {
        const int i = t0 + k * kSelThreads + tid;
        x[k] = 0.0f;
        if (t0 + k * kSelThreads < n) x[k] = i < n ? w[i] : 0.0f;
    }

    uint32_t key = 0;
    int      need = most, base_sure = 0, base_equal = 0;
    if (LEVEL > 0 && most > 0)
    {
        // the bin of the level before that holds the need-th largest of the row, from its parts' histograms
        if (LEVEL > 1)
        {
            key = a.state[2 * (bh + (LEVEL - 2) * all)];
            need = static_cast<int>(a.state[2 * (bh + (LEVEL - 2) * all) + 1]);
        }
        const int* hist = (LEVEL == 2 ? a.hist1 : a.hist0) + bh * a.parts * kSelBins;
        const int  top = kSelBins - 1 - 2 * tid;  // this thread's bins: top and top - 1
        int        c0 = 0, c1 = 0, p0 = 0, p1 = 0, mine0 = 0, mine1 = 0;  // all parts', those before this one's, this one's
        constexpr int MF = 8;  // parts whose loads go out together
        for (int q0 = 0; q0 < parts; q0 += MF)
        {
            int2 v[MF];
#pragma unroll
            for (int f = 0; f < MF; ++f)
                v[f] = q0 + f < parts ? *reinterpret_cast<const int2*>(hist + static_cast<int64_t>(q0 + f) * kSelBins + top - 1)
                                      : make_int2(0, 0);
#pragma unroll
            for (int f = 0; f < MF; ++f)
            {
                c0 += v[f].y, c1 += v[f].x;
                if (q0 + f < part) p0 += v[f].y, p1 += v[f].x;
                if (q0 + f == part) mine0 = v[f].y, mine1 = v[f].x;
            }
        }
        const int incl = wave_scan(c0 + c1);
        if (lane == 63) s_tot[wave] = incl;
        __syncthreads();
        const int tot = lane < kSelWaves ? s_tot[lane] : 0;
        const int before = incl - c0 - c1 + __shfl(wave_scan(tot) - tot, wave, 64);
        if (before < need && need <= before + c0 + c1)
        {
            const bool first = need <= before + c0;
            s_found[0] = first ? top : top - 1;
            s_found[1] = need - before - (first ? 0 : c0);
        }
        __syncthreads();
        const int bin = s_found[0];
        need = s_found[1];
        key |= static_cast<uint32_t>(bin) << (LEVEL == 1 ? 21 : (LEVEL == 2 ? 10 : 0));
        if (LEVEL < 3)
        {
            const int sure = block_sum((top > bin ? mine0 : 0) + (top - 1 > bin ? mine1 : 0), s_tot);
            if (tid == 0)
            {
                a.above[((LEVEL - 1) * all + bh) * a.parts + part] = sure;
                if (part == 0)
                {
                    a.state[2 * (bh + (LEVEL - 1) * all)] = key;
                    a.state[2 * (bh + (LEVEL - 1) * all) + 1] = static_cast<uint32_t>(need);
                }
            }
        }
        else
        {
            // tokens of the parts before this one: above the key (levels 1 to 3) and equal to it
            int sure = (top > bin ? p0 : 0) + (top - 1 > bin ? p1 : 0);
            for (int q = tid; q < part; q += kSelThreads) sure += a.above[bh * a.parts + q] + a.above[(all + bh) * a.parts + q];
            base_sure = block_sum(sure, s_tot);
            base_equal = block_sum((top == bin ? p0 : 0) + (top - 1 == bin ? p1 : 0), s_tot);
        }
    }
    if constexpr (LEVEL < 3)
    {
        constexpr int      shift = LEVEL == 0 ? 21 : (LEVEL == 1 ? 10 : 0);
        constexpr uint32_t bins = LEVEL == 2 ? 1024u : 2048u;
        constexpr uint32_t above = LEVEL == 0 ? 0u : ~uint32_t{0} << (LEVEL == 1 ? 21 : 10);
        for (int i = tid; i < kSelBins; i += kSelThreads) s_hist[i] = 0;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < PER; ++k)
        {
            const int i = t0 + k * kSelThreads + tid;
            if (i >= lo && i < hi)
            {
                const uint32_t u = weight_key(x[k]);
                if ((u & above) == key) atomicAdd(&s_hist[(u >> shift) & (bins - 1)], 1);
            }
        }
        __syncthreads();
        int* dst = (LEVEL == 1 ? a.hist1 : a.hist0) + (bh * a.parts + part) * kSelBins;
        for (int i = tid; i < kSelBins; i += kSelThreads) dst[i] = s_hist[i];
    }
    else
    {
        base_sure += min(t0, lo) + max(0, t0 - hi);  // of the row's ends
        write_kept<PER>(x, t0, n, lo, hi, most, key, need, base_sure, base_equal, kept, out, s_cnt, s_base, s_found);
    }
}

// In place: the kept weights from the copy to the front of their row.
__global__ __launch_bounds__(256) void evict_weights_back(EvictArgs a)
{
    const int64_t bh = static_cast<int64_t>(blockIdx.z) * a.num_kv_heads + blockIdx.y;
    const int     i = static_cast<int>(blockIdx.x * 256 + threadIdx.x);
    const int64_t stride = min(min(a.weight_stride, static_cast<int64_t>(a.max_blocks) * kBlockSize), static_cast<int64_t>(a.keep));
    if (i < a.kept_lens[blockIdx.z]) a.weights_out[bh * a.out_stride + i] = a.scratch[bh * stride + i];
}

namespace
{

constexpr int kCopyThreads = 256;
constexpr int kCopyRows = 128;  // (token, KV head) rows of a workgroup, at most
constexpr int kCopyUnits = 4;   // pieces of K, and of V, that a thread has in flight

// Slot (page * 16 + offset) of token t of a row in a pool of num_blocks pages, or -1 where it is on no page.
__device__ __forceinline__ int64_t slot_of(const int32_t* table, int max_blocks, int num_blocks, int t)
{
    if (t < 0 || (t >> 4) >= max_blocks) return -1;
    const int page = table[t >> 4];
    return page < 0 || page >= num_blocks ? -1 : static_cast<int64_t>(page) * kBlockSize + (t & 15);
}

}  // namespace

// The kept tokens' rows to their new slots, other pages than those they come from.  A workgroup takes wg_rows (token,
// KV head) rows (as many as give each of its threads four pieces, at most kCopyRows) in the order of their destinations, heads
// fastest, so that what it writes is a contiguous stretch of whole lines, scales included; K and V go in pieces of U (16 or
// 8 bytes) of which a row has `units`.
template <typename U>
__global__ __launch_bounds__(kCopyThreads) void evict_copy(EvictArgs a, int units, int wg_rows)
{
    __shared__ int64_t s_src[kCopyRows], s_dst[kCopyRows];
    const int b = static_cast<int>(blockIdx.y);
    const int tid = static_cast<int>(threadIdx.x);
    const int H = a.num_kv_heads;
    const int count = min(a.kept_lens[b], a.keep);
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * wg_rows;
    const int m = static_cast<int>(min(static_cast<int64_t>(count) * H - row0, static_cast<int64_t>(wg_rows)));
    if (m <= 0) return;
    if (tid < m)
    {
        const int j = static_cast<int>((row0 + tid) / H);
        const int h = static_cast<int>(row0 + tid - static_cast<int64_t>(j) * H);
        const int t = a.kept[(static_cast<int64_t>(b) * H + h) * a.keep + j];
        const int64_t src = slot_of(a.block_table + static_cast<int64_t>(b) * a.max_blocks, a.max_blocks, a.num_blocks, t);
        const int64_t dst = slot_of(a.dst_table + static_cast<int64_t>(b) * a.dst_blocks, a.dst_blocks, a.num_blocks, j);
        const bool    go = src >= 0 && dst >= 0;
        s_src[tid] = go ? src * H + h : -1;
        s_dst[tid] = dst * H + h;
        if (a.cache_dtype == I8 && go)
        {
            a.k_scale[dst * H + h] = a.k_scale[src * H + h];
            a.v_scale[dst * H + h] = a.v_scale[src * H + h];
        }
    }
    __syncthreads();
    const U* ks = static_cast<const U*>(a.k_cache);
    const U* vs = static_cast<const U*>(a.v_cache);
    U*       kd = static_cast<U*>(a.k_cache);
    U*       vd = static_cast<U*>(a.v_cache);
    const int total = m * units;
    constexpr int UN = kCopyUnits;
#pragma unroll 1
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
                const int r = i / units, c = i - r * units;
                if (s_src[r] >= 0)
                {
                    k[u] = ks[s_src[r] * units + c];
                    v[u] = vs[s_src[r] * units + c];
                    to[u] = s_dst[r] * units + c;
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

int evict_parts(int batch, int num_kv_heads, int64_t bound)
{
    // One workgroup per row and head is enough while its weights fit its registers at 8 a thread, or the rows and heads
    // give every CU one; the four launches of the other form take about 25 us whatever the row.
    if (bound <= kSelPart || static_cast<int64_t>(batch) * num_kv_heads >= 256) return 0;
    return static_cast<int>((bound + kSelPart - 1) / kSelPart);
}

hipError_t launch_evict(const EvictArgs& a, hipStream_t stream)
{
    const unsigned heads = static_cast<unsigned>(a.num_kv_heads), rows = static_cast<unsigned>(a.batch);
    const int64_t bound = std::min<int64_t>(a.weight_stride, static_cast<int64_t>(a.max_blocks) * kBlockSize);
    if (a.parts > 0)
    {
        const dim3 grid(static_cast<unsigned>(a.parts), heads, rows);
        hipLaunchKernelGGL((evict_select_part<0>), grid, dim3(kSelThreads), 0, stream, a);
        hipLaunchKernelGGL((evict_select_part<1>), grid, dim3(kSelThreads), 0, stream, a);
        hipLaunchKernelGGL((evict_select_part<2>), grid, dim3(kSelThreads), 0, stream, a);
        hipLaunchKernelGGL((evict_select_part<3>), grid, dim3(kSelThreads), 0, stream, a);
        if (a.scratch != nullptr)
            hipLaunchKernelGGL(evict_weights_back, dim3(static_cast<unsigned>((std::min<int64_t>(a.keep, bound) + 255) / 256), heads, rows),
                               dim3(256), 0, stream, a);
    }
    // weights a thread holds: as few as the rows' bound allows (fewer registers, more workgroups per CU), at most 32
    else if (bound <= 4 * kSelThreads)
        hipLaunchKernelGGL((evict_select<4>), dim3(heads, rows), dim3(kSelThreads), 0, stream, a);
    else if (bound <= 8 * kSelThreads)
        hipLaunchKernelGGL((evict_select<8>), dim3(heads, rows), dim3(kSelThreads), 0, stream, a);
    else
        hipLaunchKernelGGL((evict_select<32>), dim3(heads, rows), dim3(kSelThreads), 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || bound <= 0) return e;
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
    const int     units = row % 16 == 0 ? row / 16 : row / 8;
    const int     wg_rows = std::max(8, std::min(kCopyRows, kCopyThreads * kCopyUnits / units));
    const int64_t wgs = (static_cast<int64_t>(std::min<int64_t>(a.keep, bound)) * heads + wg_rows - 1) / wg_rows;
    if (wgs > INT32_MAX) return hipErrorInvalidConfiguration;
    const dim3 grid(static_cast<unsigned>(wgs), rows);
    if (row % 16 == 0)
        hipLaunchKernelGGL((evict_copy<u32x4>), grid, dim3(kCopyThreads), 0, stream, a, units, wg_rows);
    else
        hipLaunchKernelGGL((evict_copy<u32x2>), grid, dim3(kCopyThreads), 0, stream, a, units, wg_rows);
    return hipGetLastError();
}

}  // namespace ffkv
