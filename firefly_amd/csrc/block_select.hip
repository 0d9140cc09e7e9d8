// block_select.hip - which pages of its row a block of queries attends, per KV head: a score per page from the page's key
// bounds, and the pages with the largest.
//
//   score(page) = sum over the block's queries and the KV head's query heads of sum_d max(q_d lo_d, q_d hi_d)
//               = sum_d Q+_d hi_d + Q-_d lo_d,   Q+ = sum of max(q, 0), Q- = sum of min(q, 0)
// No query's score with any of the page's keys exceeds its share of that.  The sums over queries and heads go first, so a
// block of any size costs two dot products of head_dim per page.
//
// Scores are fp64 sums rounded once to fp32: they decide between pages, and the choice must not depend on how a row is
// split, on the batch or on the form that was launched (products of 16-bit values are exact in fp64, and the sums' errors of
// 2^-50 are far below the rounding's step).
//
// Of a block's pages - those up to its last query's - the first `sinks` and the last `recent` are taken, and of the rest
// those with the largest scores, of equal ones the lower; NaN (a NaN or infinite key) counts as the largest.  The list is in
// ascending order, -1 behind.
#include "blocks.h"
#include "mfma_common.h"

#include <algorithm>

namespace ffkv
{

namespace
{

constexpr int kScoreThreads = 256;
constexpr int kScoreWaves = kScoreThreads / 64;
constexpr int kScoreUnroll = 4;  // pages a group of lanes has in flight

// v of lane ^ MASK within groups of N lanes summed up, in every lane of the group: fp64 in two 32-bit halves.
template <int N>
__device__ __forceinline__ double group_sum64(double v)
{
    auto step = [&](auto ctrl)
    {
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(u), decltype(ctrl)::value, 0xf, 0xf, false);
        const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(u >> 32), decltype(ctrl)::value, 0xf, 0xf, false);
        v += __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
    };
    step(std::integral_constant<int, 0xb1>{});                            // quad lanes 1, 0, 3, 2
    step(std::integral_constant<int, 0x4e>{});                            // quad lanes 2, 3, 0, 1
    if constexpr (N >= 8) step(std::integral_constant<int, 0x141>{});     // lane 7 - i of its 8
    if constexpr (N >= 16) step(std::integral_constant<int, 0x140>{});    // lane 15 - i of its 16
    if constexpr (N >= 32) v += __shfl_xor(v, 16, 64);
    return v;
}

// Visible pages of the block of queries `list` of row b.
__device__ __forceinline__ int visible_pages(const SelectArgs& a, int b, int list)
{
    const int64_t last = static_cast<int64_t>(a.context_lens[b]) +
                         min((static_cast<int64_t>(list) + 1) * a.query_block, static_cast<int64_t>(a.seq_len)) - 1;
    const int64_t n = last < 0 ? 0 : (last >> 4) + 1;
    return static_cast<int>(min(n, static_cast<int64_t>(a.most_pages)));
}

// Keys order as the scores do: larger is larger, -0 equals 0, NaN is the largest.
__device__ __forceinline__ uint32_t score_key(float w)
{
    const uint32_t u = f2u(w + 0.0f);
    return w != w ? 0xffffffffu : u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}

// Q- and Q+ of a block of queries into LDS, [2][D], by all threads of the workgroup; s_part: [kScoreWaves][2][D].
template <int LPP>
__device__ __forceinline__ void sum_queries(const SelectArgs& a, int b, int list, int kvh, double* s_q, double* s_part)
{
    const int  D = a.head_dim;
    const int  tid = static_cast<int>(threadIdx.x);
    const int  lane = tid & 63, wave = tid >> 6;
    const int  c = lane % LPP;
    const bool in = 8 * c < D;
    const int  t0 = list * a.query_block;
    const int  rows = min(a.query_block, a.seq_len - t0) * a.group;
    double     down[8], up[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) down[e] = up[e] = 0.0;
    for (int r = tid / LPP; r < rows; r += kScoreThreads / LPP)
    {
        if (!in) continue;
        const int    t = r / a.group;
        const size_t at = ((static_cast<size_t>(b) * a.seq_len + t0 + t) * a.num_heads + kvh * a.group + r - t * a.group) * D + 8 * c;
        float        x[8];
        load_act8(a.q, a.q_dtype, at, x);
#pragma unroll
        for (int e = 0; e < 8; ++e)
        {
            // (a NaN goes to both)
            down[e] += x[e] > 0.0f ? 0.0 : static_cast<double>(x[e]);
            up[e] += x[e] < 0.0f ? 0.0 : static_cast<double>(x[e]);
        }
    }
#pragma unroll
    for (int off = LPP; off < 64; off <<= 1)
#pragma unroll
        for (int e = 0; e < 8; ++e)
        {
            down[e] += __shfl_xor(down[e], off, 64);
            up[e] += __shfl_xor(up[e], off, 64);
        }
    if (lane < LPP && in)
#pragma unroll
        for (int e = 0; e < 8; ++e)
        {
            s_part[(wave * 2) * D + 8 * c + e] = down[e];
            s_part[(wave * 2 + 1) * D + 8 * c + e] = up[e];
        }
    __syncthreads();
    for (int i = tid; i < 2 * D; i += kScoreThreads)
    {
        double s = 0.0;
#pragma unroll
        for (int w = 0; w < kScoreWaves; ++w) s += s_part[w * 2 * D + i];
        s_q[i] = s;
    }
    __syncthreads();
}

}  // namespace

// A workgroup scores `tile` pages of a block of queries and KV head: LPP lanes take a page's bounds, 8 dims each, and
// kScoreUnroll pages in flight.  Grid: (tile, KV head, block of queries of a row).
template <int BT, int LPP>
__global__ __launch_bounds__(kScoreThreads) void block_scores(SelectArgs a, int tile, int tiles)
{
    constexpr int GROUPS = kScoreThreads / LPP;  // pages of a round
    __shared__ double s_q[2 * LPP * 8];
    __shared__ double s_part[kScoreWaves * 2 * LPP * 8];
    const int64_t wg = blockIdx.x;
    const int     kvh = static_cast<int>(wg / tiles % a.num_kv_heads);
    const int     row = static_cast<int>(wg / tiles / a.num_kv_heads);
    const int     b = row / a.lists, list = row - b * a.lists;
    const int     n = visible_pages(a, b, list);
    const int     p0 = static_cast<int>(wg % tiles) * tile;
    if (p0 >= n) return;
    const int  p1 = min(n, p0 + tile);
    const int  D = a.head_dim;
    const int  tid = static_cast<int>(threadIdx.x);
    const int  c = tid % LPP, grp = tid / LPP;
    const bool in = 8 * c < D;
    sum_queries<LPP>(a, b, list, kvh, s_q, s_part);
    double down[8], up[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
    {
        down[e] = in ? s_q[8 * c + e] : 0.0;
        up[e] = in ? s_q[D + 8 * c + e] : 0.0;
    }
    const int32_t* table = a.block_table + static_cast<int64_t>(b) * a.max_blocks;
    float* out = a.scores + (static_cast<int64_t>(row) * a.num_kv_heads + kvh) * a.stride;
    for (int q0 = p0; q0 < p1; q0 += GROUPS * kScoreUnroll)
    {
        Raw8 lo[kScoreUnroll], hi[kScoreUnroll];
        bool ok[kScoreUnroll];
#pragma unroll
        for (int k = 0; k < kScoreUnroll; ++k)
        {
            const int p = q0 + k * GROUPS + grp;
            const int phys = p < p1 ? table[p] : -1;
            ok[k] = phys >= 0 && phys < a.num_blocks;
            if (ok[k] && in)
            {
                const size_t at = (static_cast<size_t>(phys) * a.num_kv_heads + kvh) * 2 * D + 8 * c;
                load_raw8<BT>(a.bounds, at, lo[k]);
                load_raw8<BT>(a.bounds, at + D, hi[k]);
            }
        }
#pragma unroll
        for (int k = 0; k < kScoreUnroll; ++k)
        {
            double s = 0.0;
            if (ok[k] && in)
            {
                float x[8], y[8];
                unpack8<BT>(lo[k], x);
                unpack8<BT>(hi[k], y);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                {
                    s = __builtin_fma(down[e], static_cast<double>(x[e]), s);
                    s = __builtin_fma(up[e], static_cast<double>(y[e]), s);
                }
            }
            s = group_sum64<LPP>(s);
            const int p = q0 + k * GROUPS + grp;
            if (c == 0 && p < p1) out[p] = ok[k] ? static_cast<float>(s) : kNegInf;  // on no page: last
        }
    }
}

// One workgroup per list.  The score of the last page to stay is found by three passes over the keys' bits, 11, 11 and 10 of
// them, each a histogram in LDS of the keys that agree in the bits above and a search from its top; then the pages above it
// and the first of those equal to it are written in order.  A list of up to THREADS * PER pages is read once.
template <int THREADS, int PER>
__global__ __launch_bounds__(THREADS) void block_choose(SelectArgs a)
{
    constexpr int WAVES = THREADS / 64;
    constexpr int TILE = THREADS * PER;
    constexpr int BINS = 2048;
    constexpr int BPT = BINS / THREADS;  // bins a thread sums up
    __shared__ int s_hist[BINS];
    __shared__ int s_tot[WAVES];
    __shared__ int s_found[2];
    __shared__ int s_cnt[2][PER * WAVES];
    const int64_t wg = blockIdx.x;
    const int     row = static_cast<int>(wg / a.num_kv_heads);
    const int     b = row / a.lists, list = row - b * a.lists;
    const int     n = visible_pages(a, b, list);
    const int     tid = static_cast<int>(threadIdx.x);
    const int     lane = tid & 63, wave = tid >> 6;
    const float*  w = a.scores + wg * a.stride;
    int32_t*      out = a.blocks + wg * a.count;
    if (n <= a.count)
    {
        for (int i = tid; i < a.count; i += THREADS) out[i] = i < n ? i : -1;
        return;
    }
    const int lo = a.sinks, hi = n - a.recent;  // the pages between: more than are taken of them
    const int most = a.count - a.sinks - a.recent;
    uint32_t  x[PER];
    auto load = [&](int t0)
    {
#pragma unroll
        for (int k = 0; k < PER; ++k)
        {
            const int i = t0 + k * THREADS + tid;
            x[k] = i < n ? score_key(w[i]) : 0u;
        }
    };
    const bool one = n <= TILE;
    if (one) load(0);
    uint32_t key = 0;
    int      need = most;
    if (most > 0)
        for (int pass = 0; pass < 3; ++pass)
        {
            const int      shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0);
            const uint32_t bins = pass == 2 ? 1024u : 2048u;
            const uint32_t above = pass == 0 ? 0u : ~uint32_t{0} << (pass == 1 ? 21 : 10);  // bits found so far
            for (int i = tid; i < BINS; i += THREADS) s_hist[i] = 0;
            __syncthreads();
            for (int t0 = 0; t0 < n; t0 += TILE)
            {
                if (!one) load(t0);
#pragma unroll
                for (int k = 0; k < PER; ++k)
                {
                    const int i = t0 + k * THREADS + tid;
                    if (i >= lo && i < hi && (x[k] & above) == key) atomicAdd(&s_hist[(x[k] >> shift) & (bins - 1)], 1);
                }
            }
            __syncthreads();
            const int top = BINS - 1 - BPT * tid;  // this thread's bins: top, top - 1, ..
            int       c[BPT], sum = 0;
#pragma unroll
            for (int j = 0; j < BPT; ++j) sum += c[j] = s_hist[top - j];
            const int incl = wave_scan(sum);
            if (lane == 63) s_tot[wave] = incl;
            __syncthreads();
            const int tot = lane < WAVES ? s_tot[lane] : 0;
            int       before = incl - sum + __shfl(wave_scan(tot) - tot, wave, 64);
#pragma unroll
            for (int j = 0; j < BPT; ++j)
            {
                if (before < need && need <= before + c[j])
                {
                    s_found[0] = top - j;
                    s_found[1] = need - before;
                }
                before += c[j];
            }
            __syncthreads();
            key |= static_cast<uint32_t>(s_found[0]) << shift;
            need = s_found[1];
            __syncthreads();
        }

    int base_sure = 0, base_equal = 0;
    for (int t0 = 0; t0 < n; t0 += TILE)
    {
        if (!one) load(t0);
        uint32_t sure = 0, equal = 0;  // bit k: of page k
#pragma unroll
        for (int k = 0; k < PER; ++k)
        {
            const int  i = t0 + k * THREADS + tid;
            const bool ends = i < lo || (i >= hi && i < n);
            const bool between = i >= lo && i < hi && most > 0;
            const bool s = ends || (between && x[k] > key), e = between && x[k] == key;
            sure |= static_cast<uint32_t>(s) << k;
            equal |= static_cast<uint32_t>(e) << k;
            const uint64_t bs = __ballot(s), be = __ballot(e);
            if (lane == 0) s_cnt[0][k * WAVES + wave] = __popcll(bs), s_cnt[1][k * WAVES + wave] = __popcll(be);
        }
        __syncthreads();
        int cs = base_sure, ce = base_equal;
#pragma unroll
        for (int k = 0; k < PER; ++k)
        {
            // counts of the stretches of 64 pages before this one, of this k and the k before
            int ps = cs, pe = ce;
            for (int v = 0; v < WAVES; ++v)
            {
                const int ns = s_cnt[0][k * WAVES + v], ne = s_cnt[1][k * WAVES + v];
                if (v < wave) ps += ns, pe += ne;
                cs += ns, ce += ne;
            }
            const bool     s = sure >> k & 1, e = equal >> k & 1;
            const uint64_t bs = __ballot(s), be = __ballot(e);
            const uint64_t below = (uint64_t{1} << lane) - 1;
            const int      es = pe + __popcll(be & below);
            if (s || (e && es < need)) out[ps + __popcll(bs & below) + min(es, need)] = t0 + k * THREADS + tid;
        }
        base_sure = cs, base_equal = ce;
        __syncthreads();
    }
}

namespace
{

template <int BT>
hipError_t launch_scores(const SelectArgs& a, hipStream_t stream)
{
    const int64_t lists = static_cast<int64_t>(a.batch) * a.lists * a.num_kv_heads;
    auto go = [&]<int LPP>()
    {
        constexpr int ROUND = kScoreThreads / LPP * kScoreUnroll;
        // a workgroup's tile: as many rounds as leave 2048 workgroups
        int64_t rounds = (a.most_pages + ROUND - 1) / ROUND;
        const int64_t per = std::max<int64_t>(1, std::min<int64_t>(rounds, lists * rounds / 2048));
        const int64_t tiles = (rounds + per - 1) / per;
        if (lists * tiles > INT32_MAX) return hipErrorInvalidConfiguration;
        hipLaunchKernelGGL((block_scores<BT, LPP>), dim3(static_cast<unsigned>(lists * tiles)), dim3(kScoreThreads), 0, stream, a,
                           static_cast<int>(per * ROUND), static_cast<int>(tiles));
        return hipGetLastError();
    };
    if (a.head_dim <= 64) return go.template operator()<8>();
    if (a.head_dim <= 128) return go.template operator()<16>();
    return go.template operator()<32>();
}

}  // namespace

hipError_t launch_select(const SelectArgs& a, hipStream_t stream)
{
    const int64_t lists = static_cast<int64_t>(a.batch) * a.lists * a.num_kv_heads;
    if (lists > INT32_MAX) return hipErrorInvalidConfiguration;
    hipError_t e = hipSuccess;
    // (rows that cannot have more pages than are taken need no scores)
    if (a.most_pages > a.count)
        e = a.bounds_dtype == F32 ? launch_scores<F32>(a, stream)
            : a.bounds_dtype == F16 ? launch_scores<F16>(a, stream)
                                    : launch_scores<BF16>(a, stream);
    if (e != hipSuccess) return e;
    const dim3 grid(static_cast<unsigned>(lists));
    if (a.most_pages <= 1024)
        hipLaunchKernelGGL((block_choose<256, 4>), grid, dim3(256), 0, stream, a);
    else
        hipLaunchKernelGGL((block_choose<1024, 8>), grid, dim3(1024), 0, stream, a);
    return hipGetLastError();
}

}  // namespace ffkv
