// block_select.hip - which pages of its row a block of queries attends, per KV head: a score per page from the page's key
// bounds, and the pages with the largest.
//
//   score(page) = sum over the block's queries and the KV head's query heads of sum_d max(q_d lo_d, q_d hi_d)
//               = sum_d Q-_d lo_d + Q+_d hi_d,   Q- = sum of min(q, 0), Q+ = sum of max(q, 0)
// No query's score with any of the page's keys exceeds its share of that.  The sums over queries and heads go first, so a
// block of any size costs two dot products of head_dim per page.
//
// Scores are fp64 sums rounded once to fp32: they decide between pages, and a row's choice must not depend on the rest of the
// batch or on how the pages are dealt out.  So every form adds up a score in the same order, and the sums over queries too, by
// the query rows of a block: up to kOwnRows one after the other, up to kWideRows by the groups of lanes of 512 threads, every
// so many-th row each, joined wave by wave, more by those of 1024.
//
// Of a block's pages - those up to its last query's - the first `sinks` and the last `recent` are taken, and of the rest
// those with the largest scores, of equal ones the lower; NaN (a NaN key, or infinite ones that cancel) counts as the largest.
// The list is in ascending order, -1 behind.
//
// The bounds are read once (an eighth of K; in 8-bit caches a quarter), 4 bytes a page and list are written and read again: HBM
// for long rows, and two or three launches with their chains of loads (few lists of few pages: one).
#include "blocks.h"
#include "mfma_common.h"

#include <algorithm>

namespace ffkv
{

namespace
{

constexpr int kScoreThreads = 256;
constexpr int kScorePages = 4;  // neighbouring pages that a group of lanes scores together
constexpr int kOneThreads = 512;
constexpr int kOneRounds = 4;  // of block_select_one at most
constexpr int kOwnRows = 8;    // query rows of a block that are added up one after the other
constexpr int kWideRows = 128;  // more of them than that are added up by twice the threads

template <int CTRL>
__device__ __forceinline__ double dpp64(double v)
{
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(u), CTRL, 0xf, 0xf, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(u >> 32), CTRL, 0xf, 0xf, false);
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}

// In the lower half of the lanes (the even rows of 16) a plus that of the lane 32 (16) away, in the others b.
template <bool HALF>
__device__ __forceinline__ double swap_sum64(double a, double b)
{
    const uint64_t x = __builtin_bit_cast(uint64_t, a), y = __builtin_bit_cast(uint64_t, b);
    const uint32_t x0 = static_cast<uint32_t>(x), x1 = static_cast<uint32_t>(x >> 32);
    const uint32_t y0 = static_cast<uint32_t>(y), y1 = static_cast<uint32_t>(y >> 32);
    const auto     l = HALF ? __builtin_amdgcn_permlane32_swap(x0, y0, false, false)
                            : __builtin_amdgcn_permlane16_swap(x0, y0, false, false);
    const auto     h = HALF ? __builtin_amdgcn_permlane32_swap(x1, y1, false, false)
                            : __builtin_amdgcn_permlane16_swap(x1, y1, false, false);
    return __builtin_bit_cast(double, static_cast<uint64_t>(static_cast<uint32_t>(h[0])) << 32 | static_cast<uint32_t>(l[0])) +
           __builtin_bit_cast(double, static_cast<uint64_t>(static_cast<uint32_t>(h[1])) << 32 | static_cast<uint32_t>(l[1]));
}

// The sums over LPP lanes of four values each, value k in the group's lanes with lane % 4 == k: two exchanges halve the
// values a lane holds, the rest add up across the quads (5 exchanges where four sums one by one take 16).
template <int LPP>
__device__ __forceinline__ double group_sums4(const double (&v)[4], int lane)
{
    const bool   b0 = lane & 1, b1 = lane & 2;
    const double a = (b0 ? v[1] : v[0]) + dpp64<0xb1>(b0 ? v[0] : v[1]);  // quad lanes 1, 0, 3, 2
    const double b = (b0 ? v[3] : v[2]) + dpp64<0xb1>(b0 ? v[2] : v[3]);
    double       c = (b1 ? b : a) + dpp64<0x4e>(b1 ? a : b);              // quad lanes 2, 3, 0, 1
    if constexpr (LPP == 8)
        c += dpp64<0x141>(dpp64<0x1b>(c));  // lane 7 - (i ^ 3) of its 8: the other quad's same lane
    else
    {
        c += dpp64<0x124>(c);  // lanes 4 and 8 before it in its row of 16
        c += dpp64<0x128>(c);
    }
    if constexpr (LPP == 32) c = swap_sum64<false>(c, c);
    return c;
}

// Largest x of the wave, in every lane.
__device__ __forceinline__ uint32_t wave_max(uint32_t x)
{
    auto take = [&x](auto ctrl, auto rows, auto zero)
    {
        const uint32_t o = __builtin_amdgcn_update_dpp(0, static_cast<int>(x), decltype(ctrl)::value, decltype(rows)::value, 0xf,
                                                       decltype(zero)::value);
        x = o > x ? o : x;
    };
    using std::integral_constant;
    take(integral_constant<int, 0x111>{}, integral_constant<int, 0xf>{}, integral_constant<bool, true>{});  // row_shr:1
    take(integral_constant<int, 0x112>{}, integral_constant<int, 0xf>{}, integral_constant<bool, true>{});
    take(integral_constant<int, 0x114>{}, integral_constant<int, 0xf>{}, integral_constant<bool, true>{});
    take(integral_constant<int, 0x118>{}, integral_constant<int, 0xf>{}, integral_constant<bool, true>{});
    take(integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{}, integral_constant<bool, false>{});  // row_bcast:15
    take(integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{}, integral_constant<bool, false>{});  // row_bcast:31
    return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(x), 63));
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

// A lane's share of Q- and Q+: its 8 dims of query row r of a block (rows: tokens, and the group's heads of each).
__device__ __forceinline__ size_t query_at(const SelectArgs& a, int b, int t0, int kvh, int r, int c)
{
    const int t = r / a.group;
    return ((static_cast<size_t>(b) * a.seq_len + t0 + t) * a.num_heads + kvh * a.group + r - t * a.group) * a.head_dim + 8 * c;
}
__device__ __forceinline__ void add_query(const float (&x)[8], double (&down)[8], double (&up)[8])
{
#pragma unroll
    for (int e = 0; e < 8; ++e)  // (a NaN goes to both)
    {
        down[e] += static_cast<double>(__builtin_elementwise_minimum(x[e], 0.0f));
        up[e] += static_cast<double>(__builtin_elementwise_maximum(x[e], 0.0f));
    }
}

// The sums over a wave's groups of LPP lanes to part[2][LPP * 8] in LDS: every exchange halves the values that a lane holds.
template <int LPP>
__device__ __forceinline__ void wave_sums(const double (&down)[8], const double (&up)[8], int lane, double* part)
{
    double v[16];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = down[e], v[8 + e] = up[e];
    int n = 16, first = 0;  // values held, and which the first of them is
    if constexpr (LPP == 8)
    {
        n /= 2;
        const bool odd = lane & 8;
#pragma unroll
        for (int i = 0; i < 8; ++i)  // with 8 lanes before it in its row of 16
            v[i] = (odd ? v[i + 8] : v[i]) + dpp64<0x128>(odd ? v[i] : v[i + 8]);
        first += odd ? 8 : 0;
    }
    if constexpr (LPP <= 16)
    {
        n /= 2;
#pragma unroll
        for (int i = 0; i < (LPP == 8 ? 4 : 8); ++i) v[i] = swap_sum64<false>(v[i], v[i + n]);
        first += lane & 16 ? n : 0;
    }
    n /= 2;
#pragma unroll
    for (int i = 0; i < LPP / 4; ++i) v[i] = swap_sum64<true>(v[i], v[i + n]);
    first += lane & 32 ? n : 0;
#pragma unroll
    for (int i = 0; i < LPP / 4; ++i)
    {
        const int k = first + i;
        part[(k >> 3) * (LPP * 8) + 8 * (lane % LPP) + (k & 7)] = v[i];
    }
}

// The lane's share of a page's score, in the order that every form keeps.
__device__ __forceinline__ double lane_score(const double (&down)[8], const double (&up)[8], const double (&lo)[8],
                                             const double (&hi)[8])
{
    double s = 0.0;
#pragma unroll
    for (int e = 0; e < 8; ++e)
    {
        s = __builtin_fma(down[e], lo[e], s);
        s = __builtin_fma(up[e], hi[e], s);
    }
    return s;
}

// The same for a score that came out NaN: a sum of 0 takes nothing of an infinite bound (0 * inf is NaN).  The asm keeps this rare
// case's comparisons out of the loops around it (they took 70 registers there).
__device__ __forceinline__ double sum_times(double q, double bound)
{
    asm volatile("" : "+v"(q), "+v"(bound));
    return q == 0.0 && __builtin_isinf(bound) ? 0.0 : bound;
}
__device__ __forceinline__ double lane_score_infinite(const double (&down)[8], const double (&up)[8], const double (&lo)[8],
                                                      const double (&hi)[8])
{
    double s = 0.0;
#pragma unroll
    for (int e = 0; e < 8; ++e)
    {
        s = __builtin_fma(down[e], sum_times(down[e], lo[e]), s);
        s = __builtin_fma(up[e], sum_times(up[e], hi[e]), s);
    }
    return s;
}

// The scores of four pages, that of page k in the lanes of the group with c % 4 == k; values(k, rare, lo, hi) gives their bounds.
template <int LPP, typename F>
__device__ __forceinline__ double page_scores(const double (&down)[8], const double (&up)[8], int c, F values)
{
    double s[kScorePages], lo[8], hi[8];
#pragma unroll
    for (int k = 0; k < kScorePages; ++k)
    {
        values(k, std::false_type{}, lo, hi);
        s[k] = lane_score(down, up, lo, hi);
    }
    double sum = group_sums4<LPP>(s, c);
    if (__builtin_expect(__any(sum != sum), 0))
    {
#pragma unroll
        for (int k = 0; k < kScorePages; ++k)
        {
            values(k, std::true_type{}, lo, hi);
            s[k] = lane_score_infinite(down, up, lo, hi);
        }
        sum = group_sums4<LPP>(s, c);
    }
    return sum;
}

// Four pages' bounds in flight.  FULL: head_dim fills the LPP lanes.  Pages on no table entry read page 0 instead (a pool has
// one), and lanes past head_dim the first dims: their scores are not used, their sums of queries zero.
template <int BT, int LPP, bool FULL>
struct PageBounds
{
    Raw8 lo[kScorePages], hi[kScorePages];
    int  on;  // bit k: page k is on a table entry

    // Physical pages of logical pages p .. p + 3 below end.
    __device__ __forceinline__ static void entries(const int32_t* table, int p, int end, int (&phys)[kScorePages])
    {
#pragma unroll
        for (int k = 0; k < kScorePages; ++k) phys[k] = p + k < end ? table[p + k] : -1;
    }
    __device__ __forceinline__ void load(const SelectArgs& a, const int (&phys)[kScorePages], int kvh, int c)
    {
        constexpr uint32_t EB = BT == F32 ? 4 : 2;
        const uint32_t D = FULL ? LPP * 8 : a.head_dim;
        const uint32_t stride = a.num_kv_heads * 2u * D * EB;  // bytes of a page: below 2^28
        const char*    base = static_cast<const char*>(a.bounds) + (kvh * 2u * D + (FULL || 8u * c < D ? 8u * c : 0u)) * EB;
        on = 0;
#pragma unroll
        for (int k = 0; k < kScorePages; ++k)
        {
            const bool     ok = phys[k] >= 0 && phys[k] < a.num_blocks;
            const uint32_t page = ok ? phys[k] : 0;
            on |= ok ? 1 << k : 0;
            const char* at = base + static_cast<uint64_t>(page) * stride;
            load_raw8<BT>(at, 0, lo[k]);
            load_raw8<BT>(at, D, hi[k]);
        }
    }
    // RARE: as for the first time (the values of four pages would fill 128 registers from one use to the next).
    template <bool RARE = false>
    __device__ __forceinline__ void values(int k, bool in, double (&l)[8], double (&h)[8]) const
    {
        Raw8 a = lo[k], b = hi[k];
        if constexpr (RARE)
#pragma unroll
            for (int i = 0; i < (BT == F32 ? 8 : 4); ++i) asm volatile("" : "+v"(a.w[i]), "+v"(b.w[i]));
        float x[8], y[8];
        unpack8<BT>(a, x);
        unpack8<BT>(b, y);
#pragma unroll
        for (int e = 0; e < 8; ++e)
        {
            l[e] = static_cast<double>(FULL || in ? x[e] : 0.0f);
            h[e] = static_cast<double>(FULL || in ? y[e] : 0.0f);
        }
    }
};

}  // namespace

// A step (a few query rows, one block of them).  A round is ROUND pages of `heads` KV heads, whose bounds of a page lie
// together (64 rows of 125 to 1000 pages, 8 heads, 148 MB from memory: 41.5 us with one head a round, 39.5 with two, 39.1 with
// four, 38.9 with eight, the choice's 5 among them).  The rounds of all rows and heads form one sequence, of which every
// workgroup takes an equal share, as many workgroups as fit the chip: tiles of their own left it waiting for the longest row
// (57.5 us in all).  LPP lanes take four neighbouring pages' bounds, 8 dims each, and every lane adds up its dims of the
// queries by itself; while a round is added up the next one's bounds are on their way, and the table's entries of the one
// after.  Bound by HBM and by fp64 (a conversion and a product per bound): 4.6 TB/s (4 rows of 8188 pages, 4 heads, 67 MB:
// 14.5 us; the 64 rows above 32 of 38.1 in all).
template <int BT, int QT, int LPP, bool FULL>
__global__ __launch_bounds__(kScoreThreads) void block_scores_step(SelectArgs a, int heads)
{
    const int  ROUND = kScoreThreads / LPP * kScorePages / heads;  // pages of a round
    const int  tid = static_cast<int>(threadIdx.x);
    const int  lane = tid & 63;
    const int  c = tid % LPP, grp = tid / LPP / heads, hd = tid / LPP % heads;
    const bool in = FULL || 8 * c < a.head_dim;
    auto rounds_of = [&](int b) { return (visible_pages(a, b, 0) + ROUND - 1) / ROUND; };

    // this workgroup's share (every wave on its own)
    const int H = a.num_kv_heads / heads;  // blocks of heads
    int64_t   total = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 64)
        total += uniform(wave_sum(b0 + lane < a.batch ? rounds_of(b0 + lane) : 0));
    total *= H;
    const int64_t wgs = min(static_cast<int64_t>(gridDim.x), total);
    if (blockIdx.x >= wgs) return;
    int64_t x0, x1;
    if (total < 1 << 20)  // (their product with the grid's at most 2048 workgroups in 32 bits)
    {
        const uint32_t t = static_cast<uint32_t>(total), w = static_cast<uint32_t>(wgs);
        x0 = blockIdx.x * t / w;
        x1 = (blockIdx.x + 1) * t / w;
    }
    else
    {
        x0 = blockIdx.x * total / wgs;
        x1 = (blockIdx.x + 1) * total / wgs;
    }
    // its first round: row, block of heads, round of the row
    struct Place
    {
        int b, hb, round, rounds;
    };
    Place at{0, 0, 0, 0};
    {
        int64_t base = 0;
        for (int b0 = 0;; b0 += 64)
        {
            const int r = b0 + lane < a.batch ? rounds_of(b0 + lane) : 0;
            const int upto = wave_scan(r);  // (rounds of 64 rows: below 2^31 / 64 pages each)
            const int64_t mine = base + static_cast<int64_t>(upto - r) * H;
            const uint64_t hit = __ballot(mine <= x0 && x0 < mine + static_cast<int64_t>(r) * H);
            if (hit != 0)
            {
                const int l = __ffsll(static_cast<long long>(hit)) - 1;
                at.b = b0 + l;
                at.rounds = __builtin_amdgcn_readlane(r, l);
                const int off = static_cast<int>(x0 - base) - __builtin_amdgcn_readlane(upto - r, l) * H;
                at.hb = off / at.rounds;
                at.round = off - at.hb * at.rounds;
                break;
            }
            base += static_cast<int64_t>(__builtin_amdgcn_readlane(upto, 63)) * H;
        }
    }
    auto next = [&](Place p)
    {
        if (++p.round < p.rounds) return p;
        p.round = 0;
        if (++p.hb < H) return p;
        p.hb = 0;
        do
            p.rounds = ++p.b < a.batch ? rounds_of(p.b) : 1;
        while (p.rounds == 0);
        return p;
    };
    int  phys[kScorePages];
    auto entries = [&](const Place& p)  // (those past the row's last page are not used: they lie in the table's row)
    {
        const int first = p.round * ROUND + grp * kScorePages;
        PageBounds<BT, LPP, FULL>::entries(a.block_table + static_cast<int64_t>(p.b) * a.max_blocks, first, a.most_pages, phys);
    };
    constexpr int QROWS = 4;  // query rows whose loads go out together
    const int     rows = a.seq_len * a.group;
    double        down[8], up[8];
    auto sum_queries = [&](const Place& p)
    {
#pragma unroll
        for (int e = 0; e < 8; ++e) down[e] = up[e] = 0.0;
        for (int r0 = 0; r0 < rows; r0 += QROWS)
        {
            Raw8 q[QROWS];
#pragma unroll
            for (int u = 0; u < QROWS; ++u)
                if (r0 + u < rows && in) load_raw8<QT>(a.q, query_at(a, p.b, 0, p.hb * heads + hd, r0 + u, c), q[u]);
#pragma unroll
            for (int u = 0; u < QROWS; ++u)
                if (r0 + u < rows && in)
                {
                    float x[8];
                    unpack8<QT>(q[u], x);
                    add_query(x, down, up);
                }
        }
    };
    Place ahead = next(at);
    entries(at);
    PageBounds<BT, LPP, FULL> cur, nxt;
    cur.load(a, phys, at.hb * heads + hd, c);
    if (x0 + 1 < x1) entries(ahead);
    sum_queries(at);
    auto round = [&](const PageBounds<BT, LPP, FULL>& cur, PageBounds<BT, LPP, FULL>& nxt, int64_t x)
    {
        if (x + 1 < x1) nxt.load(a, phys, ahead.hb * heads + hd, c);
        const Place after = next(ahead);
        if (x + 2 < x1) entries(after);
        const double sum = page_scores<LPP>(down, up, c, [&](int k, auto rare, double (&lo)[8], double (&hi)[8])
        {
            cur.template values<decltype(rare)::value>(k, in, lo, hi);
        });
        const int    p = at.round * ROUND + grp * kScorePages + (c & 3);
        float*       out = a.scores + (static_cast<int64_t>(at.b) * a.num_kv_heads + at.hb * heads + hd) * a.stride;
        // (behind the row's last page up to stride: read by nobody)
        if (c < 4 && p < a.most_pages) out[p] = cur.on >> c & 1 ? static_cast<float>(sum) : kNegInf;  // on no page: last
        if (x + 1 < x1 && (ahead.b != at.b || ahead.hb != at.hb)) sum_queries(ahead);
        at = ahead;
        ahead = after;
    };
    for (int64_t x = x0; x < x1; x += 2)
    {
        round(cur, nxt, x);
        if (x + 1 < x1) round(nxt, cur, x + 1);
    }
}

// Query rows of a whole block: what the order of its sums goes by (and that of a shorter last block).
__device__ __host__ __forceinline__ int64_t block_rows(int query_block, int seq_len, int group)
{
    return static_cast<int64_t>(query_block < seq_len ? query_block : seq_len) * group;
}

// Few query rows a block: Q- and Q+ by LPP lanes for each block and KV head, the rows one after the other.
template <int QT, int LPP>
__global__ __launch_bounds__(kScoreThreads) void block_queries_few(SelectArgs a, uint32_t sums)
{
    const uint32_t i = blockIdx.x * (kScoreThreads / LPP) + threadIdx.x / LPP;
    const int      c = static_cast<int>(threadIdx.x) % LPP;
    if (i >= sums || 8 * c >= a.head_dim) return;
    const Split u = split_index(i, a.num_kv_heads), v = split_index(u.div, a.lists);
    const int   kvh = u.rem, b = static_cast<int>(v.div);
    const int   t0 = v.rem * a.query_block;
    const int   rows = min(a.query_block, a.seq_len - t0) * a.group;
    constexpr int UN = 4;
    double      down[8], up[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) down[e] = up[e] = 0.0;
    for (int r0 = 0; r0 < rows; r0 += UN)
    {
        Raw8 q[UN];
#pragma unroll
        for (int k = 0; k < UN; ++k)
            if (r0 + k < rows) load_raw8<QT>(a.q, query_at(a, b, t0, kvh, r0 + k, c), q[k]);
#pragma unroll
        for (int k = 0; k < UN; ++k)
            if (r0 + k < rows)
            {
                float x[8];
                unpack8<QT>(q[k], x);
                add_query(x, down, up);
            }
    }
    double* out = a.query_sums + static_cast<int64_t>(i) * 2 * a.head_dim + 8 * c;
#pragma unroll
    for (int e = 0; e < 8; ++e)
    {
        out[e] = down[e];
        out[a.head_dim + e] = up[e];
    }
}

// More of them: Q- and Q+ of every block of queries and KV head, a workgroup each (2 x 512 tokens, 32/8 heads of 128 in blocks of
// 64: 7.1 us, where the workgroups that score would read a block's queries once for every 64 pages).  Whole calls over 2000 pages
// by 512 and 1024 threads, when a wave's sums took twice the exchanges: blocks of 16 tokens 48.8 and 50.7 us, 64 23.4 and 23.0,
// 128 23.5 and 22.4, 512 41.4 and 36.7.  (Now 47.7, 22.4, 22.0 and 36.0 by the rule; blocks of one token by the lanes above 527,
// by 1024 threads 584.)
template <int QT, int LPP, int THREADS>
__global__ __launch_bounds__(THREADS) void block_queries(SelectArgs a)
{
    constexpr int WAVES = THREADS / 64;
    constexpr int STEP = THREADS / LPP;  // query rows that the workgroup takes at a time
    constexpr int UN = 4;
    __shared__ double s_part[WAVES][2][LPP * 8];
    const int64_t wg = blockIdx.x;
    const Split   u = split_index(blockIdx.x, a.num_kv_heads), v = split_index(u.div, a.lists);
    const int     kvh = u.rem, b = static_cast<int>(v.div);
    const int     t0 = v.rem * a.query_block;
    const int     rows = min(a.query_block, a.seq_len - t0) * a.group;
    const int     tid = static_cast<int>(threadIdx.x);
    const int     lane = tid & 63, wave = tid >> 6;
    const int     c = tid % LPP;
    const bool    in = 8 * c < a.head_dim;
    double        down[8], up[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) down[e] = up[e] = 0.0;
    for (int r0 = tid / LPP; r0 < rows; r0 += UN * STEP)
    {
        Raw8 q[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u)
            if (r0 + u * STEP < rows && in) load_raw8<QT>(a.q, query_at(a, b, t0, kvh, r0 + u * STEP, c), q[u]);
#pragma unroll
        for (int u = 0; u < UN; ++u)
            if (r0 + u * STEP < rows && in)
            {
                float x[8];
                unpack8<QT>(q[u], x);
                add_query(x, down, up);
            }
    }
    wave_sums<LPP>(down, up, lane, s_part[wave][0]);
    __syncthreads();
    for (int i = tid; i < 2 * a.head_dim; i += THREADS)
    {
        const int half = i >= a.head_dim, d = i - half * a.head_dim;
        double    s = 0.0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) s += s_part[w][half][d];
        a.query_sums[wg * 2 * a.head_dim + i] = s;
    }
}

// Many blocks of queries: a workgroup holds one round of a row's pages, as fp64, and goes through `per` blocks of queries of
// the row, whose sums block_queries has left, LISTS of them at a time through LDS.  (2 x 8 blocks of 64 queries over 2000 pages,
// 8 heads: 10.5 us, the chain of table and bounds ahead of 3 us of fp64 products, of 24.2 us for the whole call; 256 to 2048
// workgroups in all were within 1 us of each other.)
template <int BT, int LPP, bool FULL>
__global__ __launch_bounds__(kScoreThreads) void block_scores_lists(SelectArgs a, int tiles, int per, int parts)
{
    constexpr int ROUND = kScoreThreads / LPP * kScorePages;
    constexpr int LISTS = 8;
    __shared__ __align__(16) double s_q[LISTS][2][LPP * 8];
    const Split u = split_index(blockIdx.x, tiles), v = split_index(u.div, parts), w = split_index(v.div, a.num_kv_heads);
    const int  p0 = u.rem * ROUND, l0 = v.rem * per, kvh = w.rem, b = static_cast<int>(w.div);
    const int  l1 = min(a.lists, l0 + per);
    const int  tid = static_cast<int>(threadIdx.x);
    const int  c = tid % LPP, grp = tid / LPP;
    const int  D = FULL ? LPP * 8 : a.head_dim;
    const bool in = FULL || 8 * c < D;
    const int  p = p0 + grp * kScorePages;
    int        phys[kScorePages];  // (entries past the row's end are read, not used: they lie in the table's row)
    PageBounds<BT, LPP, FULL>::entries(a.block_table + static_cast<int64_t>(b) * a.max_blocks, p, a.most_pages, phys);
    const int n1 = visible_pages(a, b, l1 - 1);  // earlier blocks see no more
    if (p0 >= n1) return;
#pragma unroll
    for (int k = 0; k < kScorePages; ++k) phys[k] = p + k < n1 ? phys[k] : -1;
    PageBounds<BT, LPP, FULL> raw;
    raw.load(a, phys, kvh, c);
    double lo[kScorePages][8], hi[kScorePages][8];
    uint64_t again = 0;  // some score of the wave is NaN
    for (int m0 = l0; m0 < l1; m0 += LISTS)
    {
        const int m1 = min(l1, m0 + LISTS);
        __syncthreads();  // the sums before are read
        for (int i = tid; i < (m1 - m0) * 2 * D; i += kScoreThreads)
        {
            const int l = i / (2 * D), r = i - l * 2 * D, half = r >= D;
            s_q[l][half][r - half * D] =
                a.query_sums[((static_cast<int64_t>(b) * a.lists + m0 + l) * a.num_kv_heads + kvh) * 2 * D + r];
        }
        __syncthreads();
        if (m0 == l0)
#pragma unroll
            for (int k = 0; k < kScorePages; ++k) raw.values(k, in, lo[k], hi[k]);
        for (int l = m0; l < m1; ++l)
        {
            const int n = visible_pages(a, b, l);
            if (p0 >= n) continue;
            double down[8], up[8], s[kScorePages];
#pragma unroll
            for (int e = 0; e < 8; ++e)
            {
                down[e] = in ? s_q[l - m0][0][8 * c + e] : 0.0;
                up[e] = in ? s_q[l - m0][1][8 * c + e] : 0.0;
            }
#pragma unroll
            for (int k = 0; k < kScorePages; ++k) s[k] = lane_score(down, up, lo[k], hi[k]);
            const double sum = group_sums4<LPP>(s, c);
            again |= __ballot(sum != sum);
            float*       out = a.scores + ((static_cast<int64_t>(b) * a.lists + l) * a.num_kv_heads + kvh) * a.stride;
            if (c < 4 && p + c < n) out[p + c] = raw.on >> c & 1 ? static_cast<float>(sum) : kNegInf;
        }
    }
    if (again == 0) return;
    // Infinite or NaN bounds: all from the start, a page at a time, the lane's places too (what is kept for this rare case takes
    // registers from the loop above, and a wave a SIMD: 8 % of the time and more).
    int id = tid;
    asm volatile("" : "+v"(id));
    const int  c1 = id % LPP, first = p0 + id / LPP * kScorePages;
    const bool in1 = FULL || 8 * c1 < D;
#pragma unroll 1
    for (int l = l0; l < l1; ++l)
    {
        const int n = visible_pages(a, b, l);
        if (p0 >= n) continue;
        const int64_t row = (static_cast<int64_t>(b) * a.lists + l) * a.num_kv_heads + kvh;
        const double* q = a.query_sums + row * 2 * D + (in1 ? 8 * c1 : 0);
        double        down[8], up[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
        {
            down[e] = in1 ? q[e] : 0.0;
            up[e] = in1 ? q[D + e] : 0.0;
        }
#pragma unroll 1
        for (int k = 0; k < kScorePages; ++k)
        {
            const int at = first + k;
            const int page = at < n ? a.block_table[static_cast<int64_t>(b) * a.max_blocks + at] : -1;
            const bool on = page >= 0 && page < a.num_blocks;
            const size_t base = (static_cast<size_t>(on ? page : 0) * a.num_kv_heads + kvh) * 2 * D + (in1 ? 8 * c1 : 0);
            Raw8   x, y;
            double l8[8], h8[8];
            load_raw8<BT>(a.bounds, base, x);
            load_raw8<BT>(a.bounds, base + D, y);
            float fx[8], fy[8];
            unpack8<BT>(x, fx);
            unpack8<BT>(y, fy);
#pragma unroll
            for (int e = 0; e < 8; ++e)
            {
                l8[e] = in1 ? fx[e] : 0.0f;
                h8[e] = in1 ? fy[e] : 0.0f;
            }
            const double one[kScorePages] = {lane_score_infinite(down, up, l8, h8), 0.0, 0.0, 0.0};
            const double sum = group_sums4<LPP>(one, c1);
            if (c1 == 0 && at < n) a.scores[row * a.stride + at] = on ? static_cast<float>(sum) : kNegInf;
        }
    }
}

// One workgroup per list.  The score of the last page to stay: the keys between the smallest and the largest are dealt to
// 2048 bins of one width (neighbouring scores share their leading bits: bins by those would hold nearly all of them, and
// their counts in LDS wait for each other), the bin in which it lies is divided again while it holds more than kChooseMost,
// and those left are ranked against each other.  Then the pages above it and the first of those equal to it are written in
// order.  A thread holds PER neighbouring pages, and a list of up to THREADS * PER is read once.  (512 lists of up to 1000 pages
// 5.3 us, 16 of 8188 7.5: barriers and LDS latency.)
constexpr int kChooseMost = 256;

template <int THREADS>
struct ChooseLds
{
    static constexpr int WAVES = THREADS / 64;
    static constexpr int BINS = 2048;
    __align__(16) int hist[BINS];
    int      tot[WAVES];
    uint32_t ends[2][WAVES];
    uint32_t keys[kChooseMost];
    uint32_t found[3];  // bin, of those in it how many stay, how many it holds
    int      left;
};

// The keys of the thread's pages of the tile from t0 on (rows of scores are whole 16-byte words; past the last page they hold
// anything).
template <int PER>
__device__ __forceinline__ void load_keys(const SelectArgs& a, const float* w, int t0, uint32_t (&x)[PER])
{
    const int i0 = t0 + static_cast<int>(threadIdx.x) * PER;
#pragma unroll
    for (int k = 0; k < PER; k += 4)
    {
        f32x4 v = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (i0 + k < a.most_pages) v = *reinterpret_cast<const f32x4*>(w + i0 + k);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[k + j] = score_key(v[j]);
    }
}

// The choice of a.count of n pages, more than those, by the workgroup: scores w, of which x holds the first tile's keys.
template <int THREADS, int PER>
__device__ __forceinline__ void choose_pages(const SelectArgs& a, const float* w, int n, uint32_t (&x)[PER], int32_t* out,
                                             ChooseLds<THREADS>& m)
{
    constexpr int WAVES = THREADS / 64;
    constexpr int TILE = THREADS * PER;
    constexpr int BINS = ChooseLds<THREADS>::BINS;
    constexpr int BPT = BINS / THREADS;  // bins a thread sums up
    static_assert(PER % 4 == 0 && TILE < 1 << 16, "16-byte reads; counts of a tile in 16 bits");
    const int tid = static_cast<int>(threadIdx.x);
    const int lane = tid & 63, wave = tid >> 6;
    const int lo = a.sinks, hi = n - a.recent;  // the pages between: more than are taken of them
    const int most = a.count - a.sinks - a.recent;
    auto between = [&](int t0, int k) { return t0 + tid * PER + k >= lo && t0 + tid * PER + k < hi; };
    const bool one = n <= TILE;
    uint32_t key = 0;
    int      need = most;
    if (most > 0)
    {
        // the keys' range
        uint32_t least = 0xffffffffu, largest = 0u;
        for (int t0 = 0; t0 < n; t0 += TILE)
        {
            if (!one) load_keys<PER>(a, w, t0, x);
#pragma unroll
            for (int k = 0; k < PER; ++k)
                if (between(t0, k)) least = min(least, x[k]), largest = max(largest, x[k]);
        }
        largest = wave_max(largest);
        least = ~wave_max(~least);
        if (lane == 0) m.ends[0][wave] = least, m.ends[1][wave] = largest;
        for (int i = tid; i < BINS; i += THREADS) m.hist[i] = 0;
        if (tid == 0) m.left = 0;
        __syncthreads();
        const int e = lane < WAVES ? lane : 0;
        least = ~wave_max(~m.ends[0][e]);
        largest = wave_max(m.ends[1][e]);
        for (;;)
        {
            // bins of 2^shift keys from `least` on
            const uint32_t range = largest - least;
            const int      bits = range == 0 ? 0 : 32 - __builtin_clz(range);
            const int      shift = bits > 11 ? bits - 11 : 0;
            for (int t0 = 0; t0 < n; t0 += TILE)
            {
                if (!one) load_keys<PER>(a, w, t0, x);
#pragma unroll
                for (int k = 0; k < PER; ++k)
                    if (between(t0, k) && x[k] >= least && x[k] <= largest) atomicAdd(&m.hist[(x[k] - least) >> shift], 1);
            }
            __syncthreads();
            const int top = BINS - 1 - BPT * tid;  // this thread's bins: top, top - 1, ..
            int       c[BPT], sum = 0;
#pragma unroll
            for (int j = 0; j < BPT; ++j) sum += c[j] = m.hist[top - j];
            const int incl = wave_scan(sum);
            if (lane == 63) m.tot[wave] = incl;
            __syncthreads();
            const int tot = lane < WAVES ? m.tot[lane] : 0;
            int       before = incl - sum + __builtin_amdgcn_readlane(wave_scan(tot) - tot, uniform(wave));
#pragma unroll
            for (int j = 0; j < BPT; ++j)
            {
                if (before < need && need <= before + c[j])
                {
                    m.found[0] = static_cast<uint32_t>(top - j);
                    m.found[1] = static_cast<uint32_t>(need - before);
                    m.found[2] = static_cast<uint32_t>(c[j]);
                }
                before += c[j];
            }
            for (int i = tid; i < BINS; i += THREADS) m.hist[i] = 0;
            __syncthreads();
            least += m.found[0] << shift;
            largest = min(largest - least, (1u << shift) - 1u) + least;  // (the range may end inside its last bin)
            need = static_cast<int>(m.found[1]);
            const int held = static_cast<int>(m.found[2]);
            if (held <= kChooseMost || shift == 0) break;
            __syncthreads();
        }
        if (least == largest)
            key = least;
        else
        {
            for (int t0 = 0; t0 < n; t0 += TILE)
            {
                if (!one) load_keys<PER>(a, w, t0, x);
#pragma unroll
                for (int k = 0; k < PER; ++k)
                    if (between(t0, k) && x[k] >= least && x[k] <= largest) m.keys[atomicAdd(&m.left, 1)] = x[k];
            }
            const int held = static_cast<int>(m.found[2]);
            __syncthreads();
            if (tid < held)
            {
                const uint32_t mine = m.keys[tid];
                int            above = 0, equal = 0;
                for (int j = 0; j < held; ++j)
                {
                    above += m.keys[j] > mine;
                    equal += m.keys[j] == mine;
                }
                if (above < need && need <= above + equal)  // (every one of the equal ones writes the same)
                {
                    m.found[0] = mine;
                    m.found[1] = static_cast<uint32_t>(need - above);
                }
            }
            __syncthreads();
            key = m.found[0];
            need = static_cast<int>(m.found[1]);
        }
        __syncthreads();  // m.tot is read
    }

    // The pages that stay, in order: a thread's place is the number of pages before its own that stay for sure, and of those
    // equal to the key the first `need`.
    int base_sure = 0, base_equal = 0;
    for (int t0 = 0; t0 < n; t0 += TILE)
    {
        if (!one) load_keys<PER>(a, w, t0, x);
        uint32_t sure = 0, equal = 0;  // bit k: of page k
#pragma unroll
        for (int k = 0; k < PER; ++k)
        {
            const int  i = t0 + tid * PER + k;
            const bool mid = between(t0, k) && most > 0;
            sure |= static_cast<uint32_t>(i < lo || (i >= hi && i < n) || (mid && x[k] > key)) << k;
            equal |= static_cast<uint32_t>(mid && x[k] == key) << k;
        }
        const int mine = __popc(sure) | (__popc(equal) << 16);
        const int incl = wave_scan(mine);
        if (lane == 63) m.tot[wave] = incl;
        __syncthreads();
        const int tot = lane < WAVES ? m.tot[lane] : 0;
        const int upto = wave_scan(tot);
        const int before = incl - mine + __builtin_amdgcn_readlane(upto - tot, uniform(wave));
        const int all = __builtin_amdgcn_readlane(upto, 63);
        int       es = base_equal + (before >> 16);
        int       at = base_sure + (before & 0xffff);
#pragma unroll
        for (int k = 0; k < PER; ++k)
        {
            const bool s = sure >> k & 1, q = equal >> k & 1;
            if (s || (q && es < need)) out[at + min(es, need)] = t0 + tid * PER + k;
            at += s;
            es += q;
        }
        base_sure += all & 0xffff, base_equal += all >> 16;
        __syncthreads();
    }
}

template <int THREADS, int PER>
__global__ __launch_bounds__(THREADS) void block_choose(SelectArgs a)
{
    __shared__ ChooseLds<THREADS> s_choose;
    const int64_t wg = blockIdx.x;
    const Split   u = split_index(split_index(blockIdx.x, a.num_kv_heads).div, a.lists);
    const int     b = static_cast<int>(u.div), list = u.rem;
    const float*  w = a.scores + wg * a.stride;
    int32_t*      out = a.blocks + wg * a.count;
    uint32_t      x[PER];
    if (a.most_pages > a.count) load_keys<PER>(a, w, 0, x);  // (on their way while the row's length is)
    const int n = visible_pages(a, b, list);
    if (n <= a.count)
    {
        for (int i = static_cast<int>(threadIdx.x); i < a.count; i += THREADS) out[i] = i < n ? i : -1;
        return;
    }
    choose_pages<THREADS, PER>(a, w, n, x, out, s_choose);
}

// All of a list in one workgroup: the sums of its queries, the scores of its pages, which stay in LDS, and the choice.
template <int BT, int QT, int LPP, bool FULL>
__global__ __launch_bounds__(kOneThreads) void block_select_one(SelectArgs a)
{
    constexpr int PER = 4;                        // pages of a thread in the choice
    constexpr int WAVES = kOneThreads / 64;
    constexpr int SLOTS = kOneThreads / LPP;      // groups of lanes
    constexpr int ROUND = SLOTS * kScorePages;    // pages of a round
    constexpr int UN = 4;                         // query rows whose loads go out together
    constexpr int PARTS = 2 * WAVES * 2 * LPP * 8 * 8, CHOOSE = static_cast<int>(sizeof(ChooseLds<kOneThreads>));
    static_assert(kOneRounds * ROUND <= kOneThreads * PER, "the choice holds all scores");
    __shared__ __align__(16) float s_scores[kOneThreads * PER];
    __shared__ __align__(16) uint8_t s_mem[PARTS > CHOOSE ? PARTS : CHOOSE];
    const int64_t wg = blockIdx.x;
    const Split   u = split_index(blockIdx.x, a.num_kv_heads), v = split_index(u.div, a.lists);
    const int     kvh = u.rem, list = v.rem, b = static_cast<int>(v.div);
    const int     tid = static_cast<int>(threadIdx.x);
    const int     lane = tid & 63, wave = tid >> 6;
    const int     c = tid % LPP, grp = tid / LPP;
    const bool    in = FULL || 8 * c < a.head_dim;
    int32_t*      out = a.blocks + wg * a.count;
    const int     n = visible_pages(a, b, list);
    if (n <= a.count)
    {
        for (int i = tid; i < a.count; i += kOneThreads) out[i] = i < n ? i : -1;
        return;
    }
    const int32_t* table = a.block_table + static_cast<int64_t>(b) * a.max_blocks;
    const int      rounds = (n + ROUND - 1) / ROUND;
    using Bounds = PageBounds<BT, LPP, FULL>;
    int    phys[kScorePages];
    Bounds cur, nxt;
    Bounds::entries(table, grp * kScorePages, n, phys);
    cur.load(a, phys, kvh, c);
    if (rounds > 1) Bounds::entries(table, ROUND + grp * kScorePages, n, phys);

    const int t0 = list * a.query_block;
    const int rows = min(a.query_block, a.seq_len - t0) * a.group;
    const int64_t whole = block_rows(a.query_block, a.seq_len, a.group);
    double    down[8], up[8];
    // Q- and Q+ of rows first, first + step, ..; TWO: and of those half a step behind each, apart.
    auto sum_rows = [&]<bool TWO>(int first, int step, double (&down2)[8], double (&up2)[8])
    {
        constexpr int SETS = TWO ? 2 : 1;
#pragma unroll
        for (int e = 0; e < 8; ++e) down[e] = up[e] = down2[e] = up2[e] = 0.0;
        for (int r0 = first; r0 < rows; r0 += UN * step)
        {
            Raw8 q[SETS][UN];
#pragma unroll
            for (int k = 0; k < UN; ++k)
#pragma unroll
                for (int h = 0; h < SETS; ++h)
                {
                    const int r = r0 + k * step + h * (step / 2);
                    if (r < rows && in) load_raw8<QT>(a.q, query_at(a, b, t0, kvh, r, c), q[h][k]);
                }
#pragma unroll
            for (int k = 0; k < UN; ++k)
#pragma unroll
                for (int h = 0; h < SETS; ++h)
                    if (r0 + k * step + h * (step / 2) < rows && in)
                    {
                        float x[8];
                        unpack8<QT>(q[h][k], x);
                        add_query(x, h == 0 ? down : down2, h == 0 ? up : up2);
                    }
        }
    };
    double down2[8], up2[8];
    if (whole <= kOwnRows)
        sum_rows.template operator()<false>(0, 1, down2, up2);  // every lane its dims of all rows
    else
    {
        // in the order of block_queries: twice the threads are these waves, and as many again
        double*    s_part = reinterpret_cast<double*>(s_mem);  // [wave][2][LPP * 8]
        const bool two = whole > kWideRows;
        if (two)
        {
            sum_rows.template operator()<true>(grp, 2 * SLOTS, down2, up2);
            wave_sums<LPP>(down2, up2, lane, s_part + (WAVES + wave) * (2 * LPP * 8));
        }
        else
            sum_rows.template operator()<false>(grp, SLOTS, down2, up2);
        wave_sums<LPP>(down, up, lane, s_part + wave * (2 * LPP * 8));
        __syncthreads();
        double s = 0.0;  // (as many threads as sums, or more)
        static_assert(2 * LPP * 8 <= kOneThreads, "a sum per thread");
        if (tid < 2 * LPP * 8)
            for (int w0 = 0; w0 < (two ? 2 : 1) * WAVES; w0 += WAVES)
#pragma unroll
                for (int w = 0; w < WAVES; ++w) s += s_part[(w0 + w) * (2 * LPP * 8) + tid];
        __syncthreads();
        if (tid < 2 * LPP * 8) s_part[tid] = s;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 8; ++e)
        {
            down[e] = s_part[8 * c + e];
            up[e] = s_part[LPP * 8 + 8 * c + e];
        }
    }
    for (int r = 0; r < rounds; ++r)
    {
        if (r + 1 < rounds) nxt.load(a, phys, kvh, c);
        if (r + 2 < rounds) Bounds::entries(table, (r + 2) * ROUND + grp * kScorePages, n, phys);
        const double sum = page_scores<LPP>(down, up, c, [&](int k, auto rare, double (&lo)[8], double (&hi)[8])
        {
            cur.template values<decltype(rare)::value>(k, in, lo, hi);
        });
        const int    p = r * ROUND + grp * kScorePages + (c & 3);
        if (c < 4 && p < n) s_scores[p] = cur.on >> c & 1 ? static_cast<float>(sum) : kNegInf;  // on no page: last
        cur = nxt;
    }
    __syncthreads();
    uint32_t x[PER];
    load_keys<PER>(a, s_scores, 0, x);
    choose_pages<kOneThreads, PER>(a, s_scores, n, x, out, *reinterpret_cast<ChooseLds<kOneThreads>*>(s_mem));
}

namespace
{

// Lanes that hold a page's bounds.
int bound_lanes(int head_dim) { return head_dim <= 64 ? 8 : (head_dim <= 128 ? 16 : 32); }

// Blocks of queries that a workgroup of block_scores_lists goes through, over `tiles` rounds of a row: as many as leave two
// workgroups per CU.
int64_t lists_of_workgroup(const SelectArgs& a, int64_t tiles)
{
    const int64_t rows = static_cast<int64_t>(a.batch) * a.num_kv_heads;
    return std::max<int64_t>(1, std::min<int64_t>(a.lists, (rows * tiles * a.lists + 511) / 512));
}

// Threads of block_choose: the fewest that hold a row in registers; a longer row is read again for every pass.  (Whole calls of 2
// rows, 8 heads, by 256, 512 and 1024 threads: 1000 pages 10.1, 11.1, 12.0 us; 2000 13.3, 12.0, 13.0; 4000 21.0, 16.2, 16.7; 8187
// 34.3, 25.1, 21.6.)
int choose_threads(int most_pages) { return most_pages <= 1024 ? 256 : (most_pages <= 4096 ? 512 : 1024); }

template <int BT, int QT, int LPP, bool FULL>
hipError_t launch_scores_l(const SelectArgs& a, hipStream_t stream)
{
    if (select_in_one(a))
    {
        const dim3 grid(static_cast<unsigned>(static_cast<int64_t>(a.batch) * a.lists * a.num_kv_heads));
        hipLaunchKernelGGL((block_select_one<BT, QT, LPP, FULL>), grid, dim3(kOneThreads), 0, stream, a);
        return hipGetLastError();
    }
    constexpr int ROUND = kScoreThreads / LPP * kScorePages;
    const int64_t rows = static_cast<int64_t>(a.batch) * a.num_kv_heads;
    const int64_t all = (a.most_pages + ROUND - 1) / ROUND;  // rounds of a row
    if (!select_by_lists(a.seq_len, a.lists, a.group))
    {
        int heads = 1;  // whose bounds of a page a round takes: they lie together
        while (heads < 8 && a.num_kv_heads % (2 * heads) == 0) heads *= 2;
        const void*   kernel = reinterpret_cast<const void*>(block_scores_step<BT, QT, LPP, FULL>);
        const int64_t most = rows / heads * ((a.most_pages + ROUND / heads - 1) / (ROUND / heads));  // rounds of all
        const int64_t wgs = std::min<int64_t>(decode_mfma_items(kernel, kScoreThreads, 1), most);
        hipLaunchKernelGGL((block_scores_step<BT, QT, LPP, FULL>), dim3(static_cast<unsigned>(wgs)), dim3(kScoreThreads), 0,
                           stream, a, heads);
        return hipGetLastError();
    }
    const uint32_t sums = static_cast<uint32_t>(rows * a.lists);
    constexpr uint32_t FEW = kScoreThreads / LPP;  // blocks of queries of a workgroup
    const int64_t  query_rows = block_rows(a.query_block, a.seq_len, a.group);
    if (query_rows <= kOwnRows)
        hipLaunchKernelGGL((block_queries_few<QT, LPP>), dim3(sums / FEW + (sums % FEW != 0)), dim3(kScoreThreads), 0, stream, a,
                           sums);
    else if (query_rows <= kWideRows)
        hipLaunchKernelGGL((block_queries<QT, LPP, kOneThreads>), dim3(sums), dim3(kOneThreads), 0, stream, a);
    else
        hipLaunchKernelGGL((block_queries<QT, LPP, 2 * kOneThreads>), dim3(sums), dim3(2 * kOneThreads), 0, stream, a);
    const int64_t per = lists_of_workgroup(a, all), parts = (a.lists + per - 1) / per;
    hipLaunchKernelGGL((block_scores_lists<BT, LPP, FULL>), dim3(static_cast<unsigned>(rows * parts * all)), dim3(kScoreThreads), 0,
                       stream, a, static_cast<int>(all), static_cast<int>(per), static_cast<int>(parts));
    return hipGetLastError();
}

template <int BT, int QT>
hipError_t launch_scores_q(const SelectArgs& a, hipStream_t stream)
{
    // lanes that hold a page's bounds
    if (a.head_dim == 64) return launch_scores_l<BT, QT, 8, true>(a, stream);
    if (a.head_dim < 64) return launch_scores_l<BT, QT, 8, false>(a, stream);
    if (a.head_dim < 128) return launch_scores_l<BT, QT, 16, false>(a, stream);
    if (a.head_dim == 128) return launch_scores_l<BT, QT, 16, true>(a, stream);
    return launch_scores_l<BT, QT, 32, true>(a, stream);
}

template <int BT>
hipError_t launch_scores(const SelectArgs& a, hipStream_t stream)
{
    if (a.q_dtype == F32) return launch_scores_q<BT, F32>(a, stream);
    if (a.q_dtype == F16) return launch_scores_q<BT, F16>(a, stream);
    return launch_scores_q<BT, BF16>(a, stream);
}

}  // namespace

// A step sums its few query rows in the workgroups that score, behind the first bounds' loads; several blocks of queries, or more
// than 8 query rows, are summed once, in a launch of their own.  (Whole calls over rows of 1000 pages, 8 KV heads, in place and
// apart: 4 rows with 4, 8, 12, 16 and 32 query rows 10.8, 12.0, 13.4, 14.8 and 20.3 us against 12.6; 32 rows 29.5, 29.8,
// 30.9, 31.8 and 38.5 against 33.5.)
bool select_by_lists(int seq_len, int lists, int group) { return lists > 1 || static_cast<int64_t>(seq_len) * group > kOwnRows; }

// Few lists of few pages: one launch, without a workspace, in which a list has one CU (1.5 us a round).  Rounds of 128 pages at
// head_dim 128, whole calls in the other launches and in one: 8 lists of up to 64 pages 8.3 and 6.2 us, of 250 9.1 and 6.6,
// 128 lists 9.9 and 7.8, 11.4 and 9.6; 32 lists of 1000 11.2 and 17.7; 512 lists of 64 11.9 and 14.4.  Where queries are
// summed apart, 64 lists of 495 pages 14.9 and 10.4, 128 16.1 and 14.6, 128 lists of 1995 23.0 and 31.5.  (The sums have the same
// order in either, so no row's choice depends on which it is.)
bool select_in_one(const SelectArgs& a)
{
    const int64_t lists = static_cast<int64_t>(a.batch) * a.lists * a.num_kv_heads;
    const int     rounds = select_by_lists(a.seq_len, a.lists, a.group) ? kOneRounds : 2;
    return lists <= 256 && a.most_pages <= rounds * (kOneThreads / bound_lanes(a.head_dim) * kScorePages);
}

int64_t select_threads(const SelectArgs& a)
{
    const int64_t rows = static_cast<int64_t>(a.batch) * a.num_kv_heads, lists = rows * a.lists;
    const int64_t choose = lists * choose_threads(a.most_pages);
    if (a.most_pages <= a.count || select_in_one(a) || !select_by_lists(a.seq_len, a.lists, a.group)) return choose;
    const int64_t round = kScoreThreads / bound_lanes(a.head_dim) * kScorePages;
    const int64_t tiles = (a.most_pages + round - 1) / round, per = lists_of_workgroup(a, tiles);
    const int64_t scores = rows * ((a.lists + per - 1) / per) * tiles * kScoreThreads;
    const int64_t query_rows = block_rows(a.query_block, a.seq_len, a.group);
    const int64_t sums = query_rows <= kOwnRows ? 0 : lists * (query_rows <= kWideRows ? 1 : 2) * kOneThreads;
    return std::max(choose, std::max(scores, sums));
}

hipError_t launch_select(const SelectArgs& a, hipStream_t stream)
{
    const int64_t lists = static_cast<int64_t>(a.batch) * a.lists * a.num_kv_heads;
    if (select_threads(a) > kMostThreads) return hipErrorInvalidConfiguration;
    hipError_t e = hipSuccess;
    // (rows that cannot have more pages than are taken need no scores)
    if (a.most_pages > a.count)
        e = a.bounds_dtype == F32 ? launch_scores<F32>(a, stream)
            : a.bounds_dtype == F16 ? launch_scores<F16>(a, stream)
                                    : launch_scores<BF16>(a, stream);
    if (e != hipSuccess || (a.most_pages > a.count && select_in_one(a))) return e;
    const dim3 grid(static_cast<unsigned>(lists));
    const int threads = choose_threads(a.most_pages);
    if (threads == 256)
        hipLaunchKernelGGL((block_choose<256, 4>), grid, dim3(256), 0, stream, a);
    else if (threads == 512)
        hipLaunchKernelGGL((block_choose<512, 8>), grid, dim3(512), 0, stream, a);
    else
        hipLaunchKernelGGL((block_choose<1024, 8>), grid, dim3(1024), 0, stream, a);
    return hipGetLastError();
}

}  // namespace ffkv
