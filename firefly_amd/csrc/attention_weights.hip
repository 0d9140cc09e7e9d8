// attention_weights.hip - the attention weights that the last S tokens of every row give to its cached keys, under a score
// rule: what an engine goes by when it cuts a prompt's cache.
//
// With the scores s of paged_prefill_scored.hip, for row b, KV head v and key j:
//   weights[b, v, j] = decay * prior[b, v, j] + sum over the S queries t and the query heads h of v of softmax(s_{t,h})_j
// (keys of the S tokens themselves have no earlier weight).  No values, no output: K is read twice, V not at all.
//
// The sum over queries needs every query's final maximum and denominator first, so there are three launches: the states
// (max, denominator) of every query row over each split of the keys, their fold, and the weights, which compute the scores
// again.  (Written down instead, the scores of S * G query rows take 4 S G bytes per key, more than reading its K again
// from 32 rows on.)  A workgroup of the first and third has the keys in its registers, as MFMA operands that serve all query
// rows, and the query rows pass by in LDS.
//
// Bound by vector work (per score a cap, a maximum or a sum, an exponential, 25 instructions with what is shared) and, with
// few query rows, by the latency of loads that one chunk after the other waits for.  Measured (32/8 heads of 128 dims): 32
// tokens over one row of 32.7k, bf16, 47 us (two passes of 22 over 67 MB, the fold 4); 16 x 64 tokens over int8 rows of 400 to
// 4000 under a cap 147 us (72 and 70; the products alone are 14 each at the rate of a large one, and vector instructions
// take 80 % of the issue slots).
#include "mfma_common.h"
#include "score_rule.h"
#include "weight_rows.h"

namespace ffkv
{

namespace
{

constexpr int kAwWaves = 8;
constexpr int kAwThreads = 64 * kAwWaves;
constexpr int kAwPages = 2;  // pages of keys a wave holds: 32 registers of 16-bit operands at head_dim 128
constexpr int kAwChunk = kAwWaves * kAwPages * kBlockSize;  // keys of a workgroup at a time
// q in two parts, as where it is of another type than the products.
template <int CT, int QT>
constexpr bool kAwLo = !((QT == BF16 && (kBF<CT, QT> || CT == I8)) || (QT == F16 && !kBF<CT, QT>));
// Query rows staged in LDS at a time: 32 KiB of them, at most 256 (with 64 KiB a CU has one workgroup of the states' pass
// instead of three: 16 x 64 tokens over int8 pages 255 -> 224 us).
template <int D, bool LO>
constexpr int kAwRows = []
{
    const int r = 32768 / (D * 2 * (LO ? 2 : 1)) / 16 * 16;
    return r > 256 ? 256 : r;
}();
// LDS of a workgroup that stages `rows` of them.
template <int D, bool LO>
constexpr int aw_lds(int rows, bool sum)
{
    const int q = rows * (LO ? 2 : 1) * D * 2;
    return q + rows * (16 + 8 * (sum ? 1 : kAwWaves) + 4);
}
constexpr int kAwVecRows = 256;  // the vector kernel's, of which it stages 32 at a time
constexpr int kAwVecTile = 32;
constexpr int kAwVecThreads = 256;
constexpr int kAwVecWaves = kAwVecThreads / 64;
constexpr int kAwVecChunk = kAwVecThreads;
static_assert(kAwVecChunk == kAwChunk, "one number of splits");
constexpr int kAwMost = 512;  // workgroups, but for more rows times KV heads (attention_weights_splits)

// Keys [x, y) that query token t of row b sees among its row's `total` tokens; z: its position.
__device__ __forceinline__ int3 aw_visible(const WeightArgs& a, int b, int64_t ctx, int total, int t)
{
    const int64_t at = static_cast<int64_t>(b) * a.seq_len + t;
    int64_t       hi = a.rule.key_end != nullptr ? a.rule.key_end[at] : ctx + t + 1;
    hi = hi > total ? total : (hi < 0 ? 0 : hi);
    int64_t lo = first_key(a.rule, ctx + t, a.rule.key_begin != nullptr ? a.rule.key_begin[at] : 0);
    lo = lo > hi ? hi : lo;
    return make_int3(static_cast<int>(lo), static_cast<int>(hi), static_cast<int>(ctx + t));
}

__device__ __forceinline__ int aw_total(const WeightArgs& a, int64_t ctx)
{
    int64_t total = ctx + a.seq_len;
    if (total > a.cap_tokens) total = a.cap_tokens;
    return total < 0 ? 0 : static_cast<int>(total);
}

// A workgroup's share of the call: chunks split, split + splits, .. of row b's keys for KV head kvh, and the slot of its states
// (of a row's splits, of seq_len * group states each) in a.part.  b < 0: none.
struct AwShare
{
    int     b, kvh, split, splits;
    int64_t slot;
};

// Share `i` of the call's batch * num_kv_heads * a.splits; or, with i < 0, row b's first one (kvh 0).  Every row is cut into
// pieces of the same number of chunks, the fewest that leave no more pieces than there are shares (each row a.splits
// instead: 16 x 64 tokens over rows of 400 to 4000 on int8 pages 164 us, 146 so).  All waves find it by themselves.
__device__ __forceinline__ AwShare aw_share(const WeightArgs& a, int i, int b_of)
{
    const int H = a.num_kv_heads;
    const int at = i / H, kvh = i - at * H;  // (a KV head per XCD where there are eight: 5 % faster than a stretch of rows)
    if (a.splits == 1 || a.batch == 1)
    {
        if (i < 0) return AwShare{b_of, 0, 0, a.splits, static_cast<int64_t>(b_of) * H * a.splits};
        const int b = a.splits == 1 ? at : 0, split = a.splits == 1 ? 0 : at;
        return AwShare{b, kvh, split, a.splits, (static_cast<int64_t>(b) * H + kvh) * a.splits + split};
    }
    constexpr int N = kAwMost / 2 / 64;  // batch <= kAwMost / 2, as there are two splits and more
    const int lane = static_cast<int>(threadIdx.x) & 63;
    const int budget = a.batch * a.splits;
    int       c[N], total = 0;
#pragma unroll
    for (int k = 0; k < N; ++k)
    {
        const int r = 64 * k + lane;
        c[k] = r < a.batch ? (aw_total(a, a.context_lens[r]) + kAwChunk - 1) / kAwChunk : 0;
        total += c[k];
    }
    total = __builtin_amdgcn_readlane(wave_scan(total), 63);
    int len = max(1, (total + budget - 1) / budget);
    int s[N];
    for (;; len += 1 + len / 16)  // (ends: at the longest row's length every row is one piece)
    {
        int n = 0;
#pragma unroll
        for (int k = 0; k < N; ++k)
        {
            s[k] = 64 * k + lane < a.batch ? max(1, (c[k] + len - 1) / len) : 0;
            n += s[k];
        }
        if (__builtin_amdgcn_readlane(wave_scan(n), 63) <= budget) break;
    }
    AwShare got{-1, 0, 0, 1, 0};
    int     base = 0;
#pragma unroll
    for (int k = 0; k < N; ++k)
    {
        const int      incl = wave_scan(s[k]), excl = base + incl - s[k];
        const uint64_t hit = __ballot(i < 0 ? 64 * k + lane == b_of : at >= excl && at < excl + s[k]);
        if (hit != 0)
        {
            const int l = __ffsll(static_cast<long long>(hit)) - 1;
            const int first = __builtin_amdgcn_readlane(excl, l), n = __builtin_amdgcn_readlane(s[k], l);
            got.b = 64 * k + l;
            got.splits = n;
            got.split = i < 0 ? 0 : at - first;
            got.kvh = i < 0 ? 0 : kvh;
            got.slot = static_cast<int64_t>(first) * H + static_cast<int64_t>(got.kvh) * n + got.split;
        }
        base += __builtin_amdgcn_readlane(incl, 63);
    }
    return got;
}

// Chunks [x, y) of row b that some query sees: the others' keys are not read (without queries, none).  Every wave by itself, a
// lane a query.
__device__ __forceinline__ int2 aw_chunks(const WeightArgs& a, int b, int64_t ctx, int total)
{
    if (a.seq_len == 0) return make_int2(0, 0);
    const int all = (total + kAwChunk - 1) / kAwChunk;
    if (a.rule.window <= 0 && a.rule.key_begin == nullptr && a.rule.key_end == nullptr) return make_int2(0, all);
    int lo = INT32_MAX, hi = 0;
    for (int t = static_cast<int>(threadIdx.x) & 63; t < a.seq_len; t += 64)
    {
        const int3 vis = aw_visible(a, b, ctx, total, t);
        if (vis.x < vis.y)
        {
            lo = min(lo, vis.x);
            hi = max(hi, vis.y);
        }
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1)
    {
        lo = min(lo, __shfl_xor(lo, off, 64));
        hi = max(hi, __shfl_xor(hi, off, 64));
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    hi = __builtin_amdgcn_readfirstlane(hi);
    return lo < hi ? make_int2(lo / kAwChunk, (hi + kAwChunk - 1) / kAwChunk) : make_int2(0, 0);
}

// A state's (max, denominator) joined with another's; the maxima are finite or NaN (kLowest where there was no key).
__device__ __forceinline__ float2 aw_join(float2 x, float2 y)
{
    const float m = __builtin_elementwise_maximum(x.x, y.x);
    return make_float2(m, x.y * __builtin_amdgcn_exp2f(x.x - m) + y.y * __builtin_amdgcn_exp2f(y.x - m));
}

__device__ __forceinline__ void aw_store(const WeightArgs& a, int64_t bh, int64_t ctx, int total, int key, float w)
{
    if (key >= total) return;
    const int64_t at = bh * a.weight_stride + key;
    if (a.prior != nullptr && key < ctx) w = __builtin_fmaf(a.decay, a.prior[at], w);
    a.weights[at] = w;
}

}  // namespace

// Workgroup blockIdx.x: the keys of its share (aw_share).  SUM = false: the states of query rows blockIdx.y * block_rows ..
// over them; SUM = true: the weights of them over all query rows.
template <int CT, int QT, int D, bool SUM>
__global__ __launch_bounds__(kAwThreads) __attribute__((amdgpu_waves_per_eu(D <= 128 ? 4 : 2, 8))) void attention_weights_mfma(WeightArgs a)
{
    constexpr bool BF = kBF<CT, QT>;
    using M = MType<BF>;
    using X8 = typename M::x8;
    using X4 = typename M::x4;
    constexpr int  KSTEPS = D / 32;
    constexpr bool KT = D % 32 == 16;  // a last k-step of 16 dims
    constexpr int  DT = 32 * KSTEPS;
    // int8 beside a bf16 q: f16 products with q converted whole (8 significant bits in 11), each row scaled by a power of two
    // into f16's range where one of its tile holds values of 2^15 and more
    constexpr bool QX16 = CT == I8 && QT == BF16;
    constexpr bool LO = kAwLo<CT, QT>;
    constexpr int  KP = kAwPages;
    constexpr int  CHUNK = kAwChunk;
    constexpr int  NP = LO ? 2 : 1;  // parts of q
    auto dimof = [](int j, int g)    // first of the 8 dims of k-step j in lane group g (as the decode's)
    {
        if constexpr (kElemBytes<CT> == 1 && KSTEPS % 2 == 1)
            if (j == KSTEPS - 1) return 32 * j + 8 * g;
        return dim_of<CT>(j, g);
    };
    // LDS for the query rows that a workgroup stages (a.block_rows, at most RB), aw_lds bytes: q as MFMA operands in the
    // order the lanes read them, [tile][part][k-step][lane], the last k-step's, what the rows see, (max, 1 / denominator) of
    // the rows (SUM) or every wave's states of them, slopes
    extern __shared__ __align__(16) uint8_t s_aw[];
    const int rows = a.block_rows;
    u32x4*    s_q = reinterpret_cast<u32x4*>(s_aw);
    u32x2*    s_qt = reinterpret_cast<u32x2*>(s_q + rows / 16 * NP * KSTEPS * 64);
    int4*     s_vis = reinterpret_cast<int4*>(s_qt + (KT ? rows / 16 * NP * 64 : 0));
    float2*   s_ml = reinterpret_cast<float2*>(s_vis + rows);
    float*    s_slope = reinterpret_cast<float*>(s_ml + (SUM ? 1 : kAwWaves) * rows);

    const int tid = static_cast<int>(threadIdx.x);
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15;
    const int g = lane >> 4;
    const AwShare share = aw_share(a, static_cast<int>(blockIdx.x), 0);
    const int     b = share.b, kvh = share.kvh, split = share.split, splits = share.splits;
    if (b < 0) return;
    const int bh = b * a.num_kv_heads + kvh;
    const int G = a.group;
    const int R = a.seq_len * G;
    const int64_t ctx = a.context_lens[b];
    const int total = __builtin_amdgcn_readfirstlane(aw_total(a, ctx));
    const int chunks = (total + CHUNK - 1) / CHUNK;
    const int2 live = aw_chunks(a, b, ctx, total);
    const int  first = live.x <= split ? split : split + (live.x - split + splits - 1) / splits * splits;  // of this share
    const int blocks = weight_row_blocks(R, rows);
    const int32_t* table = a.block_table + static_cast<int64_t>(b) * a.max_blocks;
    // from products to scores in log2 units, or in those of the cap (int8: times the key's scale)
    float factor = a.rule.cap > 0.0f ? a.scale_log2 * a.rule.inv_cap : a.scale_log2;
    if constexpr (CT == FP8) factor *= a.k_scale[kvh];

    // A wave stages whole tiles of 16 query rows: lane (c, g) row c's dims dimof(j, g) .. of every k-step.
    auto stage = [&](int rb)
    {
        const int r0 = rb * rows;
        const int tiles = (min(rows, R - r0) + 15) / 16;
        auto parts = [&]<int N>(const float (&x)[N], uint32_t (&hi)[N], uint32_t (&lo)[N])
        {
#pragma unroll
            for (int e = 0; e < N; ++e)
            {
                hi[e] = M::bits(x[e]);
                lo[e] = LO ? M::bits(x[e] - M::value(hi[e])) : 0u;
            }
        };
        for (int tile = wave; tile < tiles; tile += kAwWaves)
        {
            const int    r = r0 + tile * 16 + c;
            const int    t = r / G, h = r - t * G;
            const size_t at = ((static_cast<size_t>(b) * a.seq_len + t) * a.num_heads + kvh * G + h) * D;
            float        most = 0.0f;  // QX16: the largest |q| of the lane's dims
            auto stage_tile = [&](float qs)
            {
                u32x4* dst = s_q + tile * NP * KSTEPS * 64 + lane;
#pragma unroll
                for (int j = 0; j < KSTEPS; ++j)
                {
                    u32x4 hi = u32x4{0u, 0u, 0u, 0u}, lo = hi;
                    if (r < R)
                    {
                        if constexpr (QX16)
                        {
                            float    x[8];
                            uint32_t w[4];
                            load_q8<QT>(a.q, at + dimof(j, g), x);
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                            {
                                most = fmaxf(most, fmaxf(__builtin_fabsf(x[2 * e]), __builtin_fabsf(x[2 * e + 1])));
                                w[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{x[2 * e] * qs, x[2 * e + 1] * qs}, h2));
                            }
                            hi = u32x4{w[0], w[1], w[2], w[3]};
                        }
                        else if constexpr (!LO)
                            hi = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.q) + at + dimof(j, g));
                        else
                        {
                            float    x[8];
                            uint32_t p[8], w[8];
                            load_q8<QT>(a.q, at + dimof(j, g), x);
                            parts(x, p, w);
                            hi = u32x4{p[0] | (p[1] << 16), p[2] | (p[3] << 16), p[4] | (p[5] << 16), p[6] | (p[7] << 16)};
                            lo = u32x4{w[0] | (w[1] << 16), w[2] | (w[3] << 16), w[4] | (w[5] << 16), w[6] | (w[7] << 16)};
                        }
                    }
                    dst[j * 64] = hi;
                    if constexpr (LO) dst[(KSTEPS + j) * 64] = lo;
                }
                if constexpr (KT)
                {
                    float    x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    uint32_t p[4], w[4];
                    if (r < R) load_act4(a.q, QT, at + DT + 4 * g, x);
                    if constexpr (QX16)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                        {
                            most = fmaxf(most, __builtin_fabsf(x[e]));
                            x[e] *= qs;
                        }
                    parts(x, p, w);
                    s_qt[tile * NP * 64 + lane] = u32x2{p[0] | (p[1] << 16), p[2] | (p[3] << 16)};
                    if constexpr (LO) s_qt[(tile * NP + 1) * 64 + lane] = u32x2{w[0] | (w[1] << 16), w[2] | (w[3] << 16)};
                }
            };
            stage_tile(1.0f);
            float unscale = 1.0f;
            if constexpr (QX16)
                if (__any(most >= 32768.0f))  // rare: again, every row scaled by its largest finite value
                {
                    float fin = 0.0f;
                    auto  take = [&](float x)
                    { fin = fmaxf(fin, __builtin_fabsf(x) < __builtin_huge_valf() ? __builtin_fabsf(x) : 0.0f); };
                    if (r < R)
                    {
#pragma unroll 1
                        for (int j = 0; j < KSTEPS; ++j)
                        {
                            float x[8];
                            load_q8<QT>(a.q, at + dimof(j, g), x);
#pragma unroll
                            for (int e = 0; e < 8; ++e) take(x[e]);
                        }
                        if constexpr (KT)
                        {
                            float x[4];
                            load_act4(a.q, QT, at + DT + 4 * g, x);
#pragma unroll
                            for (int e = 0; e < 4; ++e) take(x[e]);
                        }
                    }
                    fin = fmaxf(fin, __shfl_xor(fin, 16, 64));
                    fin = fmaxf(fin, __shfl_xor(fin, 32, 64));
                    const int e = max(0, __builtin_amdgcn_frexp_expf(fin) - 15);
                    unscale = __builtin_ldexpf(1.0f, e);
                    stage_tile(__builtin_ldexpf(1.0f, -e));
                }
            if (g == 0)
            {
                const int3 vis = r < R ? aw_visible(a, b, ctx, total, t) : make_int3(0, 0, 0);
                s_vis[tile * 16 + c] = make_int4(vis.x, vis.y, vis.z, __builtin_bit_cast(int, unscale));
                s_slope[tile * 16 + c] = r < R && a.rule.slopes != nullptr ? a.rule.slopes[kvh * G + h] * 1.4426950408889634f : 0.0f;
                if constexpr (SUM)
                    s_ml[tile * 16 + c] = r < R ? a.fin[static_cast<int64_t>(bh) * R + r] : make_float2(0.0f, 0.0f);
            }
        }
        __syncthreads();
        return tiles;
    };

    const int rb0 = SUM ? 0 : static_cast<int>(blockIdx.y);
    int       tiles = 0;
    if constexpr (!SUM)
        for (int i = lane; i < rows; i += 64) s_ml[wave * rows + i] = make_float2(kLowest, 0.0f);

    // This wave's keys of a chunk, as loaded: lane (c, g) holds dims dimof(j, g) .. + 7 of key c of each page.  (Loading the
    // next chunk's ahead of this one's products took the registers over 128 and was no faster: one row of 32.7k tokens 58 us
    // against 51, and 184 against 187 on 16 rows of int8 pages; the first chunk's ahead of the query rows 48 against 47.)
    constexpr int NW = kElemBytes<CT> == 2 ? KSTEPS : (KSTEPS + 1) / 2;
    struct Keys
    {
        u32x4 k[KP][NW > 0 ? NW : 1];
        u32x2 kt[KP];
        f32x4 ks[CT == I8 ? KP : 1];
        int   okm;  // pages that are there
    };
    auto load_keys = [&](int ch, Keys& w)
    {
        w.okm = 0;
#pragma unroll
        for (int u = 0; u < KP; ++u)
        {
            const int  pg = (ch * CHUNK + wave * (KP * kBlockSize)) / kBlockSize + u;
            const int  phys = pg * kBlockSize < total ? __builtin_amdgcn_readfirstlane(table[pg]) : -1;
            const bool ok = phys >= 0 && phys < a.num_blocks;
            w.okm |= ok ? 1 << u : 0;
            const size_t row = (static_cast<size_t>(ok ? phys : 0) * kBlockSize + c) * a.num_kv_heads + kvh;
            const char*  kp = static_cast<const char*>(a.k_cache) + row * D * kElemBytes<CT>;
#pragma unroll
            for (int j = 0; j < NW; ++j)
            {
                w.k[u][j] = u32x4{0u, 0u, 0u, 0u};
                if (!ok) continue;
                if constexpr (kElemBytes<CT> == 2)
                    w.k[u][j] = *reinterpret_cast<const u32x4*>(kp + 2 * dimof(j, g));
                else if (2 * j + 1 < KSTEPS)  // two k-steps' codes
                    w.k[u][j] = *reinterpret_cast<const u32x4*>(kp + dimof(2 * j, g));
                else
                {
                    const u32x2 t = *reinterpret_cast<const u32x2*>(kp + dimof(2 * j, g));
                    w.k[u][j] = u32x4{t[0], t[1], 0u, 0u};
                }
            }
            if constexpr (KT)
            {
                w.kt[u] = u32x2{0u, 0u};
                if (ok)
                {
                    if constexpr (kElemBytes<CT> == 2)
                        w.kt[u] = *reinterpret_cast<const u32x2*>(kp + 2 * (DT + 4 * g));
                    else
                        w.kt[u][0] = *reinterpret_cast<const uint32_t*>(kp + DT + 4 * g);
                }
            }
            if constexpr (CT == I8)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    w.ks[u][i] =
                        ok ? a.k_scale[(static_cast<size_t>(phys) * kBlockSize + 4 * g + i) * a.num_kv_heads + kvh] : 0.0f;
        }
    };
    if (first < live.y && (!SUM || blocks == 1)) tiles = stage(rb0);
    for (int ch = SUM ? split : first; ch < (SUM ? chunks : live.y); ch += splits)
    {
        const int key0 = ch * CHUNK + wave * (KP * kBlockSize);
        if (SUM && (ch < live.x || ch >= live.y))  // seen by none: what it had
        {
            if (lane < KP * kBlockSize) aw_store(a, bh, ctx, total, key0 + lane, 0.0f);
            continue;
        }
        Keys raw_keys;
        load_keys(ch, raw_keys);
        X8        k[KP][KSTEPS > 0 ? KSTEPS : 1];
        X4        kt[KP];
        f32x4     ks[CT == I8 ? KP : 1];
        const int okm = raw_keys.okm;
#pragma unroll
        for (int u = 0; u < KP; ++u)
        {
#pragma unroll
            for (int j = 0; j < KSTEPS; ++j)
            {
                if constexpr (kElemBytes<CT> == 2)
                    k[u][j] = __builtin_bit_cast(X8, raw_keys.k[u][j]);
                else
                {
                    const u32x4 w = raw_keys.k[u][j / 2];
                    k[u][j] = __builtin_bit_cast(X8, j & 1 ? codes_to_m<CT, BF>(w[2], w[3]) : codes_to_m<CT, BF>(w[0], w[1]));
                }
            }
            if constexpr (KT)
            {
                u32x2 w = raw_keys.kt[u];
                if constexpr (kElemBytes<CT> == 1)
                {
                    const u32x4 m = codes_to_m<CT, BF>(w[0], 0u);
                    w = u32x2{m[0], m[1]};
                }
                kt[u] = __builtin_bit_cast(X4, w);
            }
            if constexpr (CT == I8) ks[u] = raw_keys.ks[u] * factor;
        }
        float acc[KP * 4];  // SUM: this lane's columns' weights of key 4g + i of page u
#pragma unroll
        for (int e = 0; e < KP * 4; ++e) acc[e] = 0.0f;
        for (int rb = rb0; rb < (SUM ? blocks : rb0 + 1); ++rb)
        {
            if (SUM && blocks > 1)
            {
                __syncthreads();  // the last block's rows are done with
                tiles = stage(rb);
            }
            for (int tile = 0; tile < tiles; ++tile)
            {
                const int4 vis = s_vis[tile * 16 + c];
                if (!__any(vis.x < vis.y && vis.x < key0 + KP * kBlockSize && vis.y > key0)) continue;
                f32x4 s[KP];
#pragma unroll
                for (int u = 0; u < KP; ++u) s[u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int j = 0; j < KSTEPS; ++j)
#pragma unroll
                    for (int p = 0; p < NP; ++p)
                    {
                        const X8 q = __builtin_bit_cast(X8, s_q[((tile * NP + p) * KSTEPS + j) * 64 + lane]);
#pragma unroll
                        for (int u = 0; u < KP; ++u) s[u] = M::mma32(k[u][j], q, s[u]);
                    }
                if constexpr (KT)
#pragma unroll
                    for (int u = 0; u < KP; ++u)
                    {
                        // (accumulated apart and joined by vector adds, as in the decode: the 16x16x16 product chained on the
                        // 16x16x32 ones' result got no wait states between them)
                        f32x4 st = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int p = 0; p < NP; ++p)
                            st = M::mma16(kt[u], __builtin_bit_cast(X4, s_qt[(tile * NP + p) * 64 + lane]), st);
                        s[u] += st;
                    }
                // Without a cap or a bias the factor is left to the exponent's multiply-add (int8 keys have one each; an fp8
                // head's scale may be negative or zero, which would turn the maximum around).
                const bool raw = CT != I8 && a.rule.cap <= 0.0f && a.rule.slopes == nullptr && factor > 0.0f;
                float      v[KP * 4];
                if (raw)
                {
#pragma unroll
                    for (int e = 0; e < KP * 4; ++e) v[e] = s[e >> 2][e & 3];
                }
                else
#pragma unroll
                for (int e = 0; e < KP * 4; ++e) v[e] = s[e >> 2][e & 3] * (CT == I8 ? ks[e >> 2][e & 3] : factor);
                if constexpr (QX16)
                    if (__any(vis.w != 0x3f800000))  // rare: the row's scale of q
#pragma unroll
                        for (int e = 0; e < KP * 4; ++e) v[e] *= __builtin_bit_cast(float, vis.w);
                if (a.rule.cap > 0.0f) cap_scores<KP * 4>(v, a.rule.cap);
                if (a.rule.slopes != nullptr)
                {
                    const float slope = -s_slope[tile * 16 + c];
                    const float d0 = static_cast<float>(key0 + 4 * g - vis.z);
#pragma unroll
                    for (int e = 0; e < KP * 4; ++e)
                        v[e] = __builtin_fmaf(slope, __builtin_fabsf(d0 + static_cast<float>(16 * (e >> 2) + (e & 3))), v[e]);
                }
                const bool masked = okm != (1 << KP) - 1 || !__all(vis.x <= key0 && vis.y >= key0 + KP * kBlockSize);
                if (masked)
                {
#pragma unroll
                    for (int e = 0; e < KP * 4; ++e)
                    {
                        const int  key = key0 + 4 * g + 16 * (e >> 2) + (e & 3);
                        const bool seen = (okm >> (e >> 2) & 1) && key >= vis.x && key < vis.y;
                        v[e] = seen ? v[e] : kNegInf;
                    }
                }
                if constexpr (SUM)
                {
                    const float2 f = s_ml[tile * 16 + c];
#pragma unroll
                    for (int e = 0; e < KP * 4; ++e)
                        v[e] = __builtin_amdgcn_exp2f(CT == I8 ? v[e] - f.x : __builtin_fmaf(v[e], raw ? factor : 1.0f, -f.x));
                    // A NaN query's state: NaN for the keys it sees alone.  (By its bits: from `f.y < infinity` in a vote the
                    // compiler made an unordered compare, which a NaN passes.)
                    if (masked && __any((f2u(f.y) & 0x7fffffffu) > 0x7f800000u))
                    {
#pragma unroll
                        for (int e = 0; e < KP * 4; ++e)
                        {
                            const int  key = key0 + 4 * g + 16 * (e >> 2) + (e & 3);
                            const bool seen = (okm >> (e >> 2) & 1) && key >= vis.x && key < vis.y;
                            acc[e] += seen ? v[e] * f.y : 0.0f;
                        }
                    }
                    else
#pragma unroll
                        for (int e = 0; e < KP * 4; ++e) acc[e] = __builtin_fmaf(v[e], f.y, acc[e]);
                }
                else
                {
                    const float k1 = raw ? factor : 1.0f;
                    float       m = kNegInf, l = 0.0f;
#pragma unroll
                    for (int e = 0; e < KP * 4; ++e) m = __builtin_elementwise_maximum(m, v[e]);
                    m = __builtin_elementwise_maximum(swap_max(m) * k1, kLowest);
#pragma unroll
                    for (int e = 0; e < KP * 4; ++e)
                        l += __builtin_amdgcn_exp2f(CT == I8 ? v[e] - m : __builtin_fmaf(v[e], k1, -m));
                    l = swap_sum(l);
                    if (g == 0)
                    {
                        float2& st = s_ml[wave * rows + tile * 16 + c];
                        st = ch == first ? make_float2(m, l) : aw_join(st, make_float2(m, l));
                    }
                }
            }
        }
        if constexpr (SUM)
        {
            // lane c of each 16 takes key 16 (c / 4) + 4g + c % 4 of the wave's
            float w = 0.0f;
#pragma unroll
            for (int e = 0; e < KP * 4; ++e)
            {
                const float t = group_sum<16>(acc[e]);
                w = c == e ? t : w;
            }
            if (c < KP * 4) aw_store(a, bh, ctx, total, key0 + 16 * (c >> 2) + 4 * g + (c & 3), w);
        }
    }
    if constexpr (!SUM)
    {
        __syncthreads();
        for (int i = tid; i < rows; i += kAwThreads)
        {
            const int r = rb0 * rows + i;
            if (r >= R) break;
            float2 st = s_ml[i];
#pragma unroll
            for (int w = 1; w < kAwWaves; ++w) st = aw_join(st, s_ml[w * rows + i]);
            a.part[share.slot * R + r] = st;
        }
    }
}

// The same with vector arithmetic (fp32 caches, and head dims that the matrix cores do not take): a thread has a key, 32
// query rows at a time pass by in LDS.  Bound by its loads: a thread reads its own key, 32 bytes at a time, and again for every
// 32 query rows (32/8 heads of 128 dims, fp32: 32 tokens over one row of 32.7k 525 us, 16 x 64 tokens over 400 to 4000 1.5 ms).
template <int CT, bool SUM>
__global__ __launch_bounds__(kAwVecThreads) void attention_weights_vector(WeightArgs a)
{
    constexpr int T = kAwVecTile;
    __shared__ float  s_q[T][256];
    __shared__ int3   s_vis[T];
    __shared__ float  s_slope[T];
    __shared__ float2 s_ml[SUM ? 1 : kAwVecWaves][SUM ? T : kAwVecRows];
    const int D = a.head_dim;
    const int tid = static_cast<int>(threadIdx.x);
    const int lane = tid & 63;
    const int wave = tid >> 6;
    const AwShare share = aw_share(a, static_cast<int>(blockIdx.x), 0);
    const int     b = share.b, kvh = share.kvh, split = share.split, splits = share.splits;
    if (b < 0) return;
    const int bh = b * a.num_kv_heads + kvh;
    const int G = a.group;
    const int R = a.seq_len * G;
    const int64_t ctx = a.context_lens[b];
    const int total = aw_total(a, ctx);
    const int chunks = (total + kAwVecChunk - 1) / kAwVecChunk;
    const int2 live = aw_chunks(a, b, ctx, total);
    const int  first = live.x <= split ? split : split + (live.x - split + splits - 1) / splits * splits;
    const int r_lo = SUM ? 0 : static_cast<int>(blockIdx.y) * kAwVecRows;
    const int r_hi = SUM ? R : min(R, r_lo + kAwVecRows);
    if constexpr (!SUM)
        for (int i = lane; i < kAwVecRows; i += 64) s_ml[wave][i] = make_float2(kLowest, 0.0f);
    for (int ch = SUM ? split : first; ch < (SUM ? chunks : live.y); ch += splits)
    {
        const int key = ch * kAwVecChunk + tid;
        if (SUM && (ch < live.x || ch >= live.y))
        {
            aw_store(a, bh, ctx, total, key, 0.0f);
            continue;
        }
        int       phys = -1;
        if (key < total) phys = a.block_table[static_cast<int64_t>(b) * a.max_blocks + (key >> 4)];
        const bool   ok = phys >= 0 && phys < a.num_blocks;
        const size_t row = (static_cast<size_t>(ok ? phys : 0) * kBlockSize + (key & 15)) * a.num_kv_heads + kvh;
        float        sk = a.scale_log2;
        if constexpr (CT == I8) sk *= ok ? a.k_scale[row] : 0.0f;
        if constexpr (CT == FP8) sk *= a.k_scale[kvh];
        float w = 0.0f;
        for (int r0 = r_lo; r0 < r_hi; r0 += T)
        {
            const int m = min(T, r_hi - r0);
            __syncthreads();  // the last rows are done with
            for (int i = tid; i < T * (D / 4); i += kAwVecThreads)
            {
                const int rr = i / (D / 4), d = 4 * (i - rr * (D / 4));
                float     x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                if (rr < m)
                {
                    const int t = (r0 + rr) / G, h = r0 + rr - t * G;
                    load_act4(a.q, a.qo_dtype,
                              ((static_cast<size_t>(b) * a.seq_len + t) * a.num_heads + kvh * G + h) * D + d, x);
                }
                *reinterpret_cast<float4*>(&s_q[rr][d]) = make_float4(x[0], x[1], x[2], x[3]);
            }
            if (tid < T)
            {
                const int r = r0 + tid;
                s_vis[tid] = tid < m ? aw_visible(a, b, ctx, total, r / G) : make_int3(0, 0, 0);
                s_slope[tid] = tid < m && a.rule.slopes != nullptr ? a.rule.slopes[kvh * G + r % G] * 1.4426950408889634f : 0.0f;
                if constexpr (SUM) s_ml[0][tid] = tid < m ? a.fin[static_cast<int64_t>(bh) * R + r] : make_float2(0.0f, 0.0f);
            }
            __syncthreads();
            float s[T];
#pragma unroll
            for (int rr = 0; rr < T; ++rr) s[rr] = 0.0f;
            for (int d = 0; d < D; d += 8)
            {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = 0.0f;
                if (ok)
                {
                    Raw8 raw;
                    load_raw8<CT>(a.k_cache, row * D + d, raw);
                    unpack8<CT>(raw, x);
                }
#pragma unroll
                for (int rr = 0; rr < T; ++rr)
#pragma unroll
                    for (int e = 0; e < 8; ++e) s[rr] = __builtin_fmaf(s_q[rr][d + e], x[e], s[rr]);
            }
#pragma unroll
            for (int rr = 0; rr < T; ++rr)
            {
                const int3 vis = s_vis[rr];
                float      v = s[rr] * sk;
                if (a.rule.cap > 0.0f) v = cap_score(v * a.rule.inv_cap, a.rule.cap);
                if (a.rule.slopes != nullptr)
                    v = __builtin_fmaf(-s_slope[rr], __builtin_fabsf(static_cast<float>(key - vis.z)), v);
                v = ok && key >= vis.x && key < vis.y ? v : kNegInf;
                if constexpr (SUM)
                {
                    const float2 f = s_ml[0][rr];
                    w += v == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(v - f.x) * f.y;
                }
                else if (rr < m)  // uniform
                {
                    float mx = group_max<32>(__builtin_elementwise_maximum(v, kLowest));
                    mx = __builtin_elementwise_maximum(mx, __shfl_xor(mx, 32, 64));
                    float l = group_sum<32>(__builtin_amdgcn_exp2f(v - mx));
                    l += __shfl_xor(l, 32, 64);
                    if (lane == 0)
                    {
                        float2& st = s_ml[wave][r0 - r_lo + rr];
                        st = aw_join(st, make_float2(mx, l));
                    }
                }
            }
        }
        if constexpr (SUM) aw_store(a, bh, ctx, total, key, w);
    }
    if constexpr (!SUM)
    {
        __syncthreads();
        for (int r = r_lo + tid; r < r_hi; r += kAwVecThreads)
        {
            float2 st = s_ml[0][r - r_lo];
#pragma unroll
            for (int v = 1; v < kAwVecWaves; ++v) st = aw_join(st, s_ml[v][r - r_lo]);
            a.part[share.slot * R + r] = st;
        }
    }
}

// The rows' states over all splits as (max, 1 / denominator): 16 rows a workgroup, 16 threads over the splits of each.
__global__ __launch_bounds__(256) void attention_weights_fold(WeightArgs a)
{
    __shared__ float2 s_st[16][17];
    const int     R = a.seq_len * a.group;
    const int     i = static_cast<int>(threadIdx.x) & 15;
    const int     sl = static_cast<int>(threadIdx.x) >> 4;
    const int     blocks = (R + 15) / 16;
    const int64_t bh = static_cast<int64_t>(blockIdx.x) / blocks;
    const int     r = static_cast<int>(blockIdx.x % blocks) * 16 + i;
    const int     b = static_cast<int>(bh / a.num_kv_heads);
    const AwShare share = aw_share(a, -1, b);
    const int64_t slot = share.slot + (bh - static_cast<int64_t>(b) * a.num_kv_heads) * share.splits;
    float2        st = make_float2(kLowest, 0.0f);
    if (r < R)
        for (int s = sl; s < share.splits; s += 16) st = aw_join(st, a.part[(slot + s) * R + r]);
    s_st[sl][i] = st;
    __syncthreads();
    if (sl != 0 || r >= R) return;
    for (int k = 1; k < 16; ++k) st = aw_join(st, s_st[k][i]);
    a.fin[bh * R + r] = make_float2(st.x, softmax_inv(st.y));
}

namespace
{

// f.operator()<CT, QT, D>() for the call's types and head_dim.
template <typename F>
auto weights_for(const WeightArgs& a, F f)
{
    auto d = [&]<int CT, int QT>()
    {
        switch (a.head_dim)
        {
            case 64:
                return f.template operator()<CT, QT, 64>();
            case 80:
                return f.template operator()<CT, QT, 80>();
            case 96:
                return f.template operator()<CT, QT, 96>();
            case 112:
                return f.template operator()<CT, QT, 112>();
            case 128:
                return f.template operator()<CT, QT, 128>();
            default:
                return f.template operator()<CT, QT, 256>();
        }
    };
    auto q = [&]<int CT>()
    {
        if (a.qo_dtype == F32) return d.template operator()<CT, F32>();
        if (a.qo_dtype == F16) return d.template operator()<CT, F16>();
        return d.template operator()<CT, BF16>();
    };
    if (a.cache_dtype == BF16) return q.template operator()<BF16>();
    if (a.cache_dtype == F16) return q.template operator()<F16>();
    if (a.cache_dtype == I8) return q.template operator()<I8>();
    return q.template operator()<FP8>();
}

template <int CT>
hipError_t launch_vector(const WeightArgs& a, bool sum, dim3 grid, hipStream_t stream)
{
    if (sum)
        hipLaunchKernelGGL((attention_weights_vector<CT, true>), grid, dim3(kAwVecThreads), 0, stream, a);
    else
        hipLaunchKernelGGL((attention_weights_vector<CT, false>), grid, dim3(kAwVecThreads), 0, stream, a);
    return hipGetLastError();
}

}  // namespace

// Splits of a row's keys, on average over the rows (aw_share): as many workgroups in all as fit the chip at once (two of eight
// waves per CU), one chunk of keys each at most; a workgroup then stages its query rows once for several chunks.  us at 512 /
// 768 / 1024 workgroups: 32 tokens over one row of 32.7k 47 / 52 / 57, 16 x 64 tokens over int8 rows of 400 to 4000
// 146 / 157 / 160 (with rows cut alike, 256 took 65 and 244 where 512 took 51 and 187).
int attention_weights_splits(int batch, int num_kv_heads, int head_dim, int cap_tokens)
{
    const int64_t chunk = kAwChunk;
    const int64_t chunks = (static_cast<int64_t>(cap_tokens) + chunk - 1) / chunk;
    const int64_t most = kAwMost / (static_cast<int64_t>(batch) * num_kv_heads);
    const int64_t n = chunks < most ? chunks : most;
    return static_cast<int>(n < 1 ? 1 : n);
}

hipError_t launch_attention_weights(const WeightArgs& a, bool mfma, hipStream_t stream)
{
    const int64_t R = static_cast<int64_t>(a.seq_len) * a.group;
    const int64_t bh = static_cast<int64_t>(a.batch) * a.num_kv_heads;
    if (bh * a.splits > INT32_MAX || bh * ((R + 15) / 16) > INT32_MAX) return hipErrorInvalidConfiguration;
    auto pass = [&](bool sum) -> hipError_t
    {
        auto grid = [&](int rows)
        { return dim3(static_cast<unsigned>(bh * a.splits), sum ? 1u : static_cast<unsigned>((R + rows - 1) / rows)); };
        if (mfma)
            return weights_for(a, [&]<int CT, int QT, int D>()
            {
                constexpr bool LO = kAwLo<CT, QT>;
                // as many query rows as the call has, up to kAwRows: the less LDS, the more workgroups per CU
                WeightArgs w = a;
                w.block_rows = weight_block_rows(R, kAwRows<D, LO>);
                const int  lds = aw_lds<D, LO>(w.block_rows, sum);
                const dim3 n = grid(w.block_rows);
                if (n.y > 65535u) return hipErrorInvalidConfiguration;
                if (sum)
                    hipLaunchKernelGGL((attention_weights_mfma<CT, QT, D, true>), n, dim3(kAwThreads), lds, stream, w);
                else
                    hipLaunchKernelGGL((attention_weights_mfma<CT, QT, D, false>), n, dim3(kAwThreads), lds, stream, w);
                return hipGetLastError();
            });
        const dim3 n = grid(kAwVecRows);
        if (n.y > 65535u) return hipErrorInvalidConfiguration;
        if (a.cache_dtype == F32) return launch_vector<F32>(a, sum, n, stream);
        if (a.cache_dtype == F16) return launch_vector<F16>(a, sum, n, stream);
        if (a.cache_dtype == BF16) return launch_vector<BF16>(a, sum, n, stream);
        if (a.cache_dtype == I8) return launch_vector<I8>(a, sum, n, stream);
        return launch_vector<FP8>(a, sum, n, stream);
    };
    if (R == 0) return pass(true);  // no queries: the earlier weights' decay alone
    hipError_t e = pass(false);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(attention_weights_fold, dim3(static_cast<unsigned>(bh * ((R + 15) / 16))), dim3(256), 0, stream, a);
    e = hipGetLastError();
    return e != hipSuccess ? e : pass(true);
}

}  // namespace ffkv
