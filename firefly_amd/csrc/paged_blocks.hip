// paged_blocks.hip - attention over listed pages of the cache alone: every query token and KV head has a list of its row's
// pages (logical ones, in any order; entries that are none, or past the query, count for nothing).
//
//   out[b, t, h] = sum over listed pages and their tokens j <= context_lens[b] + t of softmax_j(scale q.k_j) v_j
//
// Steps are bound by HBM: the listed pages are read once, at about Hq / Hkv operations a byte.  64 rows of 64 listed pages, 32/8
// heads of 128, bf16: 270 MB in 49.4 us = 5.5 TB/s (inputs resident: int8 30.3, fp32 98); 4 rows of 256, 28/4 heads, f16: 14.3 us,
// of which 3.5 of merge; 4 rows of up to 16: 7.3, a launch and its chain of loads.
//
// On the matrix cores (16- and 8-bit caches) a workgroup of four or eight waves takes a list, or a piece of one, and up to 16
// query heads of its KV head; a wave takes every fourth (eighth) page, with the products and the page loads of the plain decode
// (paged_decode_mfma.hip): S^T = K Q^T with K from its registers, an online softmax, O^T += V^T P^T with V^T read transposed
// from LDS.  Lane l holds the wave's entry 64 k + l and its page, so a page's address waits for no load.  The waves' states
// meet in LDS; pieces of a list go to the workspace and blocks_merge folds them.
//
// Blocks of tokens that share their lists take the prefill's kernel (blocks_prefill.h), whose tiles of 128 query rows read a
// list once; bound by its vector work beside the products (2 x 512 tokens in blocks of 64, 128 listed fp8 pages, 32/8 heads of
// 128: 34.4 GFLOP in 53.5 us = 640 TFLOP/s).
//
// fp32 caches and the other head dims take the vector kernel: 16 (head_dim 256: 32) lanes per token, four query heads a
// workgroup.
#define FFKV_DEVICE_BODIES_ONLY 1
#include "paged_decode_mfma.hip"
#undef FFKV_DEVICE_BODIES_ONLY
#include "blocks.h"

#include <algorithm>

namespace ffkv
{

namespace
{

constexpr int kBlocksWaves = 4;  // of the vector kernel

// LDS of a workgroup of `waves` waves and up to `heads` query heads: the waves' V tiles, and over them their accumulators and
// (max, denominator) pairs once all pages are done.
template <int D>
constexpr int blocks_lds_bytes(int waves, int heads)
{
    const int v = waves * kBlockSize * D * 2;
    const int state = waves * heads * D * 4 + waves * 16 * 8;
    return v > state ? v : state;
}
static_assert(blocks_lds_bytes<256>(8, 16) <= 160 * 1024, "a workgroup's LDS fits a CU");

// One page in flight.
template <int NW, int NWV>
struct ListedPage
{
    u32x4 k[NW];
    u32x4 v[NWV];
    int   n_tok;  // its visible tokens; 0: none of it
    float ks, vs; // int8: K and V scale of token c
};

// Entry e of a list: the logical page, or -1 where it is none of the table's.  (Whether the query sees it is looked at later:
// the page's entry in the table need not wait for the row's length.)
__device__ __forceinline__ int listed_page(const BlocksArgs& a, const int32_t* list, int e, int end)
{
    const int lp = e < end ? list[e] : -1;
    return lp >= 0 && lp < a.max_blocks ? lp : -1;
}

// Tokens of logical page lp on physical page phys that the query at pos sees; 0 where it is no page, or past the query.
__device__ __forceinline__ int listed_tokens(const BlocksArgs& a, int lp, int phys, int64_t pos)
{
    const int64_t n = pos + 1 - static_cast<int64_t>(lp) * kBlockSize;
    return phys < 0 || phys >= a.num_blocks || n <= 0 ? 0 : n < kBlockSize ? static_cast<int>(n) : kBlockSize;
}

// A state of (max, denominator, accumulator) to the output, or to its piece's place in the workspace.
template <int QT>
__device__ __forceinline__ void store_state4(const BlocksArgs& a, int64_t row_h, int split, int D, int d4, float M, float L,
                                             f32x4 o)
{
    if (a.splits == 1)
    {
        store_out4<QT>(a.out, static_cast<size_t>(row_h) * D + d4, o * softmax_inv(L));
        return;
    }
    *reinterpret_cast<f32x4*>(a.ws_acc + (row_h * a.splits + split) * D + d4) = o;
    if (d4 == 0) a.ws_ml[row_h * a.splits + split] = float2{M, L};
}

}  // namespace

template <int CT, int QT, int D, int WAVES>
__global__ __launch_bounds__(64 * WAVES) __attribute__((amdgpu_waves_per_eu(2, 8)))
void paged_blocks_decode(BlocksArgs a)
{
    extern __shared__ __align__(16) uint8_t s_blocks[];
    constexpr bool BF = kBF<CT, QT>;
    constexpr bool VBF = CT == BF16 || (kElemBytes<CT> == 1 && BF && !FFKV_DECODE_V16);
    using M = MType<BF>;
    using MV = MType<VBF>;
    using X8 = typename M::x8;
    static_assert(D % 16 == 0, "whole output tiles of 16 dims");
    constexpr int  KSTEPS = (D + 31) / 32;  // of 32 dims; head_dim 80 and 112 leave lanes of the last without any
    constexpr int  NT = D / 16;
    constexpr bool NEED_LO = !((QT == BF16 && BF) || (QT == F16 && !BF));
    constexpr bool P_LO = VBF || CT == F16;
    constexpr int  DEPTH = D == 256 ? 1 : 2;
    constexpr int  EB = kElemBytes<CT>;
    constexpr int  NW = EB == 2 ? KSTEPS : (KSTEPS + 1) / 2;
    constexpr int  VCPR = D * EB / 16;
    constexpr int  NWV = (kBlockSize * VCPR + 63) / 64;
    auto dimof = [](int j, int g)
    {
        if constexpr (EB == 1 && KSTEPS % 2 == 1)
            if (j == KSTEPS - 1) return 32 * j + 8 * g;
        return dim_of<CT>(j, g);
    };
    auto has = [&](int j, int g) { return D % 32 == 0 || dimof(j, g) < D; };
    const int lane = static_cast<int>(threadIdx.x) & 63;
    const int wave = uniform(static_cast<int>(threadIdx.x) >> 6);
    const int c = lane & 15;
    const int g = lane >> 4;
    const int G = a.group;
    const int HB = (G + 15) >> 4;
    const Split u = split_index(blockIdx.x, a.splits), v = split_index(u.div, a.num_kv_heads * HB);
    const Split w = split_index(v.div, a.seq_len);
    const int     split = u.rem, vh = v.rem, b = static_cast<int>(w.div), t = w.rem;
    const int64_t row = v.div;  // b * seq_len + t
    const int64_t rl = a.query_block == 1 ? row : static_cast<int64_t>(b) * a.lists + t / a.query_block;
    const int     kvh = vh / HB;
    const int     h0 = (vh - kvh * HB) * 16;
    const int     gc = min(16, G - h0);
    const int64_t pos = static_cast<int64_t>(a.context_lens[b]) + t;
    const int32_t* list = a.blocks + (rl * a.num_kv_heads + kvh) * a.count;
    const int32_t* table = a.block_table + static_cast<int64_t>(b) * a.max_blocks;
    // this wave's entries: begin + WAVES i, i < n
    const int begin = static_cast<int>(static_cast<int64_t>(a.count) * split / a.splits) + wave;
    const int end = static_cast<int>(static_cast<int64_t>(a.count) * (split + 1) / a.splits);
    const int n = end > begin ? (end - begin + WAVES - 1) / WAVES : 0;
    uint16_t* sv = reinterpret_cast<uint16_t*>(s_blocks) + wave * (kBlockSize * D);

    float kv_scale_log2 = a.scale_log2;
    float v_head_scale = 1.0f;
    if constexpr (CT == FP8)
    {
        kv_scale_log2 *= a.k_scale[kvh];
        v_head_scale = a.v_scale[kvh];
    }

    const int v_row_bytes = a.num_kv_heads * D * EB;
    auto      v_tok = [&](int j) { return (64 * j + lane) / VCPR; };
    auto      v_chk = [&](int j) { return (64 * j + lane) % VCPR; };

    int  tb = 0, lvec, pvec;  // lane l: logical and physical page of entry tb + l
    auto load_entries = [&]()
    {
        lvec = listed_page(a, list, begin + WAVES * (tb + lane), end);
        pvec = lvec >= 0 ? table[lvec] : -1;
    };
    load_entries();
    int  next = 0;
    auto load_next = [&](ListedPage<NW, NWV>& r)
    {
        if (next - tb >= 64)
        {
            tb += 64;
            load_entries();
        }
        const int lp = __builtin_amdgcn_readlane(lvec, next - tb);
        const int phys = __builtin_amdgcn_readlane(pvec, next - tb);
        ++next;
        r.n_tok = listed_tokens(a, lp, phys, pos);
        if (r.n_tok == 0) return;
        const size_t row_c = (static_cast<size_t>(phys) * kBlockSize + c) * a.num_kv_heads + kvh;
        if constexpr (CT == I8)
        {
            r.ks = a.k_scale[row_c];
            r.vs = a.v_scale[row_c];
        }
        const char* kp = static_cast<const char*>(a.k_cache) + row_c * D * EB;
        const char* vpage = static_cast<const char*>(a.v_cache) +
                            (static_cast<size_t>(phys) * kBlockSize * a.num_kv_heads + kvh) * D * EB;
        if constexpr (EB == 2)
        {
#pragma unroll
            for (int j = 0; j < KSTEPS; ++j)
            {
                r.k[j] = u32x4{0u, 0u, 0u, 0u};
                if (has(j, g)) r.k[j] = *reinterpret_cast<const u32x4*>(kp + dim_of<CT>(j, g) * 2);
            }
        }
        else
        {
#pragma unroll
            for (int j = 0; j < KSTEPS; j += 2)
            {
                r.k[j / 2] = u32x4{0u, 0u, 0u, 0u};
                if (!has(j, g)) continue;
                if (j + 1 < KSTEPS)
                    r.k[j / 2] = *reinterpret_cast<const u32x4*>(kp + dimof(j, g));
                else  // an odd last k-step: its 8 codes alone
                {
                    const u32x2 tk = *reinterpret_cast<const u32x2*>(kp + dimof(j, g));
                    r.k[j / 2] = u32x4{tk[0], tk[1], 0u, 0u};
                }
            }
        }
#pragma unroll
        for (int j = 0; j < NWV; ++j)
            r.v[j] = v_tok(j) < kBlockSize
                         ? load16<FFKV_DECODE_NT_V>(vpage + static_cast<uint32_t>(v_tok(j) * v_row_bytes + 16 * v_chk(j)))
                         : u32x4{0u, 0u, 0u, 0u};
    };

    // Q of the head block as MFMA B operands (column c = head, zero beyond it)
    X8 qhi[KSTEPS], qlo[KSTEPS];
#pragma unroll
    for (int j = 0; j < KSTEPS; ++j)
    {
        const size_t at = (static_cast<size_t>(row) * a.num_heads + kvh * G + h0 + c) * D + dimof(j, g);
        if constexpr (!NEED_LO)
        {
            u32x4 w = u32x4{0u, 0u, 0u, 0u};
            if (c < gc && has(j, g)) w = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.q) + at);
            qhi[j] = qlo[j] = __builtin_bit_cast(X8, w);
        }
        else
        {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = 0.0f;
            if (c < gc && has(j, g)) load_q8<QT>(a.q, at, x);
            uint32_t hi[8], lo[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
            {
                hi[e] = M::bits(x[e]);
                lo[e] = M::bits(x[e] - M::value(hi[e]));
            }
            qhi[j] = __builtin_bit_cast(X8, u32x4{hi[0] | (hi[1] << 16), hi[2] | (hi[3] << 16), hi[4] | (hi[5] << 16),
                                                  hi[6] | (hi[7] << 16)});
            qlo[j] = __builtin_bit_cast(X8, u32x4{lo[0] | (lo[1] << 16), lo[2] | (lo[3] << 16), lo[4] | (lo[5] << 16),
                                                  lo[6] | (lo[7] << 16)});
        }
    }

    float m_run = kLowest, l_run = 0.0f;
    f32x4 acc[NT];
    ValueUnits units;  // int8
#pragma unroll
    for (int i = 0; i < NT; ++i) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    // V rows into the wave's LDS tile (zero past the visible tokens) and the scores S^T = K Q^T; consumes r.k and r.v
    auto stage_page = [&](const ListedPage<NW, NWV>& r, f32x4& s)
    {
#pragma unroll
        for (int j = 0; j < NWV; ++j)
        {
            const int t = v_tok(j);
            if (t >= kBlockSize) continue;
            const bool  ok = t < r.n_tok;
            const u32x4 zero = u32x4{0u, 0u, 0u, 0u};
            if constexpr (EB == 2)
                *reinterpret_cast<u32x4*>(sv + vt_pos<D>(t, 8 * v_chk(j))) = ok ? r.v[j] : zero;
            else
            {
                *reinterpret_cast<u32x4*>(sv + vt_pos<D>(t, 16 * v_chk(j))) =
                    ok ? codes_to_m<CT, VBF>(r.v[j][0], r.v[j][1]) : zero;
                *reinterpret_cast<u32x4*>(sv + vt_pos<D>(t, 16 * v_chk(j) + 8)) =
                    ok ? codes_to_m<CT, VBF>(r.v[j][2], r.v[j][3]) : zero;
            }
        }
        s = f32x4{0.0f, 0.0f, 0.0f, 0.0f};  // lane (c, g): tokens 4g + i of head c
#pragma unroll
        for (int j = 0; j < KSTEPS; ++j)
        {
            u32x4 w;
            if constexpr (EB == 2)
                w = r.k[j];
            else
                w = (j & 1) ? codes_to_m<CT, BF>(r.k[j / 2][2], r.k[j / 2][3]) : codes_to_m<CT, BF>(r.k[j / 2][0], r.k[j / 2][1]);
            const X8 kj = __builtin_bit_cast(X8, w);
            s = M::mma32(kj, qhi[j], s);
            if constexpr (NEED_LO) s = M::mma32(kj, qlo[j], s);
        }
    };

    // Online softmax of a staged page and its products with V.  P takes a hi + lo pair of 16-bit values (16 bits in bf16, 21 in
    // f16: 64 rows of f16 pages 44.0 -> 44.3 us), on 8-bit pages f16's 11 bits: the codes' own steps are larger (with a pair int8
    // took 30.3 -> 32.1 us, fp8 25.5 -> 25.8).  int8 pages: in units of the column, as the V scales are in it.
    auto finish_page = [&](int n_tok, float tks, float tvs, f32x4 s)
    {
        float sc[4], vs[4];
        float mt = kNegInf;
#pragma unroll
        for (int i = 0; i < 4; ++i)
        {
            float x = s[i] * kv_scale_log2;
            vs[i] = 1.0f;
            if constexpr (CT == I8)  // token 4g + i's scales sit in lane 4g + i
            {
                x = s[i] * __shfl(tks, 4 * g + i, 64) * kv_scale_log2;
                vs[i] = __shfl(tvs, 4 * g + i, 64);
            }
            sc[i] = 4 * g + i < n_tok ? x : kNegInf;
            mt = fmaxf(mt, sc[i]);
        }
        mt = xor_max(mt);
        const float m_new = fmaxf(m_run, mt);
        const float alpha = __builtin_amdgcn_exp2f(m_run - m_new);
        float       pv[4], psum = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
        {
            const float p = __builtin_amdgcn_exp2f(CT == I8 ? sc[i] - m_new + units.shift : sc[i] - m_new);
            psum += p;
            pv[i] = 4 * g + i < n_tok ? p * vs[i] : 0.0f;
        }
        l_run = l_run * alpha + psum;
        if (__any(m_new > m_run))
        {
#pragma unroll
            for (int i = 0; i < NT; ++i) acc[i] *= alpha;
            units.known *= alpha;
        }
        m_run = m_new;
        if constexpr (CT == I8)
        {
            float w = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) w = fmaxf(w, __builtin_fabsf(pv[i]));
            if (__any(w > units.limit()))
            {
                const float f = new_units(units, xor_max(w));
                l_run *= f;
#pragma unroll
                for (int i = 0; i < 4; ++i) pv[i] *= f;
#pragma unroll
                for (int i = 0; i < NT; ++i) acc[i] *= f;
            }
        }
        uint32_t ph[4], pl[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
        {
            ph[i] = MV::bits(pv[i]);
            pl[i] = P_LO ? MV::bits(pv[i] - MV::value(ph[i])) : 0u;
        }
        const auto phi = __builtin_bit_cast(typename MV::x4, u32x2{ph[0] | (ph[1] << 16), ph[2] | (ph[3] << 16)});
        const auto plo = __builtin_bit_cast(typename MV::x4, u32x2{pl[0] | (pl[1] << 16), pl[2] | (pl[3] << 16)});
        // the wave's LDS writes are complete before its reads (one queue); the fence keeps the compiler to that order
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
        for (int i = 0; i < NT; ++i)
        {
            const auto raw = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
                (__attribute__((address_space(3))) bf16x4*)(sv + vt_pos<D>(4 * g + (c >> 2), 16 * i + 4 * (c & 3))));
            const auto vt = __builtin_bit_cast(typename MV::x4, raw);
            acc[i] = MV::mma16(vt, phi, acc[i]);
            if constexpr (P_LO) acc[i] = MV::mma16(vt, plo, acc[i]);
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    };

    // entry i sits in r[i % DEPTH]; right after it is staged, entry i + DEPTH is loaded into the same registers
    ListedPage<NW, NWV> r[DEPTH];
#pragma unroll
    for (int sl = 0; sl < DEPTH; ++sl)
        if (sl < n) load_next(r[sl]);
    auto step = [&]<int S>(int i)
    {
        ListedPage<NW, NWV>& cur = r[S];
        const int   n_tok = cur.n_tok;
        const float tks = cur.ks, tvs = cur.vs;
        f32x4       s;
        if (n_tok > 0) stage_page(cur, s);
        if (i + DEPTH < n) load_next(cur);
        if (n_tok > 0) finish_page(n_tok, tks, tvs, s);
    };
    for (int i = 0; i < n; i += DEPTH)
    {
        step.template operator()<0>(i);
        if constexpr (DEPTH > 1)
            if (i + 1 < n) step.template operator()<1 % DEPTH>(i + 1);
    }

    // the waves' states: accumulators [wave][head][D] over the V tiles, then (max, denominator) [wave][16]
    float*      s_acc = reinterpret_cast<float*>(s_blocks);
    float2*     s_ml = reinterpret_cast<float2*>(s_acc + WAVES * gc * D);
    const float l_tot = xor_sum(l_run);
    __syncthreads();
    if (c < gc)
    {
        const float piece_scale = seen_scale<CT>(l_tot, v_head_scale);
#pragma unroll
        for (int i = 0; i < NT; ++i)
            *reinterpret_cast<f32x4*>(s_acc + (wave * gc + c) * D + 16 * i + 4 * g) = acc[i] * piece_scale;
        if (g == 0) s_ml[wave * 16 + c] = float2{m_run - units.shift, l_tot};
    }
    __syncthreads();
    for (int k = static_cast<int>(threadIdx.x); k < gc * (D / 4); k += 64 * WAVES)
    {
        const int h = k / (D / 4);
        const int d4 = (k - h * (D / 4)) * 4;
        float     Mx = kLowest, L = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) Mx = fmaxf(Mx, s_ml[w * 16 + h].x);
        f32x4 o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < WAVES; ++w)
        {
            const float2 t = s_ml[w * 16 + h];
            const float  x = __builtin_amdgcn_exp2f(t.x - Mx);
            L += t.y * x;
            o += *reinterpret_cast<const f32x4*>(s_acc + (w * gc + h) * D + d4) * x;
        }
        store_state4<QT>(a, row * a.num_heads + kvh * G + h0 + h, split, D, d4, Mx, L, o);
    }
}

// The pieces of every (row, head), folded.  A thread takes four output dims and every SG-th piece.
template <int QT>
__global__ __launch_bounds__(256) void blocks_merge(BlocksArgs a)
{
    __shared__ f32x4  s_o[256];
    __shared__ float2 s_ml[256];
    const int     D = a.head_dim, DL = D / 4;  // lanes of a piece
    const int     SG = 256 / DL;
    const int     tid = static_cast<int>(threadIdx.x);
    const int     sg = tid / DL, d4 = (tid - sg * DL) * 4;
    const int64_t row_h = blockIdx.x;
    const float2* ml = a.ws_ml + row_h * a.splits;
    const float*  xs = a.ws_acc + row_h * a.splits * D + d4;
    float         m = kLowest, l = 0.0f;
    f32x4         o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if (sg < SG)
    {
        constexpr int MF = 4;  // pieces whose loads go out together
        for (int i0 = sg; i0 < a.splits; i0 += SG * MF)
        {
            float2 t[MF];
            f32x4  x[MF];
            float  mn = m;
#pragma unroll
            for (int f = 0; f < MF; ++f)
            {
                const int i = i0 + f * SG;
                t[f] = float2{kLowest, 0.0f};
                x[f] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                if (i < a.splits)
                {
                    t[f] = ml[i];
                    x[f] = *reinterpret_cast<const f32x4*>(xs + static_cast<int64_t>(i) * D);
                }
            }
#pragma unroll
            for (int f = 0; f < MF; ++f) mn = fmaxf(mn, t[f].x);
            const float wa = __builtin_amdgcn_exp2f(m - mn);
            l *= wa;
            o *= wa;
#pragma unroll
            for (int f = 0; f < MF; ++f)
            {
                const float w = __builtin_amdgcn_exp2f(t[f].x - mn);
                l += t[f].y * w;
                o += x[f] * w;
            }
            m = mn;
        }
    }
    s_o[tid] = o;
    s_ml[tid] = float2{m, l};
    __syncthreads();
    if (sg != 0) return;
    for (int j = 1; j < SG; ++j)
    {
        const float2 t = s_ml[j * DL + tid];
        const float  mn = fmaxf(m, t.x);
        const float  wa = __builtin_amdgcn_exp2f(m - mn), w = __builtin_amdgcn_exp2f(t.x - mn);
        l = l * wa + t.y * w;
        o = o * wa + s_o[j * DL + tid] * w;
        m = mn;
    }
    store_out4<QT>(a.out, static_cast<size_t>(row_h) * D + d4, o * softmax_inv(l));
}

// The vector kernel: a workgroup takes four query heads of a (row, KV head) and a piece of its list, a wave every fourth
// page; LPT lanes hold a token, 8 dims each, with a softmax state per group of lanes.
template <int CT, int QT, int LPT>
__global__ __launch_bounds__(64 * kBlocksWaves) void paged_blocks_vector(BlocksArgs a)
{
    constexpr int HC = 4;
    constexpr int TPW = 64 / LPT;           // tokens of a wave at a time
    constexpr int NTOK = kBlockSize / TPW;  // of a page per group of lanes
    constexpr int UN = 4;                   // tokens whose loads go out together
    constexpr int ST = kBlocksWaves * TPW;  // states of the workgroup
    __shared__ __align__(16) float s_acc[ST][HC][LPT * 8];
    __shared__ float2 s_ml[ST][HC];
    const int lane = static_cast<int>(threadIdx.x) & 63;
    const int wave = uniform(static_cast<int>(threadIdx.x) >> 6);
    const int c = lane % LPT;
    const int g = lane / LPT;
    const int D = a.head_dim;
    const bool in = 8 * c < D;
    const int G = a.group;
    const int HB = (G + HC - 1) / HC;
    const Split u = split_index(blockIdx.x, a.splits), v = split_index(u.div, a.num_kv_heads * HB);
    const Split w = split_index(v.div, a.seq_len);
    const int     split = u.rem, vh = v.rem, b = static_cast<int>(w.div), t = w.rem;
    const int64_t row = v.div;  // b * seq_len + t
    const int     kvh = vh / HB;
    const int     h0 = (vh - kvh * HB) * HC;
    const int     gc = min(HC, G - h0);
    const int64_t pos = static_cast<int64_t>(a.context_lens[b]) + t;
    const int32_t* list = a.blocks + ((static_cast<int64_t>(b) * a.lists + t / a.query_block) * a.num_kv_heads + kvh) * a.count;
    const int32_t* table = a.block_table + static_cast<int64_t>(b) * a.max_blocks;
    const int begin = static_cast<int>(static_cast<int64_t>(a.count) * split / a.splits) + wave;
    const int end = static_cast<int>(static_cast<int64_t>(a.count) * (split + 1) / a.splits);

    float q[HC][8], acc[HC][8], m[HC], l[HC];
#pragma unroll
    for (int h = 0; h < HC; ++h)
    {
        m[h] = kLowest;
        l[h] = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) q[h][e] = acc[h][e] = 0.0f;
        if (h < gc && in)
            load_q8<QT>(a.q, (static_cast<size_t>(row) * a.num_heads + kvh * G + h0 + h) * D + 8 * c, q[h]);
#pragma unroll
        for (int e = 0; e < 8; ++e) q[h][e] *= a.scale_log2;
    }
    float k_head = 1.0f, v_head = 1.0f;
    if constexpr (CT == FP8)
    {
        k_head = a.k_scale[kvh];
        v_head = a.v_scale[kvh];
    }
    for (int i0 = begin; i0 < end; i0 += 64 * kBlocksWaves)
    {
        const int lvec = listed_page(a, list, i0 + kBlocksWaves * lane, end);
        const int pvec = lvec >= 0 ? table[lvec] : -1;
        for (int i = 0; i < 64 && i0 + kBlocksWaves * i < end; ++i)
        {
            const int lp = __builtin_amdgcn_readlane(lvec, i);
            const int phys = __builtin_amdgcn_readlane(pvec, i);
            const int n_tok = listed_tokens(a, lp, phys, pos);
            if (n_tok == 0) continue;
#pragma unroll 1
            for (int u0 = 0; u0 < NTOK; u0 += UN)
            {
                Raw8  kr[UN], vr[UN];
                float ks[UN], vs[UN];
#pragma unroll
                for (int u = 0; u < UN; ++u)
                {
                    const int    tok = (u0 + u) * TPW + g;
                    const size_t row_c = (static_cast<size_t>(phys) * kBlockSize + tok) * a.num_kv_heads + kvh;
                    ks[u] = k_head;
                    vs[u] = v_head;
                    if constexpr (CT == I8)
                    {
                        ks[u] = a.k_scale[row_c];
                        vs[u] = a.v_scale[row_c];
                    }
                    if (in)
                    {
                        load_raw8<CT>(a.k_cache, row_c * D + 8 * c, kr[u]);
                        load_raw8<CT>(a.v_cache, row_c * D + 8 * c, vr[u]);
                    }
                }
#pragma unroll
                for (int u = 0; u < UN; ++u)
                {
                    const bool seen = (u0 + u) * TPW + g < n_tok;
                    float      k[8], v[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) k[e] = v[e] = 0.0f;
                    if (in && seen)
                    {
                        unpack8<CT>(kr[u], k);
                        unpack8<CT>(vr[u], v);
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (CT == I8 || CT == FP8) v[e] = seen ? v[e] * vs[u] : 0.0f;
#pragma unroll
                    for (int h = 0; h < HC; ++h)
                    {
                        float s = 0.0f;
#pragma unroll
                        for (int e = 0; e < 8; ++e) s = __builtin_fmaf(q[h][e], k[e], s);
                        s = group_sum<LPT>(s);
                        if (CT == I8 || CT == FP8) s *= ks[u];
                        s = seen ? s : kNegInf;
                        const float mn = fmaxf(m[h], s);
                        const float wa = __builtin_amdgcn_exp2f(m[h] - mn);
                        const float p = __builtin_amdgcn_exp2f(s - mn);
                        l[h] = l[h] * wa + p;
#pragma unroll
                        for (int e = 0; e < 8; ++e) acc[h][e] = __builtin_fmaf(p, v[e], acc[h][e] * wa);
                        m[h] = mn;
                    }
                }
            }
        }
    }
    const int st = wave * TPW + g;
#pragma unroll
    for (int h = 0; h < HC; ++h)
    {
#pragma unroll
        for (int e = 0; e < 8; ++e) s_acc[st][h][8 * c + e] = acc[h][e];
        if (c == 0) s_ml[st][h] = float2{m[h], l[h]};
    }
    __syncthreads();
    for (int k = static_cast<int>(threadIdx.x); k < gc * (D / 4); k += 64 * kBlocksWaves)
    {
        const int h = k / (D / 4);
        const int d4 = (k - h * (D / 4)) * 4;
        float     Mx = kLowest, L = 0.0f;
        for (int w = 0; w < ST; ++w) Mx = fmaxf(Mx, s_ml[w][h].x);
        f32x4 o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int w = 0; w < ST; ++w)
        {
            const float x = __builtin_amdgcn_exp2f(s_ml[w][h].x - Mx);
            L += s_ml[w][h].y * x;
            o += *reinterpret_cast<const f32x4*>(&s_acc[w][h][d4]) * x;
        }
        store_state4<QT>(a, row * a.num_heads + kvh * G + h0 + h, split, D, d4, Mx, L, o);
    }
}

namespace
{

bool mfma_dim(int d) { return d == 64 || d == 80 || d == 96 || d == 112 || d == 128 || d == 256; }

// Workgroups of a token in an unsplit call: KV heads, and blocks of their query heads.
int64_t blocks_heads(const BlocksArgs& a)
{
    const int heads = blocks_kernel(a) == BlocksKernel::kDecode ? 16 : 4;
    return static_cast<int64_t>(a.num_kv_heads) * ((a.group + heads - 1) / heads);
}

template <int QT, typename F>
hipError_t for_cache(const BlocksArgs& a, F f)
{
    switch (a.cache_dtype)
    {
        case F32:
            return f.template operator()<QT, F32>();
        case F16:
            return f.template operator()<QT, F16>();
        case BF16:
            return f.template operator()<QT, BF16>();
        case I8:
            return f.template operator()<QT, I8>();
        default:
            return f.template operator()<QT, FP8>();
    }
}

template <typename F>
hipError_t for_types(const BlocksArgs& a, F f)
{
    if (a.qo_dtype == F32) return for_cache<F32>(a, f);
    if (a.qo_dtype == F16) return for_cache<F16>(a, f);
    return for_cache<BF16>(a, f);
}

}  // namespace

BlocksKernel blocks_kernel(const BlocksArgs& a)
{
    if (a.cache_dtype == F32 || !mfma_dim(a.head_dim)) return BlocksKernel::kVector;
    // (The prefill has no form of head_dim 80, 96 and 112, nor of fp32 pages: their lists are attended token by token, each token
    // reading its block's list again.  2 x 512 tokens in blocks of 64, 128 bf16 pages, 32/8 heads: 546, 545 and 790 us, where 128
    // dims take 58; fp32 at 128 dims 1268.)
    if (a.query_block == 1 || a.head_dim == 80 || a.head_dim == 96 || a.head_dim == 112) return BlocksKernel::kDecode;
    // Few tokens too, while the lists that each reads for itself come from the caches: by workgroups (token, KV head) and pages of
    // a list, 32/8 heads of 128, bf16, token by token and in the prefill's tiles: 32 x 256 14.7 and 17.3 us, 64 x 256 19.5 and
    // 18.5 (int8 19.7 and 23.3), 128 x 64 14.1 and 16.1, 128 x 256 28.6 and 19.0, 256 x 16 7.7 and 13.5, 256 x 64 15.7 and
    // 17.5, 512 x 16 10.5 and 13.5, 512 x 64 25.2 and 18.3, 1024 x 16 18.5 and 13.7.
    const int64_t wgs = static_cast<int64_t>(a.batch) * a.seq_len * a.num_kv_heads * ((a.group + 15) / 16);
    return wgs <= 512 && wgs * a.count <= 16384 ? BlocksKernel::kDecode : BlocksKernel::kPrefill;
}

namespace
{

ListPrefillArgs list_prefill_args(const BlocksArgs& a)
{
    ListPrefillArgs p{};
    p.q = a.q;
    p.out = a.out;
    p.k_cache = a.k_cache;
    p.v_cache = a.v_cache;
    p.k_scale = a.k_scale;
    p.v_scale = a.v_scale;
    p.block_table = a.block_table;
    p.context_lens = a.context_lens;
    p.qo_dtype = a.qo_dtype;
    p.cache_dtype = a.cache_dtype;
    p.batch = a.batch;
    p.seq_len = a.seq_len;
    p.num_heads = a.num_heads;
    p.num_kv_heads = a.num_kv_heads;
    p.group = a.group;
    p.head_dim = a.head_dim;
    p.max_blocks = a.max_blocks;
    p.num_blocks = a.num_blocks;
    p.cap_tokens = decode_cap_tokens(a.max_blocks, 0);
    p.paged = true;
    p.scale_log2 = a.scale_log2;
    p.n_split = 1;
    p.span_tokens = p.cap_tokens;
    p.blocks = a.blocks;
    p.lists = a.lists;
    p.count = a.count;
    p.query_block = a.query_block;
    return p;
}

// The lists as rows of query_block tokens, as the prefill's plan and layout count them.
ListPrefillArgs list_rows(ListPrefillArgs p)
{
    p.batch *= p.lists;
    p.seq_len = p.query_block;
    return p;
}

// Blocks of 128 query rows of all lists.
int64_t prefill_blocks(const BlocksArgs& a)
{
    return static_cast<int64_t>(a.batch) * a.lists * a.num_kv_heads * ((static_cast<int64_t>(a.query_block) * a.group + 127) / 128);
}

}  // namespace

// (split lists and halves of them are for few)
int64_t blocks_threads(const BlocksArgs& a)
{
    if (blocks_kernel(a) == BlocksKernel::kPrefill)  // whole rounds of the XCDs, eight or four waves a workgroup
    {
        const int64_t blocks = (static_cast<int64_t>(a.query_block) * a.group + 127) / 128;
        return (static_cast<int64_t>(a.batch) * a.lists * a.num_kv_heads + 7) / 8 * 8 * blocks * (a.head_dim == 256 ? 512 : 256);
    }
    return static_cast<int64_t>(a.batch) * a.seq_len * blocks_heads(a) * 64 * kBlocksWaves;
}

// Whether the prefill's lists can be taken in two halves: a workgroup of that form fills a CU, and each half has two steps.
bool blocks_pairable(const BlocksArgs& a)
{
    return blocks_kernel(a) == BlocksKernel::kPrefill && a.head_dim <= 128 && prefill_blocks(a) <= 256 &&
           std::min(a.count, a.max_blocks) >= 16;
}

// Sets a.splits, a.waves and a.pair, and gives the workspace's layout (sizes and types of `a` set).
BlocksLayout plan_blocks(BlocksArgs& a)
{
    BlocksLayout l{};
    a.splits = 1;
    a.waves = kBlocksWaves;
    a.pair = false;
    if (blocks_kernel(a) == BlocksKernel::kPrefill)
    {
        if (static_cast<int64_t>(a.batch) * a.lists > INT32_MAX) return l;
        ListPrefillArgs p = list_rows(list_prefill_args(a));
        p.count = std::min(a.count, a.max_blocks);  // (pages of a row, but for those listed twice)
        if (a.cache_dtype == BF16)
            plan_blocks_prefill_bf16(p);
        else if (a.cache_dtype == F16)
            plan_blocks_prefill_f16(p);
        else if (a.cache_dtype == I8)
            plan_blocks_prefill_i8(p);
        else
            plan_blocks_prefill_fp8(p);
        // More than 170 blocks make two pieces a list (or none, where lists are short): the halves of a workgroup do as well
        // and need no merge through memory.  256 blocks at 32/8 heads of 128, inputs resident: 128 listed pages fp8 57.8 -> 50.9
        // us (inputs that change from call to call: 57.1 -> 53.5), bf16 63.0 -> 55.2, int8 78.1 -> 67.5; 64 pages 39.7 -> 30.2,
        // 43.0 -> 33.6, 57.8 -> 40.4; 16 pages 15.4 -> 14.6; 8 pages 11.7 -> 12.0.  160 blocks of 128 pages take three pieces:
        // 43.2 there, 49.4 in halves.
        a.pair = blocks_pairable(a) && (p.n_split == 1 || 3 * prefill_blocks(a) > 512);
        if (a.pair) return l;
        a.splits = p.n_split;
        const PrefillSplitLayout s = prefill_split_layout(p);
        return BlocksLayout{s.ml, s.acc, s.total};
    }
    const int64_t wgs = static_cast<int64_t>(a.batch) * a.seq_len * blocks_heads(a);
    const int64_t pages = std::min(a.count, a.max_blocks);
    // Eight waves where there are at most as many workgroups as CUs (32 of 16 pages: 9.0 -> 7.2 us; 512 of 64 pages 49.4 -> 52.2
    // with eight).  Lists are split where the chip has room, two pages a wave and piece (16 lists of 256 pages: 14.2 us; with
    // four 15.6, with eight 21.3), but not below 8 pages a wave, where the merge's 3 us are not won back (28 pages: 9.6
    // whole, 10.6 split).
    a.waves = blocks_kernel(a) == BlocksKernel::kDecode && wgs <= 256 ? 8 : 4;
    const int64_t most = pages < 8 * a.waves ? 1 : pages / (2 * a.waves);
    a.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(2048 / a.waves / std::max<int64_t>(wgs, 1), most)));
    if (a.splits == 1) return l;
    const int64_t parts = static_cast<int64_t>(a.batch) * a.seq_len * a.num_heads * a.splits;
    l.acc = (parts * 8 + 255) / 256 * 256;
    l.total = l.acc + parts * a.head_dim * 4;
    return l;
}

void set_blocks_workspace(BlocksArgs& a, const BlocksLayout& l, void* ws)
{
    char* w = static_cast<char*>(ws);
    a.ws_pieces = reinterpret_cast<int32_t*>(w);  // (the prefill's; the others' states begin there)
    a.ws_ml = reinterpret_cast<float2*>(w + l.ml);
    a.ws_acc = reinterpret_cast<float*>(w + l.acc);
}

hipError_t launch_blocks_prefill(const BlocksArgs& a, hipStream_t stream)
{
    ListPrefillArgs p = list_prefill_args(a);
    p.n_split = a.splits;
    p.pair = a.pair;
    p.ws_pieces = a.ws_pieces;
    p.ws_ml = reinterpret_cast<float*>(a.ws_ml);
    p.ws_acc = a.ws_acc;
    if (a.cache_dtype == BF16) return launch_blocks_prefill_bf16(p, stream);
    if (a.cache_dtype == F16) return launch_blocks_prefill_f16(p, stream);
    if (a.cache_dtype == I8) return launch_blocks_prefill_i8(p, stream);
    return launch_blocks_prefill_fp8(p, stream);
}

hipError_t launch_blocks(const BlocksArgs& a, hipStream_t stream)
{
    const BlocksKernel kernel = blocks_kernel(a);
    if (kernel == BlocksKernel::kPrefill) return launch_blocks_prefill(a, stream);
    const int64_t wgs = static_cast<int64_t>(a.batch) * a.seq_len * blocks_heads(a) * a.splits;
    const int64_t rows = static_cast<int64_t>(a.batch) * a.seq_len * a.num_heads;
    if (blocks_threads(a) > kMostThreads) return hipErrorInvalidConfiguration;
    const dim3 grid(static_cast<unsigned>(wgs)), block(static_cast<unsigned>(64 * a.waves));
    hipError_t e;
    if (kernel == BlocksKernel::kDecode)
        e = for_types(a, [&]<int QT, int CT>()
        {
            auto go = [&]<int D>()
            {
                const unsigned lds = static_cast<unsigned>(blocks_lds_bytes<D>(a.waves, std::min(a.group, 16)));
                if constexpr (CT != F32)
                {
                    if (a.waves == 8)
                        hipLaunchKernelGGL((paged_blocks_decode<CT, QT, D, 8>), grid, block, lds, stream, a);
                    else
                        hipLaunchKernelGGL((paged_blocks_decode<CT, QT, D, 4>), grid, block, lds, stream, a);
                }
                return hipGetLastError();
            };
            if (a.head_dim == 64) return go.template operator()<64>();
            if (a.head_dim == 80) return go.template operator()<80>();
            if (a.head_dim == 96) return go.template operator()<96>();
            if (a.head_dim == 112) return go.template operator()<112>();
            if (a.head_dim == 128) return go.template operator()<128>();
            return go.template operator()<256>();
        });
    else
        e = for_types(a, [&]<int QT, int CT>()
        {
            if (a.head_dim <= 128)
                hipLaunchKernelGGL((paged_blocks_vector<CT, QT, 16>), grid, block, 0, stream, a);
            else
                hipLaunchKernelGGL((paged_blocks_vector<CT, QT, 32>), grid, block, 0, stream, a);
            return hipGetLastError();
        });
    if (e != hipSuccess || a.splits == 1) return e;
    const dim3 merge(static_cast<unsigned>(rows));
    if (a.qo_dtype == F32)
        hipLaunchKernelGGL((blocks_merge<F32>), merge, dim3(256), 0, stream, a);
    else if (a.qo_dtype == F16)
        hipLaunchKernelGGL((blocks_merge<F16>), merge, dim3(256), 0, stream, a);
    else
        hipLaunchKernelGGL((blocks_merge<BF16>), merge, dim3(256), 0, stream, a);
    return hipGetLastError();
}

}  // namespace ffkv
