// rope_axes.hip - rotary embedding of q and k by positions on several axes (time, height, width), fused with the KV-page
// append, on gfx950.
//
// Pair i of a head (dims i and i + D/2, 0 <= i < D/2) of token t of row b turns by the angle
//   p[axis(i), b, t] * theta^(-2i/D):   lo' = lo cos - hi sin,   hi' = hi cos + lo sin
// axis(i) by sections (the first section_0 pairs turn by axis 0, the next section_1 by axis 1, ..) or interleaved (pair i by
// axis i mod A while that axis has pairs left, those past by axis 0).  With equal positions on all axes this is the plain
// rotary embedding.  The rotated q goes to q_out, the rotated k, rounded to its type, and v to their pages as the append
// writes them (int8 and fp8 quantized).
//
// Angles: far positions turn by 10^5 radians and more, of which fp32 keeps two digits behind the point.  The turns
// p * rate / 2 pi are one fp64 product; only their fraction, in [-1/2, 1/2], goes on to fp32 as a pair of parts, of which the
// low one enters to first order: what is left is the rounding of cos and sin to fp32 and the errors of the rate, 2^-48 of
// the angle at most: 2^-22 + |p| 2^-48 in all (theta >= 1).
//
// Bound by HBM (q read and written, k and v read and written once): 8 x 1500 f16 tokens of 32/8 heads of 128, 295 MB, 58.4 us =
// 5.1 TB/s; 32000 bf16 tokens of 28/4 heads, 590 MB, 102 us = 5.8 TB/s (device copies of as many bytes take 55.6 and 109 us: a copy
// is no bound).  A step of 4 tokens takes 3.5 us.  Into int8 and fp8 pages the 8 x 1500 tokens take 62 and 63 us, where their
// own type takes 50 (inputs resident): the quantization's vector work; alone, without pages, 38.5.
#include "blocks.h"
#include "ffkv_device.h"

#include <algorithm>

namespace ffkv
{

namespace
{

constexpr int kRopeThreads = 256;

// Write 8 values of a (token, head) row to the cache at element index dst; sc as append_row has it.
template <int CACHE>
__device__ __forceinline__ void store_cache8(void* cache, size_t dst, const float* x, float sc)
{
    Raw8 out;
    if constexpr (CACHE == I8)
    {
        quant8<true>(x, sc == 0.0f ? 1.0f : sc, out.w);
        if (sc == 0.0f) out.w[0] = out.w[1] = 0u;  // an all-zero row
    }
    else if constexpr (CACHE == FP8)
        quant8<false>(x, sc, out.w);
    else
        pack8<CACHE>(x, out);
    store_raw8<CACHE>(cache, dst, out);
}

// The scale of a row whose 16 values per lane lie over LPR lanes: int8 its absmax / 127 (NaN passed over), fp8 the head's.
// Every lane of the wave calls it.
template <int CACHE, int LPR>
__device__ __forceinline__ float row_scale(const float* scales, int h, const float* xl, const float* xh)
{
    if constexpr (CACHE == I8)
    {
        float amax = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i)
        {
            const float u = __builtin_fabsf(xl[i]), w = __builtin_fabsf(xh[i]);
            amax = u > amax ? u : amax;
            amax = w > amax ? w : amax;
        }
        amax = group_max<LPR>(amax);
        return amax == 0.0f ? 0.0f : amax / 127.0f;
    }
    return CACHE == FP8 ? scales[h] : 0.0f;
}

}  // namespace

// A wave takes 64 / (D/16) head rows of a token: its lanes evaluate the token's cos and sin, a pair each (head_dim 256: two), and
// exchange them through the wave's own stretch of LDS, without a barrier; then D/16 lanes rotate a head row, each its 8 dims of
// the low half and the matching 8 of the high half.  (A token's other waves evaluate the same table again, behind their
// loads: twice or three times the rows a wave take as long for 4 tokens, and 59.1 and 60.7 us instead of 58.3 for 12000.)
template <int SRC, int CACHE, int D, bool APPEND>
__global__ __launch_bounds__(kRopeThreads) void rope_axes_kernel(RopeAxesArgs a, int parts)
{
    constexpr int HALF = D / 2;
    constexpr int LPR = D / 16;    // lanes per head row
    constexpr int RPP = 64 / LPR;  // head rows of a pass
    constexpr int PPL = HALF > 64 ? HALF / 64 : 1;  // pairs a lane evaluates
    __shared__ float s_cs[kRopeThreads / 64][2][HALF];

    const int     tid = static_cast<int>(threadIdx.x);
    const int     lane = tid & 63;
    const int     wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int     col = lane % LPR;
    const int     sub = lane / LPR;
    const int     rows = a.num_heads + a.num_kv_heads;
    const uint32_t items = static_cast<uint32_t>(a.batch) * a.seq_len * parts;
    float*        s_cos = s_cs[wave][0];
    float*        s_sin = s_cs[wave][1];

    double rate[PPL];  // turns per position of the lane's pairs
    int    axis[PPL];
#pragma unroll
    for (int p = 0; p < PPL; ++p)
    {
        const int i = (lane + 64 * p) % HALF;
        rate[p] = exp2(i * a.rate_log2) * 0.15915494309189533577;
        if (a.interleaved)
        {
            const int ax = i % a.axes;
            axis[p] = ax > 0 && i / a.axes < a.section_end[ax] ? ax : 0;
        }
        else
            axis[p] = (i >= a.section_end[0]) + (i >= a.section_end[1]) + (i >= a.section_end[2]);
    }

    for (uint32_t item = blockIdx.x * (kRopeThreads / 64) + wave; item < items; item += gridDim.x * (kRopeThreads / 64))
    {
        // (a token's parts lie side by side: apart, its rows' lines are fetched twice, 61 -> 69 us for 12000 tokens)
        const Split    v = split_index(item, parts), u = split_index(v.div, a.seq_len);
        const uint32_t tok = v.div;
        const int      part = v.rem, b = static_cast<int>(u.div), t = u.rem;
        int           at[PPL];
#pragma unroll
        for (int p = 0; p < PPL; ++p)
            at[p] = a.positions[static_cast<int64_t>(axis[p]) * a.batch * a.seq_len + tok];
        int64_t slot = -1;  // of the token in the pools
        if constexpr (APPEND)
        {
            const int64_t pos = static_cast<int64_t>(a.context_lens ? a.context_lens[b] : 0) + t;
            if (pos >= 0 && (pos >> 4) < a.max_blocks)
            {
                const int phys = a.block_table[static_cast<int64_t>(b) * a.max_blocks + (pos >> 4)];
                if (phys >= 0 && phys < a.num_blocks) slot = static_cast<int64_t>(phys) * kBlockSize + (pos & 15);
            }
        }
        const int  row = part * RPP + sub;
        const bool in = row < rows;
        const bool isq = row < a.num_heads;
        const int  h = isq ? row : row - a.num_heads;
        Raw8       rl, rh, vl, vh;
        if (in)
        {
            const size_t at8 = static_cast<size_t>(tok) * (isq ? a.q_stride : a.k_stride) + h * D + 8 * col;
            const void*  src = isq ? a.q : a.k;
            load_raw8<SRC>(src, at8, rl);
            load_raw8<SRC>(src, at8 + HALF, rh);
            if (APPEND && !isq)
            {
                const size_t v8 = static_cast<size_t>(tok) * a.v_stride + h * D + 8 * col;
                load_raw8<SRC>(a.v, v8, vl);
                load_raw8<SRC>(a.v, v8 + HALF, vh);
            }
        }
        // the token's table, behind the loads
#pragma unroll
        for (int p = 0; p < PPL; ++p)
        {
            const double turns = static_cast<double>(at[p]) * rate[p];
            const double half_turns = 2.0 * (turns - rint(turns));  // in [-1, 1]
            const float  hi = static_cast<float>(half_turns);
            const float  lo = static_cast<float>(half_turns - static_cast<double>(hi)) * 3.14159265358979f;
            float        s, c;
            sincospif(hi, &s, &c);
            s_cos[(lane + 64 * p) % HALF] = __builtin_fmaf(-lo, s, c);
            s_sin[(lane + 64 * p) % HALF] = __builtin_fmaf(lo, c, s);
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        float c8[8], s8[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
        {
            c8[e] = s_cos[8 * col + e];
            s8[e] = s_sin[8 * col + e];
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        float xl[8], xh[8], yl[8], yh[8];
        if (in)
        {
            unpack8<SRC>(rl, xl);
            unpack8<SRC>(rh, xh);
#pragma unroll
            for (int e = 0; e < 8; ++e)
            {
                yl[e] = __builtin_fmaf(xl[e], c8[e], -(xh[e] * s8[e]));
                yh[e] = __builtin_fmaf(xh[e], c8[e], xl[e] * s8[e]);
            }
            pack8<SRC>(yl, rl);
            pack8<SRC>(yh, rh);
            if (isq || a.k_out != nullptr)
            {
                void*        dst = isq ? a.q_out : a.k_out;
                const size_t at8 = static_cast<size_t>(tok) * (isq ? a.q_out_stride : a.k_out_stride) + h * D + 8 * col;
                store_raw8<SRC>(dst, at8, rl);
                store_raw8<SRC>(dst, at8 + HALF, rh);
            }
        }
        if constexpr (APPEND)
        {
            const bool   go = in && !isq && slot >= 0;
            const size_t row_c = static_cast<size_t>(go ? slot : 0) * a.num_kv_heads + (go ? h : 0);
            if constexpr (SRC == CACHE)
            {
                if (go)
                {
                    store_raw8<CACHE>(a.k_cache, row_c * D + 8 * col, rl);
                    store_raw8<CACHE>(a.k_cache, row_c * D + HALF + 8 * col, rh);
                    store_raw8<CACHE>(a.v_cache, row_c * D + 8 * col, vl);
                    store_raw8<CACHE>(a.v_cache, row_c * D + HALF + 8 * col, vh);
                }
            }
            else if (__any(go))  // (the rows' maxima take every lane)
            {
                if (!go)
                {
#pragma unroll
                    for (int e = 0; e < 8; ++e) rl.w[e] = rh.w[e] = vl.w[e] = vh.w[e] = 0u;
                }
                // k as stored in its own type: what an append of the rotated k reads
                unpack8<SRC>(rl, xl);
                unpack8<SRC>(rh, xh);
                unpack8<SRC>(vl, yl);
                unpack8<SRC>(vh, yh);
                const float ks = row_scale<CACHE, LPR>(a.k_scale, go ? h : 0, xl, xh);
                const float vs = row_scale<CACHE, LPR>(a.v_scale, go ? h : 0, yl, yh);
                if (go)
                {
                    if (CACHE == I8 && col == 0)
                    {
                        a.k_scale[row_c] = ks;
                        a.v_scale[row_c] = vs;
                    }
                    store_cache8<CACHE>(a.k_cache, row_c * D + 8 * col, xl, ks);
                    store_cache8<CACHE>(a.k_cache, row_c * D + HALF + 8 * col, xh, ks);
                    store_cache8<CACHE>(a.v_cache, row_c * D + 8 * col, yl, vs);
                    store_cache8<CACHE>(a.v_cache, row_c * D + HALF + 8 * col, yh, vs);
                }
            }
        }
    }
}

namespace
{

template <int SRC, int CACHE, bool APPEND, int D>
hipError_t launch_axes_d(const RopeAxesArgs& a, hipStream_t stream)
{
    constexpr int RPP = 64 / (D / 16);
    const int64_t tokens = static_cast<int64_t>(a.batch) * a.seq_len;
    const int     parts = (a.num_heads + a.num_kv_heads + RPP - 1) / RPP;
    const int64_t wgs = (tokens * parts + kRopeThreads / 64 - 1) / (kRopeThreads / 64);
    if (tokens * parts > INT32_MAX) return hipErrorInvalidConfiguration;
    hipLaunchKernelGGL((rope_axes_kernel<SRC, CACHE, D, APPEND>), dim3(static_cast<unsigned>(std::min<int64_t>(wgs, 65536))),
                       dim3(kRopeThreads), 0, stream, a, parts);
    return hipGetLastError();
}

template <int SRC, int CACHE, bool APPEND>
hipError_t launch_axes_c(const RopeAxesArgs& a, hipStream_t stream)
{
    if (a.head_dim == 64) return launch_axes_d<SRC, CACHE, APPEND, 64>(a, stream);
    if (a.head_dim == 128) return launch_axes_d<SRC, CACHE, APPEND, 128>(a, stream);
    return launch_axes_d<SRC, CACHE, APPEND, 256>(a, stream);
}

template <int SRC>
hipError_t launch_axes_s(const RopeAxesArgs& a, hipStream_t stream)
{
    if (a.k_cache == nullptr) return launch_axes_c<SRC, SRC, false>(a, stream);
    switch (a.cache_dtype)
    {
        case F32:
            return launch_axes_c<SRC, F32, true>(a, stream);
        case F16:
            return launch_axes_c<SRC, F16, true>(a, stream);
        case BF16:
            return launch_axes_c<SRC, BF16, true>(a, stream);
        case I8:
            return launch_axes_c<SRC, I8, true>(a, stream);
        default:
            return launch_axes_c<SRC, FP8, true>(a, stream);
    }
}

}  // namespace

hipError_t launch_rope_axes(const RopeAxesArgs& a, hipStream_t stream)
{
    if (a.src_dtype == F32) return launch_axes_s<F32>(a, stream);
    if (a.src_dtype == F16) return launch_axes_s<F16>(a, stream);
    return launch_axes_s<BF16>(a, stream);
}

}  // namespace ffkv
