// paged_decode_scored_weights.hip - the scored decode that writes its scores down, and the attention weights from them.
#include "decode_scored.h"

namespace ffkv
{

// weights[b, kvh, j] of the tokens j of row b: the scores of the KV head's query heads against their final maxima and
// denominators.  A thread takes kWeightTokens tokens, 256 apart, so that their scores are in flight together (one token each
// took 17 us on 64 rows of 512 to 4096 tokens, this takes 10).  The row's own new token has no earlier weight.  Tokens
// at or past the row's end (or past max_context_len) are left alone.
constexpr int kWeightTokens = 4;
__global__ __launch_bounds__(256) void paged_decode_weights(ScoredDecodeArgs a)
{
    constexpr int T = kWeightTokens;
    const int     b = static_cast<int>(blockIdx.z);
    const int     kvh = static_cast<int>(blockIdx.y);
    RowSpan       s = row_span(a, b);
    if (a.num_blocks <= 0) s.lo = s.hi;  // no key is on a page, and some vector kernels then write no scores down
    const int     G = a.group;
    const float2* fin = reinterpret_cast<const float2*>(a.ws_final) + static_cast<int64_t>(b) * a.num_heads + kvh * G;
    const float*  sc = a.ws_scores + score_page(a, b, kvh, 0);
    const int64_t at = (static_cast<int64_t>(b) * a.num_kv_heads + kvh) * a.weight_stride;
    for (int j0 = static_cast<int>(blockIdx.x * 256 * T); j0 < s.hi; j0 += static_cast<int>(gridDim.x * 256 * T))
    {
        const int first = j0 + static_cast<int>(threadIdx.x);
        float     w[T], before[T];
#pragma unroll
        for (int t = 0; t < T; ++t)
        {
            const int j = first + 256 * t;
            w[t] = 0.0f;
            before[t] = a.prior != nullptr && j < s.pos && j < s.hi ? a.prior[at + j] : 0.0f;
        }
        constexpr int H = 4;  // heads whose scores are in flight together
        for (int h0 = 0; h0 < G; h0 += H)
        {
            float v[H][T];
#pragma unroll
            for (int h = 0; h < H; ++h)
#pragma unroll
                for (int t = 0; t < T; ++t)
                {
                    const int j = first + 256 * t;
                    v[h][t] = h0 + h < G && j >= s.lo && j < s.hi ? sc[(static_cast<int64_t>(j >> 4) * G + h0 + h) * kBlockSize + (j & 15)] : kNegInf;
                }
#pragma unroll
            for (int h = 0; h < H; ++h)
                if (h0 + h < G)
                {
                    const float2 f = fin[h0 + h];
                    const float  inv = softmax_inv(f.y);
#pragma unroll
                    for (int t = 0; t < T; ++t)  // (a key on no page weighs nothing, in a NaN query's row too)
                        w[t] += v[h][t] == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(v[h][t] - f.x) * inv;
                }
        }
#pragma unroll
        for (int t = 0; t < T; ++t)
        {
            const int j = first + 256 * t;
            if (j < s.hi) a.weights[at + j] = a.prior != nullptr && j < s.pos ? __builtin_fmaf(a.decay, before[t], w[t]) : w[t];
        }
    }
}

hipError_t launch_decode_scores(const ScoredDecodeArgs& a, bool row, hipStream_t stream)
{
    return scored_for(a, [&]<int CT, int QT, int D>() { return launch_scored3<CT, QT, D, true>(a, row, stream); });
}

hipError_t launch_decode_weights(const ScoredDecodeArgs& a, hipStream_t stream)
{
    // enough workgroups for the longest row's tokens, up to 64 per (row, KV head): beyond that each takes several stretches
    const int64_t blocks = (static_cast<int64_t>(a.cap_tokens) + 256 * kWeightTokens - 1) / (256 * kWeightTokens);
    const dim3    grid(static_cast<unsigned>(blocks < 1 ? 1 : (blocks > 64 ? 64 : blocks)),
                       static_cast<unsigned>(a.num_kv_heads), static_cast<unsigned>(a.batch));
    hipLaunchKernelGGL(paged_decode_weights, grid, dim3(256), 0, stream, a);
    return hipGetLastError();
}

}  // namespace ffkv
