// score_rule.h - what a score rule does to a score and to the keys a query sees: the tanh cap, the distance bias, the
// window and the given ranges, shared by the scored decode, the scored prefill and the attention weights (gfx950).
#pragma once

#include "ffkv_device.h"
#include "ffkv_internal.h"

#include <type_traits>

namespace ffkv
{

namespace
{

// cap * tanh(x) of a score x in units of its cap.  Below 0.6 tanh(x) = x + x^3 P(x^2) with P fitted to a relative error
// under 2^-23 (1 - 2 / (e^2x + 1) would lose the small scores' low bits: an absolute error of 2^-24 of the cap, 6e-6 at a
// cap of 50), above it (1 - e) / (1 + e) with e = e^-2|x|, which holds at infinity (e = 0).
constexpr float kCapNear = 0.6f;
__device__ __forceinline__ float cap_near(float x, float cap)
{
    const float t = x * x;
    float       p = -0.005908978637307882f;
    p = __builtin_fmaf(p, t, 0.0208087470382452f);
    p = __builtin_fmaf(p, t, -0.053787969052791595f);
    p = __builtin_fmaf(p, t, 0.13331978023052216f);
    p = __builtin_fmaf(p, t, -0.33333301544189453f);
    return cap * __builtin_fmaf(x * t, p, x);
}
__device__ __forceinline__ float cap_score(float x, float cap)
{
    const float ax = __builtin_fabsf(x);
    const float e = __builtin_amdgcn_exp2f(ax * -2.8853900817779268f);
    const float far = cap * __builtin_copysignf((1.0f - e) * __builtin_amdgcn_rcpf(1.0f + e), x);
    return ax < kCapNear ? cap_near(x, cap) : far;
}
// The same for N scores of every lane.  Scores are mostly well below their cap (a cap of 30 to 50 over scores of a standard
// deviation of a few), and a wave all of whose scores are near takes the polynomial alone: 8 vector instructions per score
// instead of 16 and two transcendental ones of four times the time.  (A shorter one up to 0.35 gains less than the waves that
// then pass it cost: weights of 16 x 64 tokens over int8 pages at a cap of 50, 258 us against 236.)
template <int N>
__device__ __forceinline__ void cap_scores(float (&x)[N], float cap)
{
    float most = 0.0f;
#pragma unroll
    for (int e = 0; e < N; ++e) most = fmaxf(most, __builtin_fabsf(x[e]));  // (NaN is passed over: both forms keep it)
    if (__any(most >= kCapNear))
    {
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = cap_score(x[e], cap);
    }
    else
    {
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = cap_near(x[e], cap);
    }
}

// First visible key of the query at position pos (before the row's end is looked at): the window's and the given one's.
__device__ __forceinline__ int64_t first_key(const ScoreRule& r, int64_t pos, int64_t begin)
{
    int64_t lo = begin > 0 ? begin : 0;
    if (r.window > 0 && lo < pos + 1 - r.window) lo = pos + 1 - r.window;
    return lo;
}

// What a decode kernel, and a prefill kernel, takes, with a rule or without.
template <bool RULE>
using KernelArgs = std::conditional_t<RULE, ScoredDecodeArgs, DecodeArgs>;
template <bool RULE>
using PrefillKernelArgs = std::conditional_t<RULE, ScoredPrefillArgs, PrefillArgs>;

// The rule of a kernel's arguments: none in a plain kernel's.
template <typename A>
__device__ __forceinline__ ScoreRule rule_in(const A& a)
{
    if constexpr (requires { a.rule; })
        return a.rule;
    else
        return ScoreRule{};
}

// Scores that the decode writes down for the weights: [batch, num_kv_heads, pages, group, 16 tokens], so that what a wave
// writes of a page (up to 16 heads of 64 bytes) is contiguous.
__device__ __forceinline__ int64_t score_page(const ScoredDecodeArgs& a, int b, int kvh, int page)
{
    return ((static_cast<int64_t>(b) * a.num_kv_heads + kvh) * (a.score_stride / kBlockSize) + page) * a.group * kBlockSize;
}

// Tokens that the decode of row b attends under the rule: [lo, hi).
struct RowSpan
{
    int lo, hi, pos;  // lo <= hi; pos: the query's position
};
__device__ __forceinline__ RowSpan row_span(const ScoredDecodeArgs& a, int b)
{
    const int64_t pos = a.context_lens[b];
    int64_t       hi = pos + 1;  // +1: the token appended this step
    if (hi > a.cap_tokens) hi = a.cap_tokens;
    if (hi < 0) hi = 0;
    int64_t lo = first_key(a.rule, pos, a.rule.key_begin != nullptr ? a.rule.key_begin[b] : 0);
    if (lo > hi) lo = hi;
    return RowSpan{static_cast<int>(lo), static_cast<int>(hi), static_cast<int>(pos)};
}

}  // namespace

}  // namespace ffkv
