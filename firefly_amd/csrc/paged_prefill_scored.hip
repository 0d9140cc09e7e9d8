// paged_prefill_scored.hip - prefill attention under a score rule: tanh cap, distance bias, window, and a range of visible
// keys per query (documents, prefixes).
//
// For the query of token t of row b at position i = context_lens[b] + t, head h and key j:
//   s_j = cap tanh(scale q.k_j / cap) - slope_h |i - j|,  lo <= j < hi,  out = sum_j softmax(s)_j v_j
//   lo = max(0, key_begin[b, t], i - window + 1), hi = min(row's tokens, key_end[b, t] or i + 1)
//
// The attention is the plain prefill's code (paged_prefill_dma.hip: prefill_wg with RULE).  Every mask is a range of keys
// per query, so a workgroup of 128 query rows streams the pages between the smallest lo and the largest hi of its rows, a
// step below every column's lo or past its hi costs nothing, and one that all columns see whole needs no mask.
#define FFKV_DEVICE_BODIES_ONLY 1
#include "paged_prefill_dma.hip"
#undef FFKV_DEVICE_BODIES_ONLY

namespace ffkv
{

template <int QT, int D, int CT, int RG, bool SPLIT>
__global__ __launch_bounds__(512 / RG)
__attribute__((amdgpu_waves_per_eu(RG == 2 ? (D == 256 ? 1 : 2) : 1)))
void paged_prefill_scored(PrefillArgs a)
{
    using L = PrefillLds<QT, D, CT, false, RG>;
    __shared__ __align__(16) uint8_t s_st0[L::STAGE];
    __shared__ __align__(16) uint8_t s_st1[L::STAGE];
    __shared__ __align__(16) uint8_t s_st2[L::S2];
    __shared__ __align__(16) uint8_t s_st3[L::S3];
    __shared__ int s_flags[kRuleFlags];
    prefill_wg<QT, D, CT, false, RG, SPLIT, true>(a, static_cast<int>(blockIdx.x), s_st0, s_st1, s_st2, s_st3, s_flags[0]);
}

namespace
{

// f.operator()<QT, D, CT, RG>() for the call's types and head_dim.
template <typename F>
auto prefill_for(const PrefillArgs& a, F f)
{
    auto d = [&]<int CT, int QT>()
    {
        if (a.head_dim == 64) return f.template operator()<QT, 64, CT, FFKV_PREFILL_RG>();
        if (a.head_dim == 128) return f.template operator()<QT, 128, CT, FFKV_PREFILL_RG>();
        return f.template operator()<QT, 256, CT, FFKV_PREFILL_RG256>();
    };
    auto q = [&]<int CT>()
    {
        if (a.qo_dtype == F32) return d.template operator()<CT, F32>();
        if (a.qo_dtype == F16) return d.template operator()<CT, F16>();
        return d.template operator()<CT, BF16>();
    };
    if (a.cache_dtype == F16) return q.template operator()<F16>();
    if (a.cache_dtype == BF16) return q.template operator()<BF16>();
    if (a.cache_dtype == I8) return q.template operator()<I8>();
    return q.template operator()<FP8>();
}

}  // namespace

void prefill_scored_plan(PrefillArgs& a)
{
    prefill_for(a, [&]<int QT, int D, int CT, int RG>()
    {
        prefill_plan_for(a, reinterpret_cast<const void*>(paged_prefill_scored<QT, D, CT, RG, true>), 512 / RG,
                         DmaCfg<D, kElemBytes<CT>, CT == I8, 8 / RG, false>::KP * kBlockSize, a.span_tokens);
    });
}

hipError_t launch_prefill_scored(const PrefillArgs& a, hipStream_t stream)
{
    const bool    split = a.n_split > 1;
    const int64_t groups = static_cast<int64_t>(a.batch) * a.num_kv_heads * (split ? a.n_split : 1);
    const int64_t nrb = (static_cast<int64_t>(a.seq_len) * a.group + kDmaRows - 1) / kDmaRows;
    const int64_t wgs = (groups + kXcds - 1) / kXcds * kXcds * nrb;
    if (wgs <= 0) return hipSuccess;
    if (wgs > INT32_MAX) return hipErrorInvalidConfiguration;
    const dim3       grid(static_cast<unsigned>(wgs));
    const hipError_t e = prefill_for(a, [&]<int QT, int D, int CT, int RG>()
    {
        if (split)
            hipLaunchKernelGGL((paged_prefill_scored<QT, D, CT, RG, true>), grid, dim3(512 / RG), 0, stream, a);
        else
            hipLaunchKernelGGL((paged_prefill_scored<QT, D, CT, RG, false>), grid, dim3(512 / RG), 0, stream, a);
        return hipGetLastError();
    });
    return e != hipSuccess || !split ? e : launch_prefill_merge(a, stream);
}

}  // namespace ffkv
