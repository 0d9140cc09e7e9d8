// prefill_scored.h - the scored prefill's kernel, of which paged_prefill_scored.hip instantiates the whole form and
// paged_prefill_scored_split.hip the one split over its keys (two files, as they take minutes to compile).
#pragma once

#define FFKV_DEVICE_BODIES_ONLY 1
#include "paged_prefill_dma.hip"
#undef FFKV_DEVICE_BODIES_ONLY

namespace ffkv
{

template <int QT, int D, int CT, int RG, bool SPLIT>
__global__ __launch_bounds__(512 / RG)
__attribute__((amdgpu_waves_per_eu(RG == 2 ? (D == 256 ? 1 : 2) : 1)))
void paged_prefill_scored(ScoredPrefillArgs a)
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
auto prefill_for(const ScoredPrefillArgs& a, F f)
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

namespace
{

// The main launch, for a grid of `wgs` workgroups.
template <bool SPLIT>
hipError_t launch_scored(const ScoredPrefillArgs& a, unsigned wgs, hipStream_t stream)
{
    return prefill_for(a, [&]<int QT, int D, int CT, int RG>()
    {
        hipLaunchKernelGGL((paged_prefill_scored<QT, D, CT, RG, SPLIT>), dim3(wgs), dim3(512 / RG), 0, stream, a);
        return hipGetLastError();
    });
}

}  // namespace

}  // namespace ffkv
