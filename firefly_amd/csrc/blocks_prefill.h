// blocks_prefill.h - the prefill over listed pages: its kernel, instantiated by paged_blocks_prefill_*.hip for a type of cache
// each (files of their own, as each takes a minute to compile).
#pragma once

#define FFKV_DEVICE_BODIES_ONLY 1
#include "paged_prefill_dma.hip"
#undef FFKV_DEVICE_BODIES_ONLY

namespace ffkv
{

template <int QT, int D, int CT, int RG, bool SPLIT>
__global__ __launch_bounds__(512 / RG)
__attribute__((amdgpu_waves_per_eu(RG == 2 ? (D == 256 ? 1 : 2) : 1)))
void paged_blocks_prefill(ListPrefillArgs a)
{
    using L = PrefillLds<QT, D, CT, false, RG>;
    __shared__ __align__(16) uint8_t s_st0[L::STAGE];
    __shared__ __align__(16) uint8_t s_st1[L::STAGE];
    __shared__ __align__(16) uint8_t s_st2[L::S2];
    __shared__ __align__(16) uint8_t s_st3[L::S3];
    __shared__ int s_flags[kRuleFlags];
    prefill_wg<QT, D, CT, false, RG, SPLIT, true, true>(a, static_cast<int>(blockIdx.x), s_st0, s_st1, s_st2, s_st3, s_flags[0]);
}

// Two halves of a list by the two halves of a workgroup (PAIR).
template <int QT, int D, int CT, int RG>
__global__ __launch_bounds__(1024 / RG) __attribute__((amdgpu_waves_per_eu(2)))
void paged_blocks_prefill_pair(ListPrefillArgs a)
{
    using L = PrefillLds<QT, D, CT, false, RG>;
    static_assert(2 * L::BYTES + 64 <= 160 * 1024, "both halves' stages");
    __shared__ __align__(16) uint8_t s_st0[2 * L::STAGE];
    __shared__ __align__(16) uint8_t s_st1[2 * L::STAGE];
    __shared__ __align__(16) uint8_t s_st2[2 * L::S2];
    __shared__ __align__(16) uint8_t s_st3[2 * L::S3];
    __shared__ int s_flags[2 * kRuleFlags - 1];
    prefill_wg<QT, D, CT, false, RG, false, true, true, true>(a, static_cast<int>(blockIdx.x), s_st0, s_st1, s_st2, s_st3,
                                                              s_flags[0]);
}

namespace
{

// f.operator()<QT, D, RG>() for the call's types and head_dim.
template <typename F>
auto list_prefill_for(const ListPrefillArgs& a, F f)
{
    auto d = [&]<int QT>()
    {
        if (a.head_dim == 64) return f.template operator()<QT, 64, FFKV_PREFILL_RG>();
        if (a.head_dim == 128) return f.template operator()<QT, 128, FFKV_PREFILL_RG>();
        return f.template operator()<QT, 256, FFKV_PREFILL_RG256>();
    };
    if (a.qo_dtype == F32) return d.template operator()<F32>();
    if (a.qo_dtype == F16) return d.template operator()<F16>();
    return d.template operator()<BF16>();
}

}  // namespace

// One type of cache's launch, split over the lists where a.n_split > 1.
template <int CT>
hipError_t launch_blocks_prefill_t(const ListPrefillArgs& a, hipStream_t stream)
{
    const int64_t groups = static_cast<int64_t>(a.batch) * a.lists * a.num_kv_heads * (a.n_split > 1 ? a.n_split : 1);
    const int64_t nrb = (static_cast<int64_t>(a.query_block) * a.group + kDmaRows - 1) / kDmaRows;
    const int64_t wgs = (groups + kXcds - 1) / kXcds * kXcds * nrb;
    if (wgs <= 0) return hipSuccess;
    if (wgs > INT32_MAX) return hipErrorInvalidConfiguration;
    const dim3 grid(static_cast<unsigned>(wgs));
    const hipError_t e = list_prefill_for(a, [&]<int QT, int D, int RG>()
    {
        if (a.pair)
        {
            if constexpr (D <= 128)
                hipLaunchKernelGGL((paged_blocks_prefill_pair<QT, D, CT, RG>), grid, dim3(1024 / RG), 0, stream, a);
        }
        else if (a.n_split > 1)
            hipLaunchKernelGGL((paged_blocks_prefill<QT, D, CT, RG, true>), grid, dim3(512 / RG), 0, stream, a);
        else
            hipLaunchKernelGGL((paged_blocks_prefill<QT, D, CT, RG, false>), grid, dim3(512 / RG), 0, stream, a);
        return hipGetLastError();
    });
    return e != hipSuccess || a.n_split <= 1 ? e : launch_blocks_prefill_merge(a, stream);
}

// Its plan: n_split of `a` (batch and seq_len: the lists, and the tokens of one).
template <int CT>
void plan_blocks_prefill_t(ListPrefillArgs& a)
{
    list_prefill_for(a, [&]<int QT, int D, int RG>()
    {
        constexpr int KEYS = DmaCfg<D, kElemBytes<CT>, CT == I8, 8 / RG, false>::KP * kBlockSize;
        prefill_plan_for(a, reinterpret_cast<const void*>(paged_blocks_prefill<QT, D, CT, RG, true>), 512 / RG, KEYS,
                         a.count > (1 << 26) ? 1 << 30 : a.count * kBlockSize);
    });
}

}  // namespace ffkv
