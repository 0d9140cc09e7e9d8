// decode_scored.h - the scored decode's two kernels and their launch, of which paged_decode_scored.hip instantiates the plain
// ones and paged_decode_scored_weights.hip those that write the scores down (two files, as they take minutes to compile).
#pragma once

#define FFKV_DEVICE_BODIES_ONLY 1
#include "paged_decode_mfma.hip"
#undef FFKV_DEVICE_BODIES_ONLY

namespace ffkv
{

namespace
{

constexpr int kScoredRowWaves = 8;  // waves per workgroup of the one-launch form, as in the plain decode's

template <int D>
constexpr int scored_row_lds(int heads)
{
    const int v = kScoredRowWaves * kBlockSize * D * 2;
    const int state = kScoredRowWaves * heads * D * 4 + kScoredRowWaves * 16 * 8;
    return v > state ? v : state;
}

}  // namespace

template <int CT, int QT, int D, bool SCORES>
__global__ __launch_bounds__((64 * kMfmaMaxWaves<CT, D>)) __attribute__((amdgpu_waves_per_eu(kMfmaWaves<CT, QT, D>, 8)))
void paged_decode_scored(ScoredDecodeArgs a)
{
    __shared__ uint16_t s_v[kMfmaMaxWaves<CT, D> * kBlockSize * D];
    decode_wg<CT, QT, D, false, false, true, SCORES>(a, static_cast<int>(blockIdx.x), static_cast<int>(blockIdx.y),
                                             static_cast<int>(gridDim.x), static_cast<int>(blockDim.x) >> 6, s_v);
}

template <int CT, int QT, int D, bool SCORES>
__global__ __launch_bounds__(64 * kScoredRowWaves) __attribute__((amdgpu_waves_per_eu(2, 8)))
void paged_decode_scored_row(ScoredDecodeArgs a)
{
    extern __shared__ __align__(16) uint8_t s_scored_row[];
    decode_wg<CT, QT, D, false, true, true, SCORES>(a, static_cast<int>(blockIdx.y), static_cast<int>(blockIdx.x), 0,
                                            kScoredRowWaves, reinterpret_cast<uint16_t*>(s_scored_row));
}

namespace
{

template <int CT, int QT, int D>
int scored_items3(const ScoredDecodeArgs& a)
{
    const MfmaShape sh = mfma_shape<CT, D>(a);
    return decode_mfma_items(reinterpret_cast<const void*>(paged_decode_scored<CT, QT, D, false>), 64 * sh.nw, sh.gy);
}

template <int CT, int QT, int D, bool SCORES>
hipError_t launch_scored3(const ScoredDecodeArgs& a, bool row, hipStream_t stream)
{
    if (row)
    {
        const int  hb = (a.group + 15) / 16;
        const int  lds = scored_row_lds<D>(a.group < 16 ? a.group : 16);
        const dim3 grid(static_cast<unsigned>(a.num_kv_heads * hb), static_cast<unsigned>(a.batch));
        hipLaunchKernelGGL((paged_decode_scored_row<CT, QT, D, SCORES>), grid, dim3(64 * kScoredRowWaves), static_cast<unsigned>(lds),
                           stream, a);
        return hipGetLastError();
    }
    const MfmaShape sh = mfma_shape<CT, D>(a);
    hipLaunchKernelGGL((paged_decode_scored<CT, QT, D, SCORES>), dim3(static_cast<unsigned>(a.items), static_cast<unsigned>(sh.gy)),
                       dim3(64 * sh.nw), 0, stream, a);
    const hipError_t e = hipGetLastError();
    return e != hipSuccess ? e : launch_merge<QT, D, SCORES>(a, a.items, stream);
}

// f.operator()<CT, QT, D>() for the call's types and head_dim.
template <typename F>
auto scored_for(const ScoredDecodeArgs& a, F f)
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

}  // namespace

}  // namespace ffkv
