// paged_decode_scored.hip - the decode under a score rule (tanh cap, distance bias, window, first key), and the attention
// weights that it gives to the cached tokens.
//
// For the query of row b at position i = context_lens[b], head h and key j:
//   s_j = cap tanh(scale q.k_j / cap) - slope_h (i - j),   max(0, key_begin, i - window + 1) <= j <= i
//   out = sum_j softmax(s)_j v_j,   weights[b, kv head, j] = decay * prior[b, kv head, j] + sum over its heads of softmax(s)_j
//
// The attention is the plain decode's code (paged_decode_mfma.hip: decode_wg with RULE; its two forms, the split over all
// rows' pages and the workgroup per row and KV head).  It is bound by HBM, and the rule's few vector instructions per score
// run behind the loads.  A row's pages begin at its first visible key, so a window's pages are all that is read.
//
// The weights need every row's final maximum and denominator, which exist once its last piece is done.  Reading K a second
// time would cost half the call again; instead the decode writes the scores down as it has them (4 bytes per head and
// key, where the key's K and V are 4 * head_dim bytes per KV head: 3 % more traffic at four heads of 128 dims per KV head),
// and a second pass over them computes the weights.
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

template <int CT, int QT, int D>
__global__ __launch_bounds__((64 * kMfmaMaxWaves<CT, D>)) __attribute__((amdgpu_waves_per_eu(kMfmaWaves<CT, QT, D>, 8)))
void paged_decode_scored(DecodeArgs a)
{
    __shared__ uint16_t s_v[kMfmaMaxWaves<CT, D> * kBlockSize * D];
    decode_wg<CT, QT, D, false, false, true>(a, static_cast<int>(blockIdx.x), static_cast<int>(blockIdx.y),
                                             static_cast<int>(gridDim.x), static_cast<int>(blockDim.x) >> 6, s_v);
}

template <int CT, int QT, int D>
__global__ __launch_bounds__(64 * kScoredRowWaves) __attribute__((amdgpu_waves_per_eu(2, 8)))
void paged_decode_scored_row(DecodeArgs a)
{
    extern __shared__ __align__(16) uint8_t s_scored_row[];
    decode_wg<CT, QT, D, false, true, true>(a, static_cast<int>(blockIdx.y), static_cast<int>(blockIdx.x), 0,
                                            kScoredRowWaves, reinterpret_cast<uint16_t*>(s_scored_row));
}

// weights[b, kvh, j] of the tokens j of row b, one a thread: the scores of the KV head's query heads against their final
// maxima and denominators.  The row's own new token has no earlier weight.  Tokens at or past the row's end (or past
// max_context_len) are left alone.
__global__ __launch_bounds__(256) void paged_decode_weights(DecodeArgs a)
{
    const int     b = static_cast<int>(blockIdx.z);
    const int     kvh = static_cast<int>(blockIdx.y);
    const RowSpan s = row_span(a, b);
    const int     G = a.group;
    const float2* fin = reinterpret_cast<const float2*>(a.ws_final) + static_cast<int64_t>(b) * a.num_heads + kvh * G;
    const float*  sc = a.ws_scores + (static_cast<int64_t>(b) * a.num_heads + kvh * G) * a.score_stride;
    const int64_t at = (static_cast<int64_t>(b) * a.num_kv_heads + kvh) * a.weight_stride;
    for (int j = static_cast<int>(blockIdx.x * 256 + threadIdx.x); j < s.hi; j += static_cast<int>(gridDim.x * 256))
    {
        float w = 0.0f;
        if (j >= s.lo)
            for (int h = 0; h < G; ++h)
            {
                const float2 f = fin[h];
                const float  v = sc[h * a.score_stride + j];
                // (a key on no page weighs nothing, in a NaN query's row too)
                w += v == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(v - f.x) * softmax_inv(f.y);
            }
        if (a.prior != nullptr && j < s.pos) w = __builtin_fmaf(a.decay, a.prior[at + j], w);
        a.weights[at + j] = w;
    }
}

namespace
{

template <int CT, int QT, int D>
int scored_items3(const DecodeArgs& a)
{
    const MfmaShape sh = mfma_shape<CT, D>(a);
    return decode_mfma_items(reinterpret_cast<const void*>(paged_decode_scored<CT, QT, D>), 64 * sh.nw, sh.gy);
}

template <int CT, int QT, int D>
hipError_t launch_scored3(const DecodeArgs& a, bool row, hipStream_t stream)
{
    if (row)
    {
        const int  hb = (a.group + 15) / 16;
        const int  lds = scored_row_lds<D>(a.group < 16 ? a.group : 16);
        const dim3 grid(static_cast<unsigned>(a.num_kv_heads * hb), static_cast<unsigned>(a.batch));
        hipLaunchKernelGGL((paged_decode_scored_row<CT, QT, D>), grid, dim3(64 * kScoredRowWaves), static_cast<unsigned>(lds),
                           stream, a);
        return hipGetLastError();
    }
    const MfmaShape sh = mfma_shape<CT, D>(a);
    hipLaunchKernelGGL((paged_decode_scored<CT, QT, D>), dim3(static_cast<unsigned>(a.items), static_cast<unsigned>(sh.gy)),
                       dim3(64 * sh.nw), 0, stream, a);
    const hipError_t e = hipGetLastError();
    return e != hipSuccess ? e : launch_merge<QT, D, true>(a, a.items, stream);
}

// f.operator()<CT, QT, D>() for the call's types and head_dim.
template <typename F>
auto scored_for(const DecodeArgs& a, F f)
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

int decode_scored_launch_items(const DecodeArgs& a)
{
    return scored_for(a, [&]<int CT, int QT, int D>() { return scored_items3<CT, QT, D>(a); });
}

hipError_t launch_decode_weights(const DecodeArgs& a, hipStream_t stream)
{
    // enough workgroups for the longest row's tokens, up to 64 per (row, KV head): beyond that each takes several stretches
    const int64_t blocks = (static_cast<int64_t>(a.cap_tokens) + 255) / 256;
    const dim3    grid(static_cast<unsigned>(blocks < 1 ? 1 : (blocks > 64 ? 64 : blocks)),
                       static_cast<unsigned>(a.num_kv_heads), static_cast<unsigned>(a.batch));
    hipLaunchKernelGGL(paged_decode_weights, grid, dim3(256), 0, stream, a);
    return hipGetLastError();
}

hipError_t launch_decode_scored(const DecodeArgs& a, bool mfma, bool row, hipStream_t stream)
{
    const hipError_t e = mfma ? scored_for(a, [&]<int CT, int QT, int D>() { return launch_scored3<CT, QT, D>(a, row, stream); })
                              : launch_decode_scored_generic(a, stream);
    return e != hipSuccess || a.ws_scores == nullptr ? e : launch_decode_weights(a, stream);
}

}  // namespace ffkv
