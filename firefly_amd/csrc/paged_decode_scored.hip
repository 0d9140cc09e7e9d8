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
//
// Measured (32/8 heads of 128 dims, bf16): 64 rows of 512 to 4096 tokens behind a window of 1024, capped, 56 us (4.6 TB/s); 8
// rows of 32k f16 tokens, 28/4 heads, with a distance bias 93 us (5.8 TB/s); 64 rows of 512 to 4096 tokens with their weights 136 us
// (decode 120, merge 5, weights 9), 101 without, on int8 pages 92 and 73, on fp8 pages 81 and 69; 32 rows of 512 to 4096 fp32
// tokens (the vector kernel) 125; 4 rows of up to 255 tokens 7.6 us in one launch.
#include "decode_scored.h"

namespace ffkv
{

int decode_scored_launch_items(const ScoredDecodeArgs& a)
{
    return scored_for(a, [&]<int CT, int QT, int D>() { return scored_items3<CT, QT, D>(a); });
}

hipError_t launch_decode_scored(const ScoredDecodeArgs& a, bool mfma, bool row, hipStream_t stream)
{
    if (a.ws_scores == nullptr)
        return mfma ? scored_for(a, [&]<int CT, int QT, int D>() { return launch_scored3<CT, QT, D, false>(a, row, stream); })
                    : launch_decode_scored_generic(a, stream);
    const hipError_t e = mfma ? launch_decode_scores(a, row, stream) : launch_decode_scored_generic(a, stream);
    return e != hipSuccess ? e : launch_decode_weights(a, stream);
}

}  // namespace ffkv
