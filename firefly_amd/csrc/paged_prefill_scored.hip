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
//
// Bound by vector work and matrix work that overlap in part, as the plain prefill; the cap adds eight vector instructions per
// score to the softmax's eight.  Measured (32/8 heads of 128 dims): 8 x 512 tokens over 2000 to 2900 cached ones behind a window
// of 1024 and a cap, bf16, 134 us (512 TFLOP/s of visible pairs); 2000 f16 tokens of several documents 25 to 46 us by the
// longest one (430 to 1050 tokens); 256 tokens over 7.9k on fp8 pages with a distance bias 60 us, split over the keys (8 of it the
// merge).
#include "prefill_scored.h"

namespace ffkv
{

hipError_t launch_prefill_scored(const ScoredPrefillArgs& a, hipStream_t stream)
{
    const bool    split = a.n_split > 1;
    const int64_t groups = static_cast<int64_t>(a.batch) * a.num_kv_heads * (split ? a.n_split : 1);
    const int64_t nrb = (static_cast<int64_t>(a.seq_len) * a.group + kDmaRows - 1) / kDmaRows;
    const int64_t wgs = (groups + kXcds - 1) / kXcds * kXcds * nrb;
    if (wgs <= 0) return hipSuccess;
    if (wgs > INT32_MAX) return hipErrorInvalidConfiguration;
    if (!split) return launch_scored<false>(a, static_cast<unsigned>(wgs), stream);
    const hipError_t e = launch_prefill_scored_pieces(a, static_cast<unsigned>(wgs), stream);
    return e != hipSuccess ? e : launch_prefill_merge(a, stream);
}

}  // namespace ffkv
