// paged_prefill_scored_split.hip - the scored prefill split over its keys (prefill_wg with SPLIT), and its plan.
#include "prefill_scored.h"

namespace ffkv
{

void prefill_scored_plan(ScoredPrefillArgs& a)
{
    prefill_for(a, [&]<int QT, int D, int CT, int RG>()
    {
        prefill_plan_for(a, reinterpret_cast<const void*>(paged_prefill_scored<QT, D, CT, RG, true>), 512 / RG,
                         DmaCfg<D, kElemBytes<CT>, CT == I8, 8 / RG, false>::KP * kBlockSize, a.span_tokens);
    });
}

hipError_t launch_prefill_scored_pieces(const ScoredPrefillArgs& a, unsigned wgs, hipStream_t stream)
{
    return launch_scored<true>(a, wgs, stream);
}

}  // namespace ffkv
