// paged_blocks_prefill_fp8.hip - the prefill over listed pages (blocks_prefill.h) of fp8 caches.
#include "blocks_prefill.h"

namespace ffkv
{

void       plan_blocks_prefill_fp8(ListPrefillArgs& a) { plan_blocks_prefill_t<FP8>(a); }
hipError_t launch_blocks_prefill_fp8(const ListPrefillArgs& a, hipStream_t stream) { return launch_blocks_prefill_t<FP8>(a, stream); }

}  // namespace ffkv
