// paged_blocks_prefill_bf16.hip - the prefill over listed pages (blocks_prefill.h) of bf16 caches.
#include "blocks_prefill.h"

namespace ffkv
{

void       plan_blocks_prefill_bf16(ListPrefillArgs& a) { plan_blocks_prefill_t<BF16>(a); }
hipError_t launch_blocks_prefill_bf16(const ListPrefillArgs& a, hipStream_t stream) { return launch_blocks_prefill_t<BF16>(a, stream); }

}  // namespace ffkv
