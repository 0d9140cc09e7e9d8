// paged_blocks_prefill_i8.hip - the prefill over listed pages (blocks_prefill.h) of i8 caches.
#include "blocks_prefill.h"

namespace ffkv
{

void       plan_blocks_prefill_i8(ListPrefillArgs& a) { plan_blocks_prefill_t<I8>(a); }
hipError_t launch_blocks_prefill_i8(const ListPrefillArgs& a, hipStream_t stream) { return launch_blocks_prefill_t<I8>(a, stream); }

}  // namespace ffkv
