// fa_paged_chunk64_q8.hip — the chunk kernel of fa_paged_chunk.h over pages of 8 bits at head dim 64.
#include "fa_paged_chunk.h"

namespace vxfa {

hipError_t launch_paged_chunk64_q8(const PagedAttn& a, const PagedScales& sc, hipStream_t st) { return launch_chunk<64, true>(a, &sc, st); }

}  // namespace vxfa
