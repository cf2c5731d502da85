// fa_paged_chunk_q8.hip — the chunk kernel of fa_paged_chunk.h over pages of 8 bits at head
// dim 128, and the choice between the two.
#include "fa_paged_chunk.h"

namespace vxfa {

hipError_t launch_paged_chunk_q8(const PagedAttn& a, const PagedScales& sc, int head_dim, hipStream_t st) {
    if (head_dim == 128) return launch_chunk<128, true>(a, &sc, st);
    if (head_dim == 64) return launch_paged_chunk64_q8(a, sc, st);
    return hipErrorInvalidValue;
}

}  // namespace vxfa
