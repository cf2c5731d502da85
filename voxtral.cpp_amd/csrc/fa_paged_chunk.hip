// fa_paged_chunk.hip — the chunk kernel of fa_paged_chunk.h at head dim 128, and
// the choice between the two.
#include "fa_paged_chunk.h"

namespace vxfa {

hipError_t launch_paged_chunk(const PagedAttn& a, int head_dim, hipStream_t st) {
    if (head_dim == 128) return launch_chunk<128, false>(a, nullptr, st);
    if (head_dim == 64) return launch_paged_chunk64(a, st);
    return hipErrorInvalidValue;
}

}  // namespace vxfa
