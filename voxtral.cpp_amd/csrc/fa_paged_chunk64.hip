// fa_paged_chunk64.hip — the chunk kernel of fa_paged_chunk.h at head dim 64.
#include "fa_paged_chunk.h"

namespace vxfa {

hipError_t launch_paged_chunk64(const PagedAttn& a, hipStream_t st) { return launch_chunk<64>(a, st); }

}  // namespace vxfa
