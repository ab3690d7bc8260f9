// paged_chunk.hip -- chunk attention: the types
#include "paged_chunk.h"

namespace lxq {

LuxStatus launch_paged_chunk(const ChunkArgs& a, hipStream_t st) {
    if (a.dtype == DT_F32) return chunk::launch_t<DT_F32>(a, st);
    return a.dtype == DT_F16 ? chunk::launch_t<DT_F16>(a, st) : chunk::launch_t<DT_BF16>(a, st);
}

}  // namespace lxq
