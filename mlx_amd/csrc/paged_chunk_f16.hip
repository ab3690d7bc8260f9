// paged_chunk_f16.hip -- chunk attention, f16
#include "paged_chunk.h"

namespace lxq {
template LuxStatus chunk::launch_t<DT_F16>(const ChunkArgs&, hipStream_t);
}  // namespace lxq
