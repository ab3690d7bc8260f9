// paged_chunk_f32.hip -- chunk attention, f32
#include "paged_chunk.h"

namespace lxq {
template LuxStatus chunk::launch_t<DT_F32>(const ChunkArgs&, hipStream_t);
}  // namespace lxq
