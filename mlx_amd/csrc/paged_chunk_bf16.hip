// paged_chunk_bf16.hip -- chunk attention, bf16
#include "paged_chunk.h"

namespace lxq {
template LuxStatus chunk::launch_t<DT_BF16>(const ChunkArgs&, hipStream_t);
}  // namespace lxq
