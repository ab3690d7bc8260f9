// explicit instantiation: paged attention, f32
#include "paged_attn.h"
namespace lxq {
namespace attn {
template LuxStatus launch_t<DT_F32>(const AttnArgs&, hipStream_t);
}  // namespace attn
}  // namespace lxq
