// explicit instantiation: paged attention, f16
#include "paged_attn.h"
namespace lxq {
namespace attn {
template LuxStatus launch_t<DT_F16>(const AttnArgs&, hipStream_t);
}  // namespace attn
}  // namespace lxq
