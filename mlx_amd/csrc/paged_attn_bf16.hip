// explicit instantiation: paged attention, bf16
#include "paged_attn.h"
namespace lxq {
namespace attn {
template LuxStatus launch_t<DT_BF16>(const AttnArgs&, hipStream_t);
}  // namespace attn
}  // namespace lxq
