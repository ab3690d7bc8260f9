// paged_attn.hip -- dispatch of the paged attention (kernels in paged_attn.h,
// one translation unit per type: paged_attn_{f32,f16,bf16}.hip).
#include "paged_attn.h"

namespace lxq {

LuxStatus launch_paged_attention(const AttnArgs& a, hipStream_t st) {
    switch (a.dtype) {
    case DT_F32: return attn::launch_t<DT_F32>(a, st);
    case DT_F16: return attn::launch_t<DT_F16>(a, st);
    case DT_BF16: return attn::launch_t<DT_BF16>(a, st);
    default: return LuxStatus::NotSupported;
    }
}

}  // namespace lxq
