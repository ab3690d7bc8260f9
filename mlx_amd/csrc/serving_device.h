// serving_device.h -- device helpers that the decoding step's kernels share.
#pragma once
#include "qcommon.h"
#include "serving.h"

namespace lxq {

__device__ __forceinline__ int div_by(int t, const DivBy& d) { return (int)(((uint64_t)(uint32_t)t * d.mul) >> (31 + d.sh)); }

// inclusive sum over the wave's lanes: shifts within rows of 16, then each
// row's last lane to the rows behind it
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_add(int v) {
    return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ int wave_scan(int v) {
    v = dpp_add<0x111, 0xF>(v);  // row_shr:1, 2, 4, 8
    v = dpp_add<0x112, 0xF>(v);
    v = dpp_add<0x114, 0xF>(v);
    v = dpp_add<0x118, 0xF>(v);
    v = dpp_add<0x142, 0xA>(v);     // row_bcast:15 into rows 1 and 3
    return dpp_add<0x143, 0xC>(v);  // row_bcast:31 into rows 2 and 3
}

}  // namespace lxq
