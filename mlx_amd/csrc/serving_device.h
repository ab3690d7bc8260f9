// serving_device.h -- device helpers that the kernels of decoding steps and prompts share.
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

// tanh(y) from z = 2 y log2 e: 1 - 2 / (1 + exp2(z)), off by 2^-22 at most.  Where y
// is small that is a large share of it, and times a large cap a large part of the
// score: there the series up to y^11, whose next term is below 2^-28 of y at 0.3.
__device__ __forceinline__ float tanh_of(float z) {
    const float far = fmaf(__builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z)), -2.f, 1.f);
    const float y = z * (0.5f * 0.69314718055994531f), q = y * y;
    float near = fmaf(q, -1382.f / 155925.f, 62.f / 2835.f);
    near = fmaf(q, near, -17.f / 315.f);
    near = fmaf(q, near, 2.f / 15.f);
    near = fmaf(q, near, -1.f / 3.f);
    return fabsf(y) < 0.3f ? fmaf(y * q, near, y) : far;
}

}  // namespace lxq
