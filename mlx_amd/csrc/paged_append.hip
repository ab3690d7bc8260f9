// paged_append.hip -- a step's keys and values into their slots of a paged
// cache [pages, kv heads, page size, head dim].
//
// A copy with at most one rounding: a thread moves one vector of a token's row
// of keys and the same one of its values.  Bound by HBM.
#include "qcommon.h"
#include "serving.h"

namespace lxq {
namespace {

// N elements from p (aligned to its elements only) as fp32
template <int DT, int N>
__device__ __forceinline__ void load_n(const void* p, int64_t i, float* v) {
    if constexpr (DT == DT_F32) {
#pragma unroll
        for (int e = 0; e < N; e++) v[e] = static_cast<const float*>(p)[i + e];
    } else {
#pragma unroll
        for (int e = 0; e < N; e++) {
            const uint32_t h = static_cast<const uint16_t*>(p)[i + e];
            v[e] = DT == DT_F16 ? f16_to_f32(h) : bf16_to_f32(h);
        }
    }
}

// one thread per element: the form that is right for every shape
template <int IN, int OUT>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
    const int64_t row = (int64_t)a.Hk * a.D;
    const int t = blockIdx.x;
    const int slot = a.slots[t];
    const int page = (int)(((uint64_t)(uint32_t)(slot < 0 ? 0 : slot) * a.div.mul) >> (31 + a.div.sh));
    if (slot < 0 || page >= a.pool) return;
    const int at = slot - page * a.page;
    for (int i = (int)threadIdx.x; i < row; i += 256) {
        const int h = i / a.D, d = i - h * a.D;
        const int64_t to = (((int64_t)page * a.Hk + h) * a.page + at) * a.D + d;
        float v[1];
        load_n<IN, 1>(a.k, t * a.k_row + i, v);
        store_f(a.kc, to, OUT, v[0]);
        load_n<IN, 1>(a.v, t * a.v_row + i, v);
        store_f(a.vc, to, OUT, v[0]);
    }
}

template <int IN>
void launch_in(const AppendArgs& a, hipStream_t st) {
    const dim3 g(a.T), b(256);
    if (a.cache_dt == DT_F32) hipLaunchKernelGGL((append_kernel<IN, DT_F32>), g, b, 0, st, a);
    else if (a.cache_dt == DT_F16) hipLaunchKernelGGL((append_kernel<IN, DT_F16>), g, b, 0, st, a);
    else hipLaunchKernelGGL((append_kernel<IN, DT_BF16>), g, b, 0, st, a);
}

}  // namespace

LuxStatus launch_paged_append(const AppendArgs& a, hipStream_t st) {
    if (a.in_dt == DT_F32) launch_in<DT_F32>(a, st);
    else if (a.in_dt == DT_F16) launch_in<DT_F16>(a, st);
    else launch_in<DT_BF16>(a, st);
    return hipGetLastError() == hipSuccess ? LuxStatus::Ok : LuxStatus::Internal;
}

}  // namespace lxq
