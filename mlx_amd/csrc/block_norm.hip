// block_norm.hip -- what stands between two blocks, in one pass:
//   h = rscale * r + gate * post(x),   out = pre(h)
// with post and pre RMS or layer norms (or none).
//
// A row stays in registers from its load to its two stores: NT threads hold 8
// * V of its values each, so the means and mean squares cost one reduction
// each and no second read.  A layer norm takes the mean first and then the
// mean square of what is left.  Bound by HBM at many rows, by the two
// reductions and the launch at one.
#include "qcommon.h"
#include "serving.h"

namespace lxq {
namespace {

enum : int { NORM_NONE = 0, NORM_RMS = 1, NORM_LAYER = 2 };
enum : int { GATE_NONE = 0, GATE_CHANNEL = 1, GATE_ROW = 2, GATE_FULL = 3 };

// 8 elements at p, which is aligned to its elements only (rows of any length
// and stride): gfx950's global loads take any address
typedef uint32_t u4u __attribute__((ext_vector_type(4), aligned(2)));
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));

template <int DT>
__device__ __forceinline__ void load8(const void* p, int64_t i, float* v) {
    if constexpr (DT == DT_F32) {
        const f4u a = *reinterpret_cast<const f4u*>(static_cast<const float*>(p) + i);
        const f4u b = *reinterpret_cast<const f4u*>(static_cast<const float*>(p) + i + 4);
#pragma unroll
        for (int e = 0; e < 4; e++) { v[e] = a[e]; v[4 + e] = b[e]; }
    } else {
        const u4u a = *reinterpret_cast<const u4u*>(static_cast<const uint16_t*>(p) + i);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const uint32_t h = (a[e / 2] >> (16 * (e % 2))) & 0xffffu;
            v[e] = DT == DT_F16 ? f16_to_f32(h) : bf16_to_f32(h);
        }
    }
}
template <int DT>
__device__ __forceinline__ void store8(void* p, int64_t i, const float* v) {
    if constexpr (DT == DT_F32) {
        *reinterpret_cast<f4u*>(static_cast<float*>(p) + i) = f4u{v[0], v[1], v[2], v[3]};
        *reinterpret_cast<f4u*>(static_cast<float*>(p) + i + 4) = f4u{v[4], v[5], v[6], v[7]};
    } else {
        u4u a;
#pragma unroll
        for (int e = 0; e < 4; e++) a[e] = pack2<DT>(v[2 * e], v[2 * e + 1]);
        *reinterpret_cast<u4u*>(static_cast<uint16_t*>(p) + i) = a;
    }
}

// n (1..8) of 8 elements; the others are 0
template <int DT>
__device__ __forceinline__ void load_part(const void* p, int64_t i, int n, float* v) {
    if (n >= 8) {
        load8<DT>(p, i, v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = e < n ? load_f(p, i + e, DT) : 0.f;
    }
}
template <int DT>
__device__ __forceinline__ void store_part(void* p, int64_t i, int n, const float* v) {
    if (n >= 8) {
        store8<DT>(p, i, v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (e < n) store_f(p, i + e, DT, v[e]);
    }
}
__device__ __forceinline__ void load_weight(const void* p, int64_t i, int n, int dt, float* v) {
    if (dt == DT_F32) load_part<DT_F32>(p, i, n, v);
    else if (dt == DT_F16) load_part<DT_F16>(p, i, n, v);
    else load_part<DT_BF16>(p, i, n, v);
}

// the sum over the NT threads of a row
template <int NT>
__device__ __forceinline__ float row_sum(float v, float* part) {
    v = wave_sum(v);
    if constexpr (NT > 64) {
        __syncthreads();  // the last sum's readers
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int i = 0; i < NT / 64; i++) v += part[i];
    }
    return v;
}

// v = norm(v) * weight + bias; elements past the row stay 0 until the last line
template <int NT, int V>
__device__ __forceinline__ void normalize(float (*v)[8], const int* n, int kind, float inv_d, float eps, const void* w,
                                          const void* b, int w_dt, int col, float* part) {
    float mean = 0.f;
    if (kind == NORM_LAYER) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < V; i++)
#pragma unroll
            for (int e = 0; e < 8; e++) s += v[i][e];
        mean = row_sum<NT>(s, part) * inv_d;
    }
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < V; i++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
            if (kind == NORM_LAYER) v[i][e] = e < n[i] ? v[i][e] - mean : 0.f;
            q = fmaf(v[i][e], v[i][e], q);
        }
    const float r = 1.f / sqrtf(row_sum<NT>(q, part) * inv_d + eps);
#pragma unroll
    for (int i = 0; i < V; i++) {
        if (n[i] <= 0) continue;
        float f[8], g[8];
#pragma unroll
        for (int e = 0; e < 8; e++) { f[e] = 1.f; g[e] = 0.f; }
        if (w) load_weight(w, col + i * NT * 8, n[i], w_dt, f);
        if (b) load_weight(b, col + i * NT * 8, n[i], w_dt, g);
#pragma unroll
        for (int e = 0; e < 8; e++) v[i][e] = fmaf(v[i][e] * r, f[e], g[e]);
    }
}

// NT threads per row, 256 / NT rows per block where NT < 256
template <int NT, int V, int XT, int RT>
__global__ __launch_bounds__(NT < 256 ? 256 : NT) void block_norm_kernel(NormArgs a) {
    __shared__ float part[NT / 64];
    constexpr int kRows = NT < 256 ? 256 / NT : 1;
    static_assert(NT == 64 || NT >= 256, "a wave or a block per row");
    const int t = (int)blockIdx.x * kRows + (kRows > 1 ? (int)threadIdx.x / NT : 0);
    if (kRows > 1 && t >= a.T) return;
    const int col = (kRows > 1 ? (int)threadIdx.x % NT : (int)threadIdx.x) * 8;
    const float inv_d = 1.f / (float)a.D;
    int n[V];
    float v[V][8];
#pragma unroll
    for (int i = 0; i < V; i++) {
        n[i] = a.D - (col + i * NT * 8);
        n[i] = n[i] > 8 ? 8 : n[i];
#pragma unroll
        for (int e = 0; e < 8; e++) v[i][e] = 0.f;
        if (a.x && n[i] > 0) load_part<XT>(a.x, t * a.x_row + col + i * NT * 8, n[i], v[i]);
    }
    if (a.post != NORM_NONE) normalize<NT, V>(v, n, a.post, inv_d, a.eps, a.pw, a.pb, a.w_dt, col, part);
    const float row_gate = a.gate_mode == GATE_ROW ? load_f(a.gate, t * a.g_row, XT) : 1.f;
#pragma unroll
    for (int i = 0; i < V; i++) {
        if (n[i] <= 0) continue;
        const int c = col + i * NT * 8;
        if (a.gate_mode == GATE_CHANNEL || a.gate_mode == GATE_FULL) {
            float g[8];
            load_part<XT>(a.gate, (a.gate_mode == GATE_FULL ? t * a.g_row : 0) + c, n[i], g);
#pragma unroll
            for (int e = 0; e < 8; e++) v[i][e] *= g[e];
        } else if (a.gate_mode == GATE_ROW) {
#pragma unroll
            for (int e = 0; e < 8; e++) v[i][e] *= row_gate;
        }
        if (a.r) {
            float r[8];
            load_part<RT>(a.r, t * a.r_row + c, n[i], r);
#pragma unroll
            for (int e = 0; e < 8; e++) v[i][e] = fmaf(r[e], a.rscale, v[i][e]);
        }
#pragma unroll
        for (int e = 0; e < 8; e++) v[i][e] = e < n[i] ? v[i][e] : 0.f;
        if (a.h) store_part<RT>(a.h, t * a.h_row + c, n[i], v[i]);
    }
    if (!a.out) return;
    if (a.pre != NORM_NONE) normalize<NT, V>(v, n, a.pre, inv_d, a.eps, a.nw, a.nb, a.w_dt, col, part);
#pragma unroll
    for (int i = 0; i < V; i++)
        if (n[i] > 0) store_part<XT>(a.out, t * a.o_row + col + i * NT * 8, n[i], v[i]);
}

template <int NT, int V, int XT>
void launch_x(const NormArgs& a, hipStream_t st) {
    const int rows = NT < 256 ? 256 / NT : 1;
    const dim3 g((a.T + rows - 1) / rows), b(NT < 256 ? 256 : NT);
    if (a.r_dt == DT_F32) hipLaunchKernelGGL((block_norm_kernel<NT, V, XT, DT_F32>), g, b, 0, st, a);
    else if (a.r_dt == DT_F16) hipLaunchKernelGGL((block_norm_kernel<NT, V, XT, DT_F16>), g, b, 0, st, a);
    else hipLaunchKernelGGL((block_norm_kernel<NT, V, XT, DT_BF16>), g, b, 0, st, a);
}
template <int NT, int V>
void launch(const NormArgs& a, hipStream_t st) {
    if (a.x_dt == DT_F32) launch_x<NT, V, DT_F32>(a, st);
    else if (a.x_dt == DT_F16) launch_x<NT, V, DT_F16>(a, st);
    else launch_x<NT, V, DT_BF16>(a, st);
}

}  // namespace

LuxStatus launch_block_norm(const NormArgs& a, hipStream_t st) {
    if (a.D <= 512) launch<64, 1>(a, st);
    else if (a.D <= 2048) launch<256, 1>(a, st);
    else if (a.D <= 4096) launch<256, 2>(a, st);
    else if (a.D <= 8192) launch<256, 4>(a, st);
    else if (a.D <= 16384) launch<512, 4>(a, st);
    else if (a.D <= 32768) launch<1024, 4>(a, st);
    else launch<1024, 8>(a, st);
    return hipGetLastError() == hipSuccess ? LuxStatus::Ok : LuxStatus::Internal;
}

}  // namespace lxq
