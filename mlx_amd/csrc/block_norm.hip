// block_norm.hip -- what stands between two blocks, in one pass:
//   h = rscale * r + gate * post(x),   out = pre(h)
// with post and pre RMS or layer norms (or none).
//
// A row stays in registers from its load to its two stores: the NT threads of a
// block hold 8 * V of its values each, so the means and mean squares cost one
// reduction each and no second read.  A layer norm takes the mean first and then the
// mean square of what is left.  Bound by HBM at many rows (8192 of 4096 bf16 with
// a post norm and the residual, 268 MB: 52.8 us, 5.1 TB/s), by the two
// reductions and the launch at one (4096 f16: 3.9 us).
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
// AWAY: past the caches
template <bool AWAY, class P>
__device__ __forceinline__ void put(void* p, P v) {
    if constexpr (AWAY) __builtin_nontemporal_store(v, static_cast<P*>(p));
    else *static_cast<P*>(p) = v;
}
template <int DT, bool AWAY>
__device__ __forceinline__ void store8(void* p, int64_t i, const float* v) {
    if constexpr (DT == DT_F32) {
        put<AWAY>(static_cast<float*>(p) + i, f4u{v[0], v[1], v[2], v[3]});
        put<AWAY>(static_cast<float*>(p) + i + 4, f4u{v[4], v[5], v[6], v[7]});
    } else {
        u4u a;
#pragma unroll
        for (int e = 0; e < 4; e++) a[e] = pack2<DT>(v[2 * e], v[2 * e + 1]);
        put<AWAY>(static_cast<uint16_t*>(p) + i, a);
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
template <int DT, bool AWAY>
__device__ __forceinline__ void store_part(void* p, int64_t i, int n, const float* v) {
    if (n >= 8) {
        store8<DT, AWAY>(p, i, v);
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

// the sum over a block of up to 16 waves
template <int NT>
__device__ __forceinline__ float block_sum(float v, float* part) {
    v = wave_sum(v);
    constexpr int waves = NT / 64;
    const int lane = threadIdx.x & 63;
    if constexpr (waves > 1) {
        __syncthreads();  // the last sum's readers
        if (lane == 0) part[threadIdx.x >> 6] = v;
        __syncthreads();
        v = row16_sum(lane < waves ? part[lane] : 0.f);
        v = lane_f(v, 0);
    }
    return v;
}

// v - mean, and what its mean square scales it by; elements past the row stay 0
template <int NT, int V>
__device__ __forceinline__ float center(float (*v)[8], const int* n, int kind, float inv_d, float eps, float* part) {
    if (kind == NORM_LAYER) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < V; i++)
#pragma unroll
            for (int e = 0; e < 8; e++) s += v[i][e];
        const float mean = block_sum<NT>(s, part) * inv_d;
#pragma unroll
        for (int i = 0; i < V; i++)
#pragma unroll
            for (int e = 0; e < 8; e++) v[i][e] = e < n[i] ? v[i][e] - mean : 0.f;
    }
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < V; i++)
#pragma unroll
        for (int e = 0; e < 8; e++) q = fmaf(v[i][e], v[i][e], q);
    return 1.f / sqrtf(block_sum<NT>(q, part) * inv_d + eps);
}

// v = norm(v) * weight + bias
template <int NT, int V>
__device__ __forceinline__ void normalize(float (*v)[8], const int* n, int kind, float inv_d, float eps, const void* w, const void* b,
                                          int w_dt, int col, float* part) {
    const float r = center<NT, V>(v, n, kind, inv_d, eps, part);
#pragma unroll
    for (int i = 0; i < V; i++) {
        if (n[i] <= 0) continue;
        const int c = col + i * NT * 8;
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; e++) v[i][e] *= r;
        if (w) {
            load_weight(w, c, n[i], w_dt, f);
#pragma unroll
            for (int e = 0; e < 8; e++) v[i][e] *= f[e];
        }
        if (b) {
            load_weight(b, c, n[i], w_dt, f);
#pragma unroll
            for (int e = 0; e < 8; e++) v[i][e] += f[e];
        }
    }
}

// a block per row
template <int NT, int V, bool AWAY, int XT, int RT>
__global__ __launch_bounds__(NT) void block_norm_kernel(NormArgs a, int first) {
    __shared__ float part[16];
    constexpr int hop = NT * 8;
    const int t = first + (int)blockIdx.x, col = (int)threadIdx.x * 8;
    const float inv_d = 1.f / (float)a.D;
    const bool gates = a.gate_mode == GATE_CHANNEL || a.gate_mode == GATE_FULL;
    const int64_t g_at = a.gate_mode == GATE_FULL ? t * a.g_row : 0;
    int n[V];
    float v[V][8];
#pragma unroll
    for (int i = 0; i < V; i++) {
        const int c = col + i * hop;
        n[i] = a.D - c;
        n[i] = n[i] > 8 ? 8 : n[i];
#pragma unroll
        for (int e = 0; e < 8; e++) v[i][e] = 0.f;
        if (a.x && n[i] > 0) load_part<XT>(a.x, t * a.x_row + c, n[i], v[i]);
    }
    const float row_gate = a.gate_mode == GATE_ROW ? load_f(a.gate, t * a.g_row, XT) : 1.f;
    if (a.post != NORM_NONE) normalize<NT, V>(v, n, a.post, inv_d, a.eps, a.pw, a.pb, a.w_dt, col, part);
#pragma unroll
    for (int i = 0; i < V; i++) {
        if (n[i] <= 0) continue;
        const int c = col + i * hop;
        float f[8];
        if (gates) {
            load_part<XT>(a.gate, g_at + c, n[i], f);
#pragma unroll
            for (int e = 0; e < 8; e++) v[i][e] *= f[e];
        } else if (a.gate_mode == GATE_ROW) {
#pragma unroll
            for (int e = 0; e < 8; e++) v[i][e] *= row_gate;
        }
        if (a.r) {
            load_part<RT>(a.r, t * a.r_row + c, n[i], f);
#pragma unroll
            for (int e = 0; e < 8; e++) v[i][e] = fmaf(f[e], a.rscale, v[i][e]);
        }
#pragma unroll
        for (int e = 0; e < 8; e++) v[i][e] = e < n[i] ? v[i][e] : 0.f;
        if (a.h) store_part<RT, AWAY>(a.h, t * a.h_row + c, n[i], v[i]);
    }
    if (!a.out) return;
    if (a.pre != NORM_NONE) normalize<NT, V>(v, n, a.pre, inv_d, a.eps, a.nw, a.nb, a.w_dt, col, part);
#pragma unroll
    for (int i = 0; i < V; i++)
        if (n[i] > 0) store_part<XT, AWAY>(a.out, t * a.o_row + col + i * hop, n[i], v[i]);
}

// Rows too long for the registers (past 32768): x and the residual are read again
// for each sum, out of the caches; h and out are written by the last pass.
template <int XT, int RT>
__global__ __launch_bounds__(1024) void block_norm_long_kernel(NormArgs a, int first) {
    constexpr int NT = 1024;
    __shared__ float part[16];
    const int t = first + (int)blockIdx.x;
    const float inv_d = 1.f / (float)a.D;
    const float row_gate = a.gate_mode == GATE_ROW ? load_f(a.gate, t * a.g_row, XT) : 1.f;
    float mean1 = 0.f, scale1 = 1.f;
    auto affine = [&](float* v, int c, int n, float mean, float scale, const void* w, const void* b) {
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = (v[e] - mean) * scale;
        if (w) {
            load_weight(w, c, n, a.w_dt, f);
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] *= f[e];
        }
        if (b) {
            load_weight(b, c, n, a.w_dt, f);
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] += f[e];
        }
    };
    auto x_at = [&](int c, int n, float* v) {
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = 0.f;
        if (a.x) load_part<XT>(a.x, t * a.x_row + c, n, v);
    };
    auto h_at = [&](int c, int n, float* v) {
        float f[8];
        x_at(c, n, v);
        if (a.post != NORM_NONE) affine(v, c, n, mean1, scale1, a.pw, a.pb);
        if (a.gate_mode == GATE_CHANNEL || a.gate_mode == GATE_FULL) {
            load_part<XT>(a.gate, (a.gate_mode == GATE_FULL ? t * a.g_row : 0) + c, n, f);
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] *= f[e];
        }
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] *= row_gate;
        if (a.r) {
            load_part<RT>(a.r, t * a.r_row + c, n, f);
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = fmaf(f[e], a.rscale, v[e]);
        }
    };
    // the mean, and what the mean square of the rest scales it by
    auto statistics = [&](int kind, float& mean, float& scale, auto at) {
        float v[8], s = 0.f;
        if (kind == NORM_LAYER) {
            for (int c = (int)threadIdx.x * 8; c < a.D; c += NT * 8) {
                const int n = a.D - c;
                at(c, n, v);
#pragma unroll
                for (int e = 0; e < 8; e++) s += e < n ? v[e] : 0.f;
            }
            mean = block_sum<NT>(s, part) * inv_d;
        }
        s = 0.f;
        for (int c = (int)threadIdx.x * 8; c < a.D; c += NT * 8) {
            const int n = a.D - c;
            at(c, n, v);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float d = e < n ? v[e] - mean : 0.f;
                s = fmaf(d, d, s);
            }
        }
        scale = 1.f / sqrtf(block_sum<NT>(s, part) * inv_d + a.eps);
    };
    if (a.post != NORM_NONE) statistics(a.post, mean1, scale1, x_at);
    float mean2 = 0.f, scale2 = 1.f;
    if (a.out && a.pre != NORM_NONE) statistics(a.pre, mean2, scale2, h_at);
    for (int c = (int)threadIdx.x * 8; c < a.D; c += NT * 8) {
        const int n = a.D - c;
        float v[8];
        h_at(c, n, v);
        if (a.h) store_part<RT, false>(a.h, t * a.h_row + c, n, v);
        if (!a.out) continue;
        if (a.pre != NORM_NONE) affine(v, c, n, mean2, scale2, a.nw, a.nb);
        store_part<XT, false>(a.out, t * a.o_row + c, n, v);
    }
}

// NT threads and V vectors of 8 per thread; NT = 0: the long form
template <int NT, int V, bool AWAY, int XT, int RT>
void launch_xr(const NormArgs& a, hipStream_t st) {
    launch_blocks(a.T, NT ? NT : 1024, [&](int first, unsigned n) {
        if constexpr (NT == 0) hipLaunchKernelGGL((block_norm_long_kernel<XT, RT>), dim3(n), dim3(1024), 0, st, a, first);
        else hipLaunchKernelGGL((block_norm_kernel<NT, V, AWAY, XT, RT>), dim3(n), dim3(NT), 0, st, a, first);
    });
}
template <int NT, int V, bool AWAY, int XT>
void launch_x(const NormArgs& a, hipStream_t st) {
    if (a.r_dt == DT_F32) launch_xr<NT, V, AWAY, XT, DT_F32>(a, st);
    else if (a.r_dt == DT_F16) launch_xr<NT, V, AWAY, XT, DT_F16>(a, st);
    else launch_xr<NT, V, AWAY, XT, DT_BF16>(a, st);
}
template <int NT, int V, bool AWAY>
LuxStatus launch(const NormArgs& a, hipStream_t st) {
    if (a.x_dt == DT_F32) launch_x<NT, V, AWAY, DT_F32>(a, st);
    else if (a.x_dt == DT_F16) launch_x<NT, V, AWAY, DT_F16>(a, st);
    else launch_x<NT, V, AWAY, DT_BF16>(a, st);
    return hipGetLastError() == hipSuccess ? LuxStatus::Ok : LuxStatus::Internal;
}

// many rows: by the vectors of 8 in a row
template <bool AWAY>
LuxStatus launch_many(const NormArgs& a, int v, hipStream_t st) {
    if (v <= 64) return launch<64, 1, AWAY>(a, st);
    if (v <= 64 * 2) return launch<64, 2, AWAY>(a, st);
    if (v <= 128 * 2) return launch<128, 2, AWAY>(a, st);
    if (v <= 128 * 3) return launch<128, 3, AWAY>(a, st);
    if (v <= 256 * 2 && a.x_dt != DT_F32) return launch<256, 2, AWAY>(a, st);
    if (v <= 512) return launch<512, 1, AWAY>(a, st);
    if (v <= 256 * 3) return launch<256, 3, AWAY>(a, st);
    if (v <= 512 * 2) return launch<512, 2, AWAY>(a, st);
    if (v <= 512 * 3) return launch<512, 3, AWAY>(a, st);
    return launch<1024, 2, AWAY>(a, st);
}

}  // namespace

// Threads per row and vectors of 8 per thread.  Up to two rows per CU each
// trip to memory shows, and more threads shorten it (64 rows of 4096 bf16: 256
// x 2 5.7 us, 512 x 1 4.5; one row of 16384: 512 x 4 7.4, 1024 x 2 5.8).  With
// more rows the threads that a row leaves idle and those that a barrier holds
// cost more (8192 rows of 1024 bf16: 64 x 2 13.0, 128 x 1 14.9, 256 x 1 18.5; of
// 2100 f16: 128 x 3 43.9, 256 x 2 49.6; of 4096 bf16: 256 x 2 54.9, 512 x 1
// 56.2; of 4096 f32: 512 x 1 97, 256 x 2 104; 2048 rows of 16384 f16: 1024 x 2
// 63.7, 512 x 4 78).
// Results that the L2s (32 MB) cannot hold leave past the caches: 4096 rows of
// 4608 bf16 51.6 us with plain stores, 34.6 so, 8192 of 2100 f16 44.2 and 31.7,
// 8192 of 4096 bf16 54.4 and 53.5.
LuxStatus launch_block_norm(const NormArgs& a, hipStream_t st) {
    const int v = (a.D + 7) / 8;
    if (a.T > 512 && v <= 1024 * 2) {
        const int64_t each = (a.h ? (a.r_dt == DT_F32 ? 4 : 2) : 0) + (a.out ? (a.x_dt == DT_F32 ? 4 : 2) : 0);
        return each * a.T * a.D >= (32 << 20) ? launch_many<true>(a, v, st) : launch_many<false>(a, v, st);
    }
    if (v <= 64) return launch<64, 1, false>(a, st);
    if (v <= 512) return launch<512, 1, false>(a, st);
    if (v <= 1024) return launch<1024, 1, false>(a, st);
    if (v <= 1024 * 2) return launch<1024, 2, false>(a, st);
    if (v <= 1024 * 4) return launch<1024, 4, false>(a, st);
    return launch<0, 0, false>(a, st);
}

}  // namespace lxq
