// paged_append.hip -- a step's keys and values into their slots of a paged
// cache [pages, kv heads, page size, head dim].
//
// A copy with at most one rounding.  A thread moves 8 elements of a token's keys
// and the same 8 of its values; consecutive threads take a token's row in
// order, so both sides run in whole lines.  Bound by HBM (8192 tokens of 8 heads
// of 128, f32 to f16, 101 MB: 15.9 us, 6.3 TB/s with part of the input cached),
// and by the launch where there are few tokens (64 tokens, bf16: 3.6 us).
#include "serving_device.h"

namespace lxq {
namespace {

// rows of k and v start anywhere
typedef uint32_t u4u __attribute__((ext_vector_type(4), aligned(2)));
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

// AWAY: past the caches
template <bool AWAY>
__device__ __forceinline__ void put(void* p, u4 v) {
    if constexpr (AWAY) __builtin_nontemporal_store(v, static_cast<u4*>(p));
    else *static_cast<u4*>(p) = v;
}

// 8 elements from -> to
template <int IN, int OUT, bool AWAY>
__device__ __forceinline__ void move8(const void* from, int64_t i, void* to, int64_t o) {
    constexpr int ES = OUT == DT_F32 ? 4 : 2;
    char* dst = static_cast<char*>(to) + o * ES;
    if constexpr (IN != DT_F32 && IN == OUT) {
        put<AWAY>(dst, *reinterpret_cast<const u4u*>(static_cast<const uint16_t*>(from) + i));
    } else {
        float v[8];
        if constexpr (IN == DT_F32) {
            const f4u a = *reinterpret_cast<const f4u*>(static_cast<const float*>(from) + i);
            const f4u b = *reinterpret_cast<const f4u*>(static_cast<const float*>(from) + i + 4);
#pragma unroll
            for (int e = 0; e < 4; e++) { v[e] = a[e]; v[4 + e] = b[e]; }
        } else {
            const u4u a = *reinterpret_cast<const u4u*>(static_cast<const uint16_t*>(from) + i);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const uint32_t h = (a[e / 2] >> (16 * (e % 2))) & 0xffffu;
                v[e] = IN == DT_F16 ? f16_to_f32(h) : bf16_to_f32(h);
            }
        }
        if constexpr (OUT == DT_F32) {
            u4 a, b;
#pragma unroll
            for (int e = 0; e < 4; e++) { a[e] = __float_as_uint(v[e]); b[e] = __float_as_uint(v[4 + e]); }
            put<AWAY>(dst, a);
            put<AWAY>(dst + 16, b);
        } else {
            u4 a;
#pragma unroll
            for (int e = 0; e < 4; e++) a[e] = pack2<OUT>(v[2 * e], v[2 * e + 1]);
            put<AWAY>(dst, a);
        }
    }
}

// page of a slot, -1 where the token is left out
__device__ __forceinline__ int page_of(const AppendArgs& a, int slot) {
    const int page = slot < 0 ? -1 : div_by(slot, a.div);
    return page < a.pool ? page : -1;
}

// `per` tokens per block, `vecs` vectors of 8 per token: 256 / vecs tokens, or
// one in several rounds
template <int IN, int OUT, bool AWAY>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a, int first, int vecs, int per, int vecs_of_head) {
    const int mine = vecs < 256 ? (int)threadIdx.x / vecs : 0;
    const int64_t t = (int64_t)(first + (int)blockIdx.x) * per + mine;
    if (mine >= per || t >= a.T) return;
    const int slot = a.slots[t], page = page_of(a, slot);
    if (page < 0) return;
    const int at = slot - page * a.page;
    for (int i = (int)threadIdx.x - mine * vecs; i < vecs; i += 256) {
        const int h = i / vecs_of_head;
        const int64_t to = (((int64_t)page * a.Hk + h) * a.page + at) * a.D + (i - h * vecs_of_head) * 8;
        move8<IN, OUT, AWAY>(a.k, t * a.k_row + i * 8, a.kc, to);
        move8<IN, OUT, AWAY>(a.v, t * a.v_row + i * 8, a.vc, to);
    }
}

// head_dim no multiple of 8, or a cache that starts off 16 bytes: one element per thread
template <int IN, int OUT>
__global__ __launch_bounds__(256) void append_any_kernel(AppendArgs a, int first) {
    const int row = a.Hk * a.D, t = first + (int)blockIdx.x;
    const int slot = a.slots[t], page = page_of(a, slot);
    if (page < 0) return;
    const int at = slot - page * a.page;
    for (int i = (int)threadIdx.x; i < row; i += 256) {
        const int h = i / a.D;
        const int64_t to = (((int64_t)page * a.Hk + h) * a.page + at) * a.D + (i - h * a.D);
        store_f(a.kc, to, OUT, load_f(a.k, t * a.k_row + i, IN));
        store_f(a.vc, to, OUT, load_f(a.v, t * a.v_row + i, IN));
    }
}

template <int IN, int OUT>
void launch(const AppendArgs& a, hipStream_t st) {
    const int row = a.Hk * a.D;
    if (a.D % 8 || (reinterpret_cast<uintptr_t>(a.kc) | reinterpret_cast<uintptr_t>(a.vc)) % 16) {
        launch_blocks(a.T, 256, [&](int first, unsigned n) {
            hipLaunchKernelGGL((append_any_kernel<IN, OUT>), dim3(n), dim3(256), 0, st, a, first);
        });
        return;
    }
    const int vecs = row / 8, per = vecs < 256 ? 256 / vecs : 1;
    // 16-bit results that the L2s (32 MB) cannot hold leave past the caches (8192
    // tokens of 8 heads of 128, f32 to f16 16.0 us, 18.0 with plain stores); the
    // two stores of 8 f32 values are half lines, which costs more than it gains
    // (8192 tokens of 16 heads of 128 54.3 us plain, 66.8 so)
    const bool away = OUT != DT_F32 && (int64_t)a.T * row * 4 >= (32 << 20);
    launch_blocks(((int64_t)a.T + per - 1) / per, 256, [&](int first, unsigned n) {
        if (away) hipLaunchKernelGGL((append_kernel<IN, OUT, OUT != DT_F32>), dim3(n), dim3(256), 0, st, a, first, vecs, per, a.D / 8);
        else hipLaunchKernelGGL((append_kernel<IN, OUT, false>), dim3(n), dim3(256), 0, st, a, first, vecs, per, a.D / 8);
    });
}
template <int IN>
void launch_in(const AppendArgs& a, hipStream_t st) {
    if (a.cache_dt == DT_F32) launch<IN, DT_F32>(a, st);
    else if (a.cache_dt == DT_F16) launch<IN, DT_F16>(a, st);
    else launch<IN, DT_BF16>(a, st);
}

}  // namespace

LuxStatus launch_paged_append(const AppendArgs& a, hipStream_t st) {
    if (a.in_dt == DT_F32) launch_in<DT_F32>(a, st);
    else if (a.in_dt == DT_F16) launch_in<DT_F16>(a, st);
    else launch_in<DT_BF16>(a, st);
    return hipGetLastError() == hipSuccess ? LuxStatus::Ok : LuxStatus::Internal;
}

}  // namespace lxq
