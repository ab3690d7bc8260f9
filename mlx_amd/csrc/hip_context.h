// hip_context.h -- the plugin's context and buffer records and the checks that
// its entry points share (hip_backend.hip, serving_ops.hip).
#pragma once
#include <hip/hip_runtime.h>

#include "../../include/lux_gpu_backend_abi.h"
#include "../../include/lux_gpu_prompt_backend.h"
#include "../../include/lux_gpu_serving_backend.h"
#include "prompt.h"

namespace lxh {

struct HipContext {
    int device = 0;
    hipStream_t stream = nullptr;
    char name[256] = {0};
    int compute_units = 0;
    int max_wg = 0;
    // kernel workspace (partial sums, tile counters and flags of the kernels
    // that split K: split-K small-M GEMM, group-wise GEMM, the large GEMMs' K
    // parts and split last round), allocated and zeroed once here so that no
    // launch allocates; used only by work on `stream`, which orders its users
    void* ws = nullptr;
    size_t ws_bytes = 0;
    // launches on ws so far: each GEMM launch gets the next number as its
    // epoch (the split tiles meet by it; never 0)
    uint32_t epoch = 0;
    // arrival counters of the attention's split pairs (three per range) and of the
    // parts of a row of logits (one per row), zero
    // between launches; without them neither is split
    void* counts = nullptr;
    // partial results of the chunk attention's split tiles, allocated by the first
    // one; like ws, used only by work on `stream`
    void* parts = nullptr;
};
constexpr int kCountWords = 2048;

struct HipBuffer {
    void* ptr = nullptr;
    size_t size = 0;
    bool owned = true;  // false: a view of memory that the caller frees
    size_t tail = lxq::kTailPad;  // readable bytes behind it (a view's: to its allocation's end)
};

inline HipContext* C(LuxBackendContext* c) { return reinterpret_cast<HipContext*>(c); }
inline HipBuffer* B(LuxBackendBuffer* b) { return reinterpret_cast<HipBuffer*>(b); }

inline LuxBackendError map_err(hipError_t e) {
    switch (e) {
    case hipSuccess: return LUX_BACKEND_OK;
    case hipErrorOutOfMemory: return LUX_BACKEND_ERROR_OUT_OF_MEMORY;
    case hipErrorInvalidValue: return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    case hipErrorNoDevice:
    case hipErrorInvalidDevice: return LUX_BACKEND_ERROR_DEVICE_LOST;
    default: return LUX_BACKEND_ERROR_INTERNAL;
    }
}

inline LuxBackendError map_status(lxq::LuxStatus s) {
    switch (s) {
    case lxq::LuxStatus::Ok: return LUX_BACKEND_OK;
    case lxq::LuxStatus::Invalid: return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    case lxq::LuxStatus::OutOfMemory: return LUX_BACKEND_ERROR_OUT_OF_MEMORY;
    case lxq::LuxStatus::NotSupported: return LUX_BACKEND_ERROR_NOT_SUPPORTED;
    default: return LUX_BACKEND_ERROR_INTERNAL;
    }
}

inline size_t dtype_size(int dt) { return dt == LUX_DTYPE_FLOAT32 ? 4 : 2; }
inline bool dtype_ok(int dt) {
    return dt == LUX_DTYPE_FLOAT32 || dt == LUX_DTYPE_FLOAT16 || dt == LUX_DTYPE_BFLOAT16;
}

inline bool fits(HipBuffer* b, size_t need) { return b && (need == 0 || (b->ptr && b->size >= need)); }
// an operand whose kernels take its first `need` bytes in vectors of `align`
// bytes and may read `past` bytes behind them: an allocation of the plugin's
// is made for that, a view may start and end anywhere
inline bool reaches(HipBuffer* b, size_t need, size_t align, size_t past) {
    if (!fits(b, need)) return false;
    return need == 0 || b->owned ||
           (reinterpret_cast<uintptr_t>(b->ptr) % align == 0 && b->size - need + b->tail >= past);
}
// operands of the quantized ops: those that they read in vectors, and those that
// they take element by element or in vectors that may start on any of `align` bytes
inline bool read_by(HipBuffer* b, size_t need) { return reaches(b, need, 16, lxq::kTailPad); }
inline bool taken_by(HipBuffer* b, size_t need, size_t align) { return reaches(b, need, align, 0); }

}  // namespace lxh

// the table of include/lux_gpu_serving_backend.h
const lux_gpu_serving_vtbl* lux_hip_serving_table();
// and of include/lux_gpu_prompt_backend.h
const lux_gpu_prompt_vtbl* lux_hip_prompt_table();
