// serving_ops.hip -- entry points of the decoding step's operators
// (include/lux_gpu_serving_backend.h): argument checks, then one launcher.
#include <new>

#include "extent.h"
#include "hip_context.h"
#include "serving.h"
#include "spans.h"

using namespace lxh;

namespace {

LuxBackendError op_paged_plan(LuxBackendContext* c, const lux_paged_plan_args* p) {
    HipContext* ctx = C(c);
    if (!ctx || !p || p->struct_size != sizeof(*p)) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    const int R = p->requests, T = p->max_tokens, cols = p->max_pages;
    if (R < 0 || T < 0 || cols <= 0 || p->page_size <= 0 || p->num_pages < 0 || p->free_count < 0)
        return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    if (!rows_ok(1, p->page_size, p->num_pages) || !rows_ok(1, p->page_size, cols) ||
        (int64_t)R * cols >= (1ll << 31) - 1)
        return LUX_BACKEND_ERROR_NOT_SUPPORTED;
    lxq::PlanArgs a;
    Spans s;
    const size_t r = (size_t)R * 4, t = (size_t)T * 4;
    a.seq = static_cast<const int32_t*>(s.in(p->seq_lens, 0, r, 4));
    a.fresh = static_cast<const int32_t*>(s.in(p->new_lens, 0, r, 4));
    a.free_pages = static_cast<const int32_t*>(s.in(p->free_pages, 0, (size_t)p->free_count * 4, 4));
    a.head = static_cast<const int32_t*>(s.in(p->free_head, 0, 4, 4));
    a.table = static_cast<int32_t*>(s.out(p->block_table, 0, r * cols, 4));
    a.slots = static_cast<int32_t*>(s.out(p->slots, 0, t, 4));
    a.positions = p->positions ? static_cast<int32_t*>(s.out(p->positions, 0, t, 4)) : nullptr;
    a.request = p->token_request ? static_cast<int32_t*>(s.out(p->token_request, 0, t, 4)) : nullptr;
    a.starts = static_cast<int32_t*>(s.out(p->token_starts, 0, r + 4, 4));
    a.lens = static_cast<int32_t*>(s.out(p->kv_lens, 0, r, 4));
    a.counts = static_cast<int32_t*>(s.out(p->counts, 0, 16, 4));
    if (!s.ok || !s.apart()) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    a.R = R; a.T = T; a.columns = cols; a.page = p->page_size; a.pool = p->num_pages; a.F = p->free_count;
    a.div = lxq::DivBy(p->page_size);
    a.ws = ctx->ws_bytes > lxq::kWorkspaceWords ? reinterpret_cast<int32_t*>(static_cast<char*>(ctx->ws) + lxq::kWorkspaceWords) : nullptr;
    a.ws_words = a.ws ? (ctx->ws_bytes - lxq::kWorkspaceWords) / 4 : 0;
    if (hipSetDevice(ctx->device) != hipSuccess) return LUX_BACKEND_ERROR_DEVICE_LOST;
    return map_status(lxq::launch_paged_plan(a, ctx->stream));
}

LuxBackendError op_paged_append(LuxBackendContext* c, const lux_paged_append_args* p) {
    HipContext* ctx = C(c);
    if (!ctx || !p || p->struct_size != sizeof(*p)) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    if (p->tokens < 0 || !cache_ok(p->kv_heads, p->head_dim, p->page_size, p->num_pages))
        return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    const int64_t row = (int64_t)p->kv_heads * p->head_dim;
    if (!stride_ok(p->k_row_stride, row) || !stride_ok(p->v_row_stride, row) || !offset_ok(p->k_offset) ||
        !offset_ok(p->v_offset))
        return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    if (!dtype_ok(p->in_dtype) || !dtype_ok(p->cache_dtype) || row >= (1ll << 31) ||
        !rows_ok(p->kv_heads, p->page_size, p->num_pages))
        return LUX_BACKEND_ERROR_NOT_SUPPORTED;
    lxq::AppendArgs a;
    Spans s;
    const size_t ie = dtype_size(p->in_dtype), ce = dtype_size(p->cache_dtype);
    const size_t cache = (size_t)p->num_pages * p->page_size * row * ce;
    a.k_row = p->k_row_stride ? p->k_row_stride : row;
    a.v_row = p->v_row_stride ? p->v_row_stride : row;
    a.k = s.in(p->k, (size_t)p->k_offset * ie, extent(p->tokens, a.k_row, row, ie), ie);
    a.v = s.in(p->v, (size_t)p->v_offset * ie, extent(p->tokens, a.v_row, row, ie), ie);
    a.slots = static_cast<const int32_t*>(s.in(p->slots, 0, (size_t)p->tokens * 4, 4));
    a.kc = s.out(p->k_cache, 0, cache, ce);
    a.vc = s.out(p->v_cache, 0, cache, ce);
    if (!s.ok || !s.apart()) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    if (p->tokens == 0 || p->num_pages == 0) return LUX_BACKEND_OK;
    a.T = p->tokens; a.Hk = p->kv_heads; a.D = p->head_dim; a.page = p->page_size; a.pool = p->num_pages;
    a.in_dt = p->in_dtype; a.cache_dt = p->cache_dtype;
    a.div = lxq::DivBy(p->page_size);
    if (hipSetDevice(ctx->device) != hipSuccess) return LUX_BACKEND_ERROR_DEVICE_LOST;
    return map_status(lxq::launch_paged_append(a, ctx->stream));
}

LuxBackendError op_paged_attention(LuxBackendContext* c, const lux_paged_attention_args* p) {
    HipContext* ctx = C(c);
    if (!ctx || !p || p->struct_size != sizeof(*p)) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    if (p->requests < 0 || p->heads <= 0 || !cache_ok(p->kv_heads, p->head_dim, p->page_size, p->num_pages) ||
        p->heads % p->kv_heads || p->max_pages <= 0 || p->window < 0 || !cap_ok(p->softcap))
        return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    const int64_t row = (int64_t)p->heads * p->head_dim;
    if (!stride_ok(p->q_row_stride, row) || !stride_ok(p->out_row_stride, row) || !offset_ok(p->q_offset) ||
        !offset_ok(p->out_offset))
        return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    if (!dtype_ok(p->dtype) || p->head_dim % 8 || p->head_dim > 256 || row >= (1ll << 31) ||
        !rows_ok(p->kv_heads, p->page_size, p->num_pages) || !rows_ok(1, p->page_size, p->max_pages) ||
        (int64_t)p->requests * p->heads >= (1ll << 31))
        return LUX_BACKEND_ERROR_NOT_SUPPORTED;
    lxq::AttnArgs a;
    Spans s;
    const size_t e = dtype_size(p->dtype), R = (size_t)p->requests;
    const size_t cache = (size_t)p->num_pages * p->page_size * p->kv_heads * p->head_dim * e;
    a.q_row = p->q_row_stride ? p->q_row_stride : row;
    a.out_row = p->out_row_stride ? p->out_row_stride : row;
    a.q = s.in(p->q, (size_t)p->q_offset * e, extent(p->requests, a.q_row, row, e), e);
    a.kc = s.in(p->k_cache, 0, cache, 16);
    a.vc = s.in(p->v_cache, 0, cache, 16);
    a.table = static_cast<const int32_t*>(s.in(p->block_table, 0, R * p->max_pages * 4, 4));
    a.lens = static_cast<const int32_t*>(s.in(p->kv_lens, 0, R * 4, 4));
    a.out = s.out(p->out, (size_t)p->out_offset * e, extent(p->requests, a.out_row, row, e), e);
    a.lse = p->lse ? static_cast<float*>(s.out(p->lse, 0, R * p->heads * 4, 4)) : nullptr;
    if (!s.ok || !s.apart()) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    if (p->requests == 0) return LUX_BACKEND_OK;
    a.R = p->requests; a.H = p->heads; a.Hk = p->kv_heads; a.G = p->heads / p->kv_heads; a.D = p->head_dim;
    a.page = p->page_size; a.pool = p->num_pages; a.columns = p->max_pages; a.window = p->window;
    a.dtype = p->dtype; a.scale = p->scale; a.softcap = p->softcap;
    a.div = lxq::DivBy(p->page_size);
    a.ws = ctx->ws_bytes > lxq::kWorkspaceWords ? reinterpret_cast<float*>(static_cast<char*>(ctx->ws) + lxq::kWorkspaceWords) : nullptr;
    a.ws_bytes = a.ws ? ctx->ws_bytes - lxq::kWorkspaceWords : 0;
    a.count = static_cast<uint32_t*>(ctx->counts);
    a.counts = ctx->counts ? kCountWords : 0;
    a.cus = ctx->compute_units;
    if (hipSetDevice(ctx->device) != hipSuccess) return LUX_BACKEND_ERROR_DEVICE_LOST;
    return map_status(lxq::launch_paged_attention(a, ctx->stream));
}

bool norm_ok(int k) { return k >= LUX_NORM_NONE && k <= LUX_NORM_LAYER; }

LuxBackendError op_block_norm(LuxBackendContext* c, const lux_block_norm_args* p) {
    HipContext* ctx = C(c);
    if (!ctx || !p || p->struct_size != sizeof(*p)) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    const int T = p->rows, D = p->dim;
    if (T < 0 || D <= 0 || !norm_ok(p->post_norm) || !norm_ok(p->pre_norm) || p->gate_mode < LUX_GATE_NONE ||
        p->gate_mode > LUX_GATE_FULL || (!p->x && !p->residual) || (!p->residual_out && !p->out) ||
        (p->gate_mode != LUX_GATE_NONE && !p->gate))
        return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    for (int64_t st : {p->x_row_stride, p->residual_row_stride, p->residual_out_row_stride, p->out_row_stride})
        if (!stride_ok(st, D)) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    if (!stride_ok(p->gate_row_stride, p->gate_mode == LUX_GATE_ROW ? 1 : D)) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    if (!dtype_ok(p->x_dtype) || !dtype_ok(p->residual_dtype) || !dtype_ok(p->weight_dtype) || D > 65536)
        return LUX_BACKEND_ERROR_NOT_SUPPORTED;
    lxq::NormArgs a = {};
    Spans s;
    const size_t xe = dtype_size(p->x_dtype), re = dtype_size(p->residual_dtype), we = dtype_size(p->weight_dtype);
    a.x_row = p->x_row_stride ? p->x_row_stride : D;
    a.r_row = p->residual_row_stride ? p->residual_row_stride : D;
    a.h_row = p->residual_out_row_stride ? p->residual_out_row_stride : D;
    a.o_row = p->out_row_stride ? p->out_row_stride : D;
    a.post = p->x ? p->post_norm : LUX_NORM_NONE;
    a.pre = p->out ? p->pre_norm : LUX_NORM_NONE;
    a.gate_mode = p->x ? p->gate_mode : LUX_GATE_NONE;
    const int64_t grow = a.gate_mode == LUX_GATE_ROW ? 1 : D;
    a.g_row = p->gate_row_stride ? p->gate_row_stride : grow;
    if (p->x) a.x = s.in(p->x, 0, extent(T, a.x_row, D, xe), xe);
    if (p->residual) a.r = s.in(p->residual, 0, extent(T, a.r_row, D, re), re);
    const int x_at = 0, r_at = p->x ? 1 : 0;
    if (a.gate_mode != LUX_GATE_NONE)
        a.gate = s.in(p->gate, 0, extent(a.gate_mode == LUX_GATE_CHANNEL ? 1 : T, a.g_row, grow, xe), xe);
    if (a.post != LUX_NORM_NONE) {
        if (p->post_weight) a.pw = s.in(p->post_weight, 0, D * we, we);
        if (p->post_bias) a.pb = s.in(p->post_bias, 0, D * we, we);
    }
    if (a.pre != LUX_NORM_NONE) {
        if (p->pre_weight) a.nw = s.in(p->pre_weight, 0, D * we, we);
        if (p->pre_bias) a.nb = s.in(p->pre_bias, 0, D * we, we);
    }
    const int h_at = s.count;
    if (p->residual_out) a.h = s.out(p->residual_out, 0, extent(T, a.h_row, D, re), re);
    const int o_at = s.count;
    if (p->out) a.out = s.out(p->out, 0, extent(T, a.o_row, D, xe), xe);
    if (!s.ok) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    // in place: each thread reads its elements before it writes them
    for (int i = 0; i < s.count; i++)
        for (int j = 0; j < i; j++) {
            if (!(s.s[i].out || s.s[j].out) || !s.s[i].meets(s.s[j])) continue;
            const bool h_is_r = p->residual_out && p->residual && i == h_at && j == r_at && a.h == a.r && a.h_row == a.r_row;
            const bool o_is_x = p->out && p->x && i == o_at && j == x_at && a.out == a.x && a.o_row == a.x_row;
            if (!h_is_r && !o_is_x) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
        }
    if (T == 0) return LUX_BACKEND_OK;
    a.T = T; a.D = D; a.x_dt = p->x_dtype; a.r_dt = p->residual_dtype; a.w_dt = p->weight_dtype;
    a.rscale = p->residual_scale; a.eps = p->eps;
    if (hipSetDevice(ctx->device) != hipSuccess) return LUX_BACKEND_ERROR_DEVICE_LOST;
    return map_status(lxq::launch_block_norm(a, ctx->stream));
}

bool on_device(const HipContext* ctx, const void* p) {
    hipPointerAttribute_t at;
    if (hipPointerGetAttributes(&at, p) != hipSuccess) {
        (void)hipGetLastError();
        return false;
    }
    return at.type == hipMemoryTypeDevice && at.device == ctx->device;
}

// readable bytes behind a view of device memory: to the end of the allocation it lies in
size_t behind(char* p, size_t bytes) {
    hipDeviceptr_t base = nullptr;
    size_t size = 0;
    if (hipMemGetAddressRange(&base, &size, p) != hipSuccess) {
        (void)hipGetLastError();
        return 0;
    }
    const char *end = static_cast<char*>(base) + size, *mine = p + bytes;
    return end > mine ? (size_t)(end - mine) : 0;
}

LuxBackendBuffer* buffer_wrap(LuxBackendContext* c, void* ptr, size_t bytes) {
    HipContext* ctx = C(c);
    if (!ctx || (bytes && !ptr) || hipSetDevice(ctx->device) != hipSuccess) return nullptr;
    if (bytes && (!on_device(ctx, ptr) || !on_device(ctx, static_cast<char*>(ptr) + bytes - 1))) return nullptr;
    HipBuffer* b = new (std::nothrow) HipBuffer();
    if (!b) return nullptr;
    b->ptr = bytes ? ptr : nullptr;
    b->size = bytes;
    b->owned = false;
    b->tail = bytes ? behind(static_cast<char*>(ptr), bytes) : 0;
    return reinterpret_cast<LuxBackendBuffer*>(b);
}

const lux_gpu_serving_vtbl g_serving = {
    LUX_GPU_SERVING_EXT_VERSION, sizeof(lux_gpu_serving_vtbl),
    op_paged_plan, op_paged_append, op_paged_attention, op_block_norm, buffer_wrap, {},
};

}  // namespace

const lux_gpu_serving_vtbl* lux_hip_serving_table() { return &g_serving; }
