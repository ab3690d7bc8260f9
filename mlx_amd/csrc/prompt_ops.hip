// prompt_ops.hip -- entry points of the operators of prompts and of pages in use
// (include/lux_gpu_prompt_backend.h): argument checks, then one launcher.
#include "prompt.h"
#include "spans.h"

using namespace lxh;

namespace {

LuxBackendError op_paged_chunk_attention(LuxBackendContext* c, const lux_paged_chunk_args* p) {
    HipContext* ctx = C(c);
    if (!ctx || !p || p->struct_size != sizeof(*p)) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    if (p->requests < 0 || p->tokens < 0 || p->heads <= 0 ||
        !cache_ok(p->kv_heads, p->head_dim, p->page_size, p->num_pages) || p->heads % p->kv_heads || p->max_pages <= 0 ||
        p->window < 0 || !cap_ok(p->softcap))
        return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    const int64_t row = (int64_t)p->heads * p->head_dim;
    if (!stride_ok(p->q_row_stride, row) || !stride_ok(p->out_row_stride, row) || !offset_ok(p->q_offset) ||
        !offset_ok(p->out_offset))
        return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    const int64_t reach = (int64_t)p->max_pages * p->page_size;
    if (!dtype_ok(p->dtype) || p->head_dim % 8 || p->head_dim > 256 || row >= (1ll << 31) ||
        !rows_ok(p->kv_heads, p->page_size, p->num_pages) || reach + p->tokens >= (1ll << 31) ||
        ((int64_t)p->tokens + 256ll * p->requests) * (reach / 64 + 1) >= (1ll << 39))
        return LUX_BACKEND_ERROR_NOT_SUPPORTED;
    lxq::ChunkArgs a;
    Spans s;
    const size_t e = dtype_size(p->dtype), R = (size_t)p->requests, T = (size_t)p->tokens;
    const size_t cache = (size_t)p->num_pages * p->page_size * p->kv_heads * p->head_dim * e;
    a.q_row = p->q_row_stride ? p->q_row_stride : row;
    a.out_row = p->out_row_stride ? p->out_row_stride : row;
    a.q = s.in(p->q, (size_t)p->q_offset * e, extent(p->tokens, a.q_row, row, e), e);
    a.kc = s.in(p->k_cache, 0, cache, 16);
    a.vc = s.in(p->v_cache, 0, cache, 16);
    a.table = static_cast<const int32_t*>(s.in(p->block_table, 0, R * p->max_pages * 4, 4));
    a.starts = static_cast<const int32_t*>(s.in(p->token_starts, 0, R * 4 + 4, 4));
    a.seq = static_cast<const int32_t*>(s.in(p->seq_lens, 0, R * 4, 4));
    a.lens = static_cast<const int32_t*>(s.in(p->kv_lens, 0, R * 4, 4));
    a.out = s.out(p->out, (size_t)p->out_offset * e, extent(p->tokens, a.out_row, row, e), e);
    a.lse = p->lse ? static_cast<float*>(s.out(p->lse, 0, T * p->heads * 4, 4)) : nullptr;
    if (!s.ok || !s.apart()) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    if (p->requests == 0 || p->tokens == 0) return LUX_BACKEND_OK;
    a.R = p->requests; a.T = p->tokens; a.H = p->heads; a.Hk = p->kv_heads; a.G = p->heads / p->kv_heads; a.D = p->head_dim;
    a.page = p->page_size; a.pool = p->num_pages; a.columns = p->max_pages; a.window = p->window;
    a.dtype = p->dtype; a.scale = p->scale; a.softcap = p->softcap;
    a.div = lxq::DivBy(p->page_size);
    a.ws = static_cast<char*>(ctx->parts);
    a.cus = ctx->compute_units;
    if (hipSetDevice(ctx->device) != hipSuccess) return LUX_BACKEND_ERROR_DEVICE_LOST;
    return map_status(lxq::launch_paged_chunk(a, ctx->stream));
}

const lux_gpu_prompt_vtbl g_prompt = {
    LUX_GPU_PROMPT_EXT_VERSION, sizeof(lux_gpu_prompt_vtbl), op_paged_chunk_attention, nullptr, nullptr, nullptr, nullptr, nullptr, {},
};

}  // namespace

const lux_gpu_prompt_vtbl* lux_hip_prompt_table() { return &g_prompt; }
