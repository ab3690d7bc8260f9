// prompt_ops.hip -- entry points of the operators of prompts and of pages in use
// (include/lux_gpu_prompt_backend.h): argument checks, then one launcher.
#include "prompt.h"
#include "spans.h"

using namespace lxh;

namespace {

// The memory for partial results of the context's chunk attentions: programs without
// prompts go without it.  The first call may be one that is captured: an allocation is
// no part of a graph, and relaxed capture lets it pass.
char* chunk_parts(HipContext* ctx) {
    if (!ctx->parts) {
        hipStreamCaptureMode mode = hipStreamCaptureModeRelaxed;
        if (hipThreadExchangeStreamCaptureMode(&mode) != hipSuccess) return nullptr;
        if (hipMalloc(&ctx->parts, lxq::kChunkPartBytes) != hipSuccess) {
            (void)hipGetLastError();
            ctx->parts = nullptr;
        }
        (void)hipThreadExchangeStreamCaptureMode(&mode);
    }
    return static_cast<char*>(ctx->parts);
}

LuxBackendError op_paged_chunk_attention(LuxBackendContext* c, const lux_paged_chunk_args* p) {
    HipContext* ctx = C(c);
    if (!ctx || !p || p->struct_size != sizeof(*p)) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    if (p->requests < 0 || p->tokens < 0 || p->heads <= 0 ||
        !cache_ok(p->kv_heads, p->head_dim, p->page_size, p->num_pages) || p->heads % p->kv_heads || p->max_pages <= 0 ||
        p->window < 0 || !cap_ok(p->softcap) || !(p->scale - p->scale == 0.f))
        return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    const int64_t row = (int64_t)p->heads * p->head_dim;
    if (!stride_ok(p->q_row_stride, row) || !stride_ok(p->out_row_stride, row) || !offset_ok(p->q_offset) ||
        !offset_ok(p->out_offset))
        return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    const int64_t reach = (int64_t)p->max_pages * p->page_size;
    if (!dtype_ok(p->dtype) || p->head_dim % 8 || p->head_dim > 256 || row >= (1ll << 31) ||
        !rows_ok(p->kv_heads, p->page_size, p->num_pages) || reach + p->tokens >= (1ll << 31))
        return LUX_BACKEND_ERROR_NOT_SUPPORTED;
    // the stages of all tiles for one head, of the smallest tiles and shortest stages
    const int group = p->heads / p->kv_heads;
    if ((p->tokens / (group < 64 ? 64 / group : 1) + (int64_t)p->requests) * (reach / 32 + 1) >= (1ll << 31))
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
    a.cus = ctx->compute_units;
    if (hipSetDevice(ctx->device) != hipSuccess) return LUX_BACKEND_ERROR_DEVICE_LOST;
    a.ws = chunk_parts(ctx);
    if (!a.ws) return LUX_BACKEND_ERROR_OUT_OF_MEMORY;
    return map_status(lxq::launch_paged_chunk(a, ctx->stream));
}

// words behind those that the GEMMs keep
int32_t* words(const HipContext* ctx, size_t& n) {
    n = ctx->ws && ctx->ws_bytes > lxq::kWorkspaceWords ? (ctx->ws_bytes - lxq::kWorkspaceWords) / 4 : 0;
    return n ? reinterpret_cast<int32_t*>(static_cast<char*>(ctx->ws) + lxq::kWorkspaceWords) : nullptr;
}

// requests, table, pool and list that the records of pages in use have alike.  A wave
// looks at up to 256 columns at a time, in 31 bits
template <class A>
LuxBackendError pages_ok(const A* p) {
    if (p->requests < 0 || p->max_pages <= 0 || p->page_size <= 0 || p->num_pages < 0 || p->free_count < 0)
        return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    if (!rows_ok(1, p->page_size, p->num_pages) || !rows_ok(1, p->page_size, p->max_pages) ||
        (int64_t)p->requests * p->max_pages >= (1ll << 31) - 1 || p->num_pages > (1 << 22) || p->max_pages > INT32_MAX - 256)
        return LUX_BACKEND_ERROR_NOT_SUPPORTED;
    return LUX_BACKEND_OK;
}

const int32_t* ints_in(Spans& s, LuxBackendBuffer* b, size_t n) { return static_cast<const int32_t*>(s.in(b, 0, n * 4, 4)); }
int32_t* ints_out(Spans& s, LuxBackendBuffer* b, size_t n) { return static_cast<int32_t*>(s.out(b, 0, n * 4, 4)); }

// no output over another argument, but `out` (an index of s) may be `in` itself
bool apart_but(const Spans& s, int out, int in) {
    for (int i = 0; i < s.count; i++)
        for (int j = 0; j < i; j++) {
            if (!(s.s[i].out || s.s[j].out) || !s.s[i].meets(s.s[j])) continue;
            if (i == out && j == in && s.s[i].p == s.s[j].p) continue;
            return false;
        }
    return true;
}

LuxBackendError op_paged_fork(LuxBackendContext* c, const lux_paged_fork_args* p) {
    HipContext* ctx = C(c);
    if (!ctx || !p || p->struct_size != sizeof(*p) || p->forks < 0) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    if (LuxBackendError e = pages_ok(p)) return e;
    if (p->forks > (1 << 20)) return LUX_BACKEND_ERROR_NOT_SUPPORTED;
    lxq::ForkArgs a;
    Spans s;
    const size_t F = (size_t)p->forks, R = (size_t)p->requests;
    a.src = ints_in(s, p->src, F);
    a.dst = ints_in(s, p->dst, F);
    a.free_pages = ints_in(s, p->free_pages, p->free_count);
    a.head = ints_in(s, p->free_head, 1);
    a.lens = ints_out(s, p->lens, R);
    a.table = ints_out(s, p->block_table, R * p->max_pages);
    a.shares = ints_out(s, p->shares, p->num_pages);
    a.copy_src = ints_out(s, p->copy_src, F);
    a.copy_dst = ints_out(s, p->copy_dst, F);
    a.counts = ints_out(s, p->counts, 4);
    if (!s.ok || !s.apart()) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    a.F = p->forks; a.R = p->requests; a.columns = p->max_pages; a.page = p->page_size; a.pool = p->num_pages;
    a.free_count = p->free_count;
    a.div = lxq::DivBy(p->page_size);
    a.ws = words(ctx, a.ws_words);
    if (hipSetDevice(ctx->device) != hipSuccess) return LUX_BACKEND_ERROR_DEVICE_LOST;
    return map_status(lxq::launch_paged_fork(a, ctx->stream));
}

LuxBackendError op_paged_release(LuxBackendContext* c, const lux_paged_release_args* p) {
    HipContext* ctx = C(c);
    if (!ctx || !p || p->struct_size != sizeof(*p)) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    if (LuxBackendError e = pages_ok(p)) return e;
    lxq::ReleaseArgs a;
    Spans s;
    const size_t R = (size_t)p->requests;
    a.lens = ints_in(s, p->lens, R);
    a.keep = ints_in(s, p->keep_lens, R);
    a.table = ints_in(s, p->block_table, R * p->max_pages);
    a.head = ints_in(s, p->free_head, 1);
    a.shares = ints_out(s, p->shares, p->num_pages);
    a.free_pages = ints_out(s, p->free_pages, p->free_count);
    a.kv = ints_out(s, p->kv_lens, R);
    a.counts = ints_out(s, p->counts, 4);
    if (!s.ok || !apart_but(s, 6, 0)) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    a.R = p->requests; a.columns = p->max_pages; a.page = p->page_size; a.pool = p->num_pages; a.free_count = p->free_count;
    a.div = lxq::DivBy(p->page_size);
    a.ws = words(ctx, a.ws_words);
    if (hipSetDevice(ctx->device) != hipSuccess) return LUX_BACKEND_ERROR_DEVICE_LOST;
    return map_status(lxq::launch_paged_release(a, ctx->stream));
}

LuxBackendError op_paged_compact(LuxBackendContext* c, const lux_paged_compact_args* p) {
    HipContext* ctx = C(c);
    if (!ctx || !p || p->struct_size != sizeof(*p)) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    if (LuxBackendError e = pages_ok(p)) return e;
    if (p->limit < 0 || p->limit > p->num_pages || p->max_moves < 0) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    lxq::CompactArgs a;
    Spans s;
    const size_t R = (size_t)p->requests, N = (size_t)p->num_pages;
    a.table = ints_in(s, p->block_table, R * p->max_pages);
    a.shares = ints_in(s, p->shares, N);
    a.lens = ints_in(s, p->lens, R);
    a.table_out = ints_out(s, p->table_out, R * p->max_pages);
    a.shares_out = ints_out(s, p->shares_out, N);
    a.free_pages = ints_out(s, p->free_pages, p->free_count);
    a.copy_src = ints_out(s, p->copy_src, p->max_moves);
    a.copy_dst = ints_out(s, p->copy_dst, p->max_moves);
    a.counts = ints_out(s, p->counts, 4);
    if (!s.ok) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    // table_out may be block_table, shares_out shares: as if they were left out
    if (a.table_out == a.table) s.s[0].n = 0;
    if (a.shares_out == a.shares) s.s[1].n = 0;
    if (!s.apart()) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    a.R = p->requests; a.columns = p->max_pages; a.page = p->page_size; a.pool = p->num_pages; a.free_count = p->free_count;
    a.limit = p->limit; a.max_moves = p->max_moves;
    a.div = lxq::DivBy(p->page_size); a.by_columns = lxq::DivBy(p->max_pages > 0 ? p->max_pages : 1);
    a.ws = words(ctx, a.ws_words);
    if (hipSetDevice(ctx->device) != hipSuccess) return LUX_BACKEND_ERROR_DEVICE_LOST;
    return map_status(lxq::launch_paged_compact(a, ctx->stream));
}

LuxBackendError op_paged_copy(LuxBackendContext* c, const lux_paged_copy_args* p) {
    HipContext* ctx = C(c);
    if (!ctx || !p || p->struct_size != sizeof(*p)) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    if (p->pages < 0 || p->layers < 0 || !cache_ok(p->kv_heads, p->head_dim, p->page_size, p->num_pages))
        return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    const int64_t head = (int64_t)p->page_size * p->head_dim;
    if (!dtype_ok(p->dtype) || !rows_ok(p->kv_heads, p->page_size, p->num_pages) || head >= (1ll << 31) ||
        head * p->kv_heads >= (1ll << 31))
        return LUX_BACKEND_ERROR_NOT_SUPPORTED;
    const int64_t page = head * p->kv_heads, one = page * p->num_pages;
    if (!stride_ok(p->layer_stride, one)) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    lxq::CopyArgs a;
    Spans s;
    const size_t e = dtype_size(p->dtype);
    const int64_t stride = p->layer_stride ? p->layer_stride : one;
    const size_t cache = extent(p->layers, stride, one, e);
    a.src = ints_in(s, p->copy_src, p->pages);
    a.dst = ints_in(s, p->copy_dst, p->pages);
    a.kc = s.out(p->k_cache, 0, cache, e);
    a.vc = s.out(p->v_cache, 0, cache, e);
    if (!s.ok || !s.apart()) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    if (p->pages == 0 || p->layers == 0 || p->num_pages == 0) return LUX_BACKEND_OK;
    a.n = p->pages; a.layers = p->layers; a.pool = p->num_pages;
    a.page_bytes = page * (int64_t)e; a.layer_bytes = stride * (int64_t)e;
    a.esz = (int)e;
    if (hipSetDevice(ctx->device) != hipSuccess) return LUX_BACKEND_ERROR_DEVICE_LOST;
    return map_status(lxq::launch_paged_copy(a, ctx->stream));
}

LuxBackendError op_token_logprobs(LuxBackendContext* c, const lux_token_logprobs_args* p) {
    HipContext* ctx = C(c);
    if (!ctx || !p || p->struct_size != sizeof(*p)) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    if (p->rows < 0 || p->vocab <= 0 || p->top < 0 || p->top > p->vocab || !(p->scale > 0.f && p->scale <= 0x1.fffffep127f) ||
        !stride_ok(p->row_stride, p->vocab) || !offset_ok(p->logits_offset) || (p->logprobs && !p->tokens))
        return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    if (!dtype_ok(p->dtype) || p->vocab > (1 << 24) || p->top > 64) return LUX_BACKEND_ERROR_NOT_SUPPORTED;
    lxq::LogprobArgs a = {};
    Spans s;
    const size_t e = dtype_size(p->dtype), T = (size_t)p->rows;
    a.row = p->row_stride ? p->row_stride : p->vocab;
    a.logits = s.in(p->logits, (size_t)p->logits_offset * e, extent(p->rows, a.row, p->vocab, e), e);
    if (p->logprobs) a.tokens = ints_in(s, p->tokens, T);
    if (p->logprobs) a.logprobs = static_cast<float*>(s.out(p->logprobs, 0, T * 4, 4));
    if (p->entropy) a.entropy = static_cast<float*>(s.out(p->entropy, 0, T * 4, 4));
    if (p->lse) a.lse = static_cast<float*>(s.out(p->lse, 0, T * 4, 4));
    if (p->top && p->top_ids) a.top_ids = ints_out(s, p->top_ids, T * p->top);
    if (p->top && p->top_logprobs) a.top_lp = static_cast<float*>(s.out(p->top_logprobs, 0, T * p->top * 4, 4));
    if (!s.ok || !s.apart()) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    if (p->rows == 0) return LUX_BACKEND_OK;
    a.T = p->rows; a.V = p->vocab; a.dtype = p->dtype; a.scale = p->scale;
    a.top = a.top_ids || a.top_lp ? p->top : 0;
    size_t n;
    a.ws = reinterpret_cast<char*>(words(ctx, n));
    a.ws_bytes = n * 4;
    a.count = static_cast<uint32_t*>(ctx->counts);
    a.counts = ctx->counts ? kCountWords : 0;
    a.cus = ctx->compute_units;
    if (hipSetDevice(ctx->device) != hipSuccess) return LUX_BACKEND_ERROR_DEVICE_LOST;
    return map_status(lxq::launch_token_logprobs(a, ctx->stream));
}

const lux_gpu_prompt_vtbl g_prompt = {
    LUX_GPU_PROMPT_EXT_VERSION, sizeof(lux_gpu_prompt_vtbl), op_paged_chunk_attention, op_paged_fork, op_paged_release,
    op_paged_compact, op_paged_copy, op_token_logprobs, {},
};

}  // namespace

const lux_gpu_prompt_vtbl* lux_hip_prompt_table() { return &g_prompt; }
