/*
 * lux_gpu_serving_backend.h -- the operators of a decoding step over a paged
 * key-value cache, beside the quantized matmul (lux_gpu_quant_backend.h).
 *
 * The table is reached through lux_gpu_quant_vtbl::serving (NULL in plugins
 * that predate it); there is no further exported symbol.  No counterpart in
 * the reference: its vtable has no attention, no cache and no fused norm
 * (reference include/lux/gpu/backend_plugin.h:82-382).  The ops take the
 * base vtable's contexts and device buffers.  Each takes one record of
 * arguments, which a caller may keep and pass again at the next step:
 * nothing is remembered between calls.
 *
 * Cache.  A layer's keys, and its values, are T[num_pages, kv_heads,
 * page_size, head_dim], contiguous.  Request r's token at position t is at
 * place t % page_size of page block_table[r, t / page_size]
 * (int32[requests, max_pages]); its slot is page * page_size + place.  A page
 * id outside [0, num_pages) names no page: its tokens take part in nothing.
 *
 * Errors: NULL handle, negative or impossible size, a struct_size that is not
 * the record's, a buffer smaller than the sizes need, a stride below the row
 * length, an output that overlaps an input or another output (from first to last
 * element, rows between those of the other included; but where an op allows it)
 * -> INVALID_ARGUMENT; a dtype, head_dim, dim or pool size outside
 * the stated ones -> NOT_SUPPORTED; HIP launch failure -> INTERNAL.  All ops
 * are asynchronous on the context's stream and make no allocation.  Strides
 * and offsets are in elements; a stride of 0 stands for the row length.
 */
#ifndef LUX_GPU_SERVING_BACKEND_H
#define LUX_GPU_SERVING_BACKEND_H

#include "lux_gpu_backend_abi.h"

#ifdef __cplusplus
extern "C" {
#endif

#define LUX_GPU_SERVING_EXT_VERSION 1

/*
 * The plan of a step: which pages the new tokens take, and where each token
 * goes.  Request r holds seq_lens[r] tokens and gets new_lens[r] more (each
 * taken as 0 where negative, seq_lens as the table's capacity C = max_pages *
 * page_size where above).  With have = ceil(seq / page_size) and need =
 * min(ceil((seq + new) / page_size), max_pages) - have, requests take their
 * pages in order from free_pages, from entry free_head[0] on (0 where it is
 * negative); entries at or past free_count are not there.  All arrays int32.
 *   block_table[r, have .. have + need): the pages taken, -1 where none was
 *             left; other entries stay
 *   kv_lens[r] = min(seq + new, pages held * page_size): what attention may
 *             read, and the next step's seq_lens
 *   token_starts[r] = the new tokens before request r; [requests]: all of them
 *   slots[t], positions[t], token_request[t], t < max_tokens: the t-th new
 *             token's slot (-1 where its position is at or past kv_lens or
 *             its page is none), position and request; -1, 0, -1 past the
 *             last token.  Tokens past max_tokens get no entry.
 *   counts = {entry of free_pages after the last one taken, new tokens,
 *             pages needed and not there, new tokens past kv_lens}
 * The next step's free_head may be this step's counts; the two buffers of one
 * step are distinct.  The sum of new_lens has to stay below 2^31.
 */
typedef struct lux_paged_plan_args {
    uint32_t struct_size;
    int32_t requests, max_tokens, max_pages, page_size;
    int32_t num_pages;  /* of the pool */
    int32_t free_count; /* entries of free_pages */
    int32_t _pad;
    LuxBackendBuffer* seq_lens;      /* [requests] */
    LuxBackendBuffer* new_lens;      /* [requests] */
    LuxBackendBuffer* free_pages;    /* [free_count] */
    LuxBackendBuffer* free_head;     /* [1] */
    LuxBackendBuffer* block_table;   /* [requests, max_pages], in and out */
    LuxBackendBuffer* slots;         /* [max_tokens] */
    LuxBackendBuffer* positions;     /* [max_tokens], or NULL */
    LuxBackendBuffer* token_request; /* [max_tokens], or NULL */
    LuxBackendBuffer* token_starts;  /* [requests + 1] */
    LuxBackendBuffer* kv_lens;       /* [requests] */
    LuxBackendBuffer* counts;        /* [4] */
} lux_paged_plan_args;

/*
 * k_cache, v_cache at slots[t] = k[t], v[t] (rounded to cache_dtype, RNE), for
 * each t < tokens whose slot is in [0, num_pages * page_size); other tokens
 * are left out.  Two tokens of one call with the same slot: each value is one
 * of the two.
 * Row t of k is k_offset + t * k_row_stride elements in, its heads next to
 * each other; so for v.
 */
typedef struct lux_paged_append_args {
    uint32_t struct_size;
    int32_t tokens, kv_heads, head_dim, page_size, num_pages;
    int32_t in_dtype, cache_dtype; /* LuxBackendDtype: FLOAT32, FLOAT16 or BFLOAT16 */
    int64_t k_offset, k_row_stride, v_offset, v_row_stride;
    LuxBackendBuffer* k;       /* [tokens, kv_heads * head_dim] */
    LuxBackendBuffer* v;
    LuxBackendBuffer* slots;   /* int32[tokens] */
    LuxBackendBuffer* k_cache; /* [num_pages, kv_heads, page_size, head_dim] */
    LuxBackendBuffer* v_cache;
} lux_paged_append_args;

/*
 * Attention of one token per request over its cached tokens: row r of q is
 * request r's.  (A plan numbers tokens; where some requests of a step get
 * none, the token of request r is row token_starts[r] of its arrays.)  Head i reads
 * the keys and values of head i / (heads / kv_heads).  Over the positions t
 * of [max(0, n - window), n), n = kv_lens[r] cut to [0, max_pages *
 * page_size] (window 0: all of [0, n)), but those whose page is none:
 *   s_t = scale * q . k_t, or softcap * tanh(scale * q . k_t / softcap) where
 *   softcap > 0 (2^-100 to 2^100; others but 0 are INVALID_ARGUMENT);
 *   out = sum_t exp(s_t) v_t / sum_t exp(s_t);
 *   lse = log(sum_t exp(s_t))
 * A request with no position gives out = 0 and lse = -infinity.  A score
 * that leaves fp32 when multiplied by log2 e is infinite (2.36e38).  Cache places
 * that no position of a request names are never part of its result, whatever
 * they hold.  Scores, sums and the running statistics are fp32; with 16-bit
 * types exp(s - max) enters the product with v as the sum of two values of
 * that type, neither of them 0 (in f16 from 2^-38 of the largest on).  So an
 * infinite value in a place that counts is the channel's result, two opposite
 * ones NaN.
 * head_dim: a multiple of 8, at most 256; heads a multiple of kv_heads;
 * num_pages * kv_heads * page_size below 2^31; the caches start on 16 bytes.
 */
typedef struct lux_paged_attention_args {
    uint32_t struct_size;
    int32_t requests, heads, kv_heads, head_dim, page_size, num_pages, max_pages;
    int32_t window;
    int32_t dtype; /* of q, the cache and out: FLOAT32, FLOAT16 or BFLOAT16 */
    float scale, softcap;
    int64_t q_offset, q_row_stride, out_offset, out_row_stride;
    LuxBackendBuffer* q;           /* [requests, heads * head_dim] */
    LuxBackendBuffer* k_cache;     /* [num_pages, kv_heads, page_size, head_dim] */
    LuxBackendBuffer* v_cache;
    LuxBackendBuffer* block_table; /* int32[requests, max_pages] */
    LuxBackendBuffer* kv_lens;     /* int32[requests] */
    LuxBackendBuffer* out;         /* [requests, heads * head_dim] */
    LuxBackendBuffer* lse;         /* f32[requests, heads], or NULL */
} lux_paged_attention_args;

typedef enum {
    LUX_NORM_NONE = 0,  /* v as it is */
    LUX_NORM_RMS = 1,   /* v / sqrt(mean(v^2) + eps) * weight + bias */
    LUX_NORM_LAYER = 2, /* the same of v - mean(v) */
} LuxNormKind;

typedef enum {
    LUX_GATE_NONE = 0,
    LUX_GATE_CHANNEL = 1, /* gate[dim] */
    LUX_GATE_ROW = 2,     /* gate[rows] */
    LUX_GATE_FULL = 3,    /* gate[rows, dim] */
} LuxGateMode;

/*
 * Between two blocks, per row of dim values:
 *   h = residual_scale * residual + gate * post_norm(x)   (x NULL: the first term alone)
 *   residual_out = h;  out = pre_norm(h)
 * x is a block's output, post_norm the norm after it, pre_norm the norm before
 * the next block.  In fp32, h unrounded into pre_norm; each output is rounded
 * once.  A NULL weight is 1, a NULL bias 0.  residual NULL: h = gate *
 * post_norm(x).  Rows of gate are gate_row_stride apart (GATE_ROW: its values).
 * residual_out or out may be NULL, not both.  residual_out may be residual
 * itself, and out may be x (same place, stride and dtype).  dim: at most 65536.
 */
typedef struct lux_block_norm_args {
    uint32_t struct_size;
    int32_t rows, dim;
    int32_t post_norm, pre_norm; /* LuxNormKind */
    int32_t gate_mode;           /* LuxGateMode */
    int32_t x_dtype;             /* of x, gate and out */
    int32_t residual_dtype;      /* of residual and residual_out */
    int32_t weight_dtype;        /* of the weights and biases */
    float residual_scale, eps;
    int32_t _pad;
    int64_t x_row_stride, residual_row_stride, gate_row_stride, residual_out_row_stride, out_row_stride;
    LuxBackendBuffer* x;
    LuxBackendBuffer* residual;
    LuxBackendBuffer* post_weight; /* [dim] */
    LuxBackendBuffer* post_bias;
    LuxBackendBuffer* gate;
    LuxBackendBuffer* pre_weight;
    LuxBackendBuffer* pre_bias;
    LuxBackendBuffer* residual_out;
    LuxBackendBuffer* out;
} lux_block_norm_args;

typedef struct lux_gpu_serving_vtbl {
    uint32_t ext_version; /* LUX_GPU_SERVING_EXT_VERSION */
    uint32_t struct_size; /* sizeof(lux_gpu_serving_vtbl) of the plugin */

    LuxBackendError (*op_paged_plan)(LuxBackendContext* ctx, const lux_paged_plan_args* args);
    LuxBackendError (*op_paged_append)(LuxBackendContext* ctx, const lux_paged_append_args* args);
    LuxBackendError (*op_paged_attention)(LuxBackendContext* ctx, const lux_paged_attention_args* args);
    LuxBackendError (*op_block_norm)(LuxBackendContext* ctx, const lux_block_norm_args* args);

    /* a buffer over `bytes` bytes of device memory that the caller owns (a
     * part of another allocation, another library's tensor) and keeps until
     * buffer_free, which leaves the memory alone.  NULL where device_ptr is
     * no memory of the context's device.  Work of other streams on that memory
     * is the caller's to order.  The serving ops read nothing past `bytes`.
     * The quantized ops read their inputs (but a fused bias) in vectors: they
     * refuse a wrapped one (INVALID_ARGUMENT) that does not start on 16 bytes or
     * has not 256 readable bytes behind what they need of it, in the buffer or in
     * the rest of the allocation that it lies in.  Their outputs start on an
     * element (op_dequantize's on 16 bytes, codes on 4).  The base table's ops ask for
     * 4 bytes (matmul: and 12 readable ones behind its inputs). */
    LuxBackendBuffer* (*buffer_wrap)(LuxBackendContext* ctx, void* device_ptr, size_t bytes);

    void* _reserved[5];
} lux_gpu_serving_vtbl;

/* layout pins: LP64 */
#if defined(__LP64__)
#ifdef __cplusplus
static_assert(sizeof(lux_paged_plan_args) == 120, "plan record");
static_assert(sizeof(lux_paged_append_args) == 104, "append record");
static_assert(sizeof(lux_paged_attention_args) == 136, "attention record");
static_assert(sizeof(lux_block_norm_args) == 160, "norm record");
static_assert(sizeof(lux_gpu_serving_vtbl) == 88, "serving table");
#else
_Static_assert(sizeof(lux_paged_plan_args) == 120, "plan record");
_Static_assert(sizeof(lux_paged_append_args) == 104, "append record");
_Static_assert(sizeof(lux_paged_attention_args) == 136, "attention record");
_Static_assert(sizeof(lux_block_norm_args) == 160, "norm record");
_Static_assert(sizeof(lux_gpu_serving_vtbl) == 88, "serving table");
#endif
#endif

#ifdef __cplusplus
}
#endif

#endif /* LUX_GPU_SERVING_BACKEND_H */
