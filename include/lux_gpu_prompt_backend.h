/*
 * lux_gpu_prompt_backend.h -- the operators of prompts and of pages in use,
 * beside those of a decoding step (lux_gpu_serving_backend.h): attention of
 * chunks of new tokens over the paged cache, pages that requests share, copy,
 * give back and move, and the log probabilities of tokens.
 *
 * The table is reached through lux_gpu_quant_vtbl::prompt (NULL in plugins
 * that predate it); there is no further exported symbol.  No counterpart in
 * the reference: its vtable has no cache and no attention, its softmax returns
 * the probabilities (reference include/lux/gpu/backend_plugin.h:82-382).
 * Records, buffers, the cache's layout, strides and errors are those of the
 * serving table: nothing is remembered between calls, all ops are asynchronous
 * on the context's stream and make no allocation, but for the 102 MB of workspace
 * that the first chunk attention of a context allocates (captured or not) and the
 * context keeps (OUT_OF_MEMORY where there are none); NULL handle, impossible size
 * or stride, wrong struct_size, a buffer too small, an output over an input or
 * another output (but where an op allows it) -> INVALID_ARGUMENT; a dtype,
 * head_dim, pool or count outside the stated ones -> NOT_SUPPORTED; HIP launch
 * failure -> INTERNAL.
 *
 * Pages in use.  A page that several requests name has its count in shares:
 * the requests that hold it beyond the first (0 for a page that one request
 * holds, and for a free one).  So a plan, which takes free pages, leaves
 * shares alone.  A program that shares pages keeps one array of zeros, one
 * entry per page, and passes it to every fork, release and compaction.  The
 * free list is the plan's: free_pages from entry free_head[0] on (0 where it is
 * negative, free_count where above); each op writes the next head as counts[0].
 * Counts and free_head of one call are distinct buffers.  A request's table
 * entries behind ceil(its length / page_size) mean nothing.  Forks, releases and
 * compactions take up to 2^22 pages, 2^20 forks, max_pages below 2^31 - 256, and
 * products of num_pages, or max_pages, and page_size, and of requests and max_pages
 * below 2^31 - 1.
 */
#ifndef LUX_GPU_PROMPT_BACKEND_H
#define LUX_GPU_PROMPT_BACKEND_H

#include "lux_gpu_backend_abi.h"

#ifdef __cplusplus
extern "C" {
#endif

#define LUX_GPU_PROMPT_EXT_VERSION 1

/*
 * Attention of a chunk of new tokens per request over the request's cached
 * tokens, the chunk's own among them (append comes first).  Rows of q from
 * token_starts[r] to token_starts[r + 1] are request r's, in order (any
 * number, 0 and 1 included); the i-th is at position p = seq_lens[r] + i, with
 * seq_lens[r] cut to [0, max_pages * page_size].  A plan's token_starts, seq_lens
 * (its input) and kv_lens are these arrays.
 * token_starts does not decrease; rows of q below token_starts[0] and from
 * token_starts[requests] on are no request's: out and lse stay there as they were.
 * Head j reads the keys and values of head j / (heads / kv_heads).  Over the
 * positions t of [max(0, p + 1 - window), min(p + 1, n)), n = kv_lens[r] cut to
 * [0, max_pages * page_size] (window 0: from 0 on), but those whose page is none:
 *   s_t = scale * q . k_t, or softcap * tanh(scale * q . k_t / softcap) where
 *   softcap > 0 (2^-100 to 2^100; others but 0 and a scale that is not finite are
 *   INVALID_ARGUMENT);
 *   out = sum_t exp(s_t) v_t / sum_t exp(s_t);  lse = log(sum_t exp(s_t))
 * A row with no position gives out = 0 and lse = -infinity.  Places that a row
 * does not see are never part of its result, whatever they hold; an infinite
 * value in one it sees is the channel's result, two opposite ones NaN (rows
 * with such values are computed again one by one, many times slower).  Scores, sums
 * and the running statistics are fp32; with 16-bit types exp(s - max) enters the
 * product with v rounded to the type, or, of a request with at most 16 new tokens times
 * heads / kv_heads (one that decodes), as two values of it, as in op_paged_attention.
 * head_dim: a multiple of 8, at most 256; heads a multiple of kv_heads;
 * num_pages * kv_heads * page_size and max_pages * page_size + tokens below 2^31,
 * and so is (tokens / n + requests) * (max_pages * page_size / 32 + 1), where n is
 * 64 / (heads / kv_heads), at least 1; the caches start on 16 bytes.
 */
typedef struct lux_paged_chunk_args {
    uint32_t struct_size;
    int32_t requests, tokens, heads, kv_heads, head_dim, page_size, num_pages, max_pages;
    int32_t window;
    int32_t dtype; /* of q, the cache and out: FLOAT32, FLOAT16 or BFLOAT16 */
    float scale, softcap;
    int32_t _pad;
    int64_t q_offset, q_row_stride, out_offset, out_row_stride;
    LuxBackendBuffer* q;            /* [tokens, heads * head_dim] */
    LuxBackendBuffer* k_cache;      /* [num_pages, kv_heads, page_size, head_dim] */
    LuxBackendBuffer* v_cache;
    LuxBackendBuffer* block_table;  /* int32[requests, max_pages] */
    LuxBackendBuffer* token_starts; /* int32[requests + 1] */
    LuxBackendBuffer* seq_lens;     /* int32[requests]: tokens held before the new ones */
    LuxBackendBuffer* kv_lens;      /* int32[requests]: and with them */
    LuxBackendBuffer* out;          /* [tokens, heads * head_dim] */
    LuxBackendBuffer* lse;          /* f32[tokens, heads], or NULL */
} lux_paged_chunk_args;

/*
 * Requests that begin as copies of others.  Fork f, where src[f] and dst[f] are
 * different requests of [0, requests), dst[f] holds nothing (its length is 0 or
 * less) and no fork before f that was made has the same dst: dst gets src's length
 * (before the call) and its pages.  With n that length cut to [0, max_pages *
 * page_size], the n / page_size full pages are shared; for the rest of n dst takes
 * a page of its own from the free list, in the forks' order, and
 *   copy_src[f], copy_dst[f] = the page of src's that holds the rest, the page
 *             taken (for op_paged_copy, on every layer's cache); -1 otherwise
 * Where the list has no page left, dst keeps the full pages alone.  Where src's
 * page is none, so is dst's, and nothing is taken.  Other forks are left out.
 *   counts = {entry of free_pages after the last one taken, columns of full pages
 *             that dsts got (of a page that is none, too), pages needed and not
 *             there, forks left out}
 */
typedef struct lux_paged_fork_args {
    uint32_t struct_size;
    int32_t forks, requests, max_pages, page_size;
    int32_t num_pages;  /* of the pool */
    int32_t free_count; /* entries of free_pages */
    int32_t _pad;
    LuxBackendBuffer* src;         /* int32[forks] */
    LuxBackendBuffer* dst;         /* int32[forks] */
    LuxBackendBuffer* lens;        /* int32[requests], in and out */
    LuxBackendBuffer* block_table; /* int32[requests, max_pages], in and out */
    LuxBackendBuffer* shares;      /* int32[num_pages], in and out */
    LuxBackendBuffer* free_pages;  /* int32[free_count] */
    LuxBackendBuffer* free_head;   /* int32[1] */
    LuxBackendBuffer* copy_src;    /* int32[forks] */
    LuxBackendBuffer* copy_dst;    /* int32[forks] */
    LuxBackendBuffer* counts;      /* int32[4] */
} lux_paged_fork_args;

/*
 * Requests that end or are cut: kv_lens[r] = min(n, max(0, keep_lens[r])) with n
 * = lens[r] cut to [0, max_pages * page_size].  The pages of the columns from
 * ceil(kv_lens / page_size) to ceil(n / page_size) lose a holder each; a page
 * without one goes back to the list.  The pages that go back take the entries
 * right before free_head, in ascending order; where the list has fewer entries
 * there, the lowest pages get none and are lost.  Table entries stay.  kv_lens may
 * be lens itself.  A request cut inside a page that others share does not own the
 * page: new tokens there are theirs too; fork it from one of them instead.
 *   counts = {first entry of free_pages that holds a page, pages that went back,
 *             entries whose page is still held, pages lost}
 */
typedef struct lux_paged_release_args {
    uint32_t struct_size;
    int32_t requests, max_pages, page_size, num_pages, free_count;
    LuxBackendBuffer* lens;        /* int32[requests] */
    LuxBackendBuffer* keep_lens;   /* int32[requests] */
    LuxBackendBuffer* block_table; /* int32[requests, max_pages] */
    LuxBackendBuffer* shares;      /* int32[num_pages], in and out */
    LuxBackendBuffer* free_pages;  /* int32[free_count], in and out */
    LuxBackendBuffer* free_head;   /* int32[1] */
    LuxBackendBuffer* kv_lens;     /* int32[requests] */
    LuxBackendBuffer* counts;      /* int32[4] */
} lux_paged_release_args;

/*
 * Pages that move below a limit, so that the pool can shrink to `limit` pages.
 * Live pages are those that a request names in the columns of its length (cut as
 * above).  The i-th live page from limit on, in ascending order, moves to the i-th
 * page below limit that is not live, for i < moves: all of them, as far as there
 * is room and max_moves allow.
 *   copy_src[i], copy_dst[i] = from and to, -1 from i = moves on (for
 *             op_paged_copy, on every layer's cache: no page is in both)
 *   table_out = the table with the live entries' new names, others as they are;
 *             it may be block_table itself
 *   shares_out = shares, each moved page's at its new place and 0 at its old one;
 *             it may be shares itself
 *   free_pages: the pages below limit that are not live after the moves, in
 *             ascending order, in the last entries of the list (where it is
 *             shorter, the highest of them); entries before them stay
 *   counts = {first of these entries, moves, live pages left from limit on,
 *             live pages}
 * With limit = num_pages nothing moves and the list is made anew.
 */
typedef struct lux_paged_compact_args {
    uint32_t struct_size;
    int32_t requests, max_pages, page_size, num_pages, free_count;
    int32_t limit;     /* 0 .. num_pages */
    int32_t max_moves; /* entries of copy_src and copy_dst */
    LuxBackendBuffer* lens;        /* int32[requests] */
    LuxBackendBuffer* block_table; /* int32[requests, max_pages] */
    LuxBackendBuffer* shares;      /* int32[num_pages] */
    LuxBackendBuffer* table_out;   /* int32[requests, max_pages] */
    LuxBackendBuffer* shares_out;  /* int32[num_pages] */
    LuxBackendBuffer* free_pages;  /* int32[free_count], out */
    LuxBackendBuffer* copy_src;    /* int32[max_moves] */
    LuxBackendBuffer* copy_dst;    /* int32[max_moves] */
    LuxBackendBuffer* counts;      /* int32[4] */
} lux_paged_compact_args;

/*
 * Page copy_dst[i] = page copy_src[i], in the key and the value cache of every
 * layer, for each i < pages with both ids in [0, num_pages).  The pages written
 * are distinct and none of them is read (as a fork's and a compaction's are):
 * otherwise such a page's contents are parts of either.  Layer l's cache
 * is l * layer_stride elements in (0: one pool after the other); a program whose
 * layers' caches are separate buffers calls once per layer.
 */
typedef struct lux_paged_copy_args {
    uint32_t struct_size;
    int32_t pages, layers, kv_heads, head_dim, page_size, num_pages;
    int32_t dtype; /* FLOAT32, FLOAT16 or BFLOAT16 */
    int64_t layer_stride;
    LuxBackendBuffer* copy_src; /* int32[pages] */
    LuxBackendBuffer* copy_dst; /* int32[pages] */
    LuxBackendBuffer* k_cache;  /* [layers][num_pages, kv_heads, page_size, head_dim] */
    LuxBackendBuffer* v_cache;
} lux_paged_copy_args;

/*
 * Scores of a row of logits, x = scale * logits (scale > 0 and finite; x log2(e)
 * of finite logits is finite in fp32):
 *   lse = log(sum_v exp(x_v));  logprobs = x[token] - lse, -infinity for a token
 *   outside [0, vocab);  entropy = lse - sum_v exp(x_v - lse) x_v, terms of
 *   probability 0 left out
 *   top_ids, top_logprobs = the `top` largest logits' places and x - lse, in
 *   descending order, the lowest place first among equals (0 and -0 are equal, NaN
 *   is larger than all and equal to itself)
 * A row of -infinity alone gives lse = -infinity, logprobs -infinity, entropy 0;
 * +infinity or NaN in a row makes its lse that and NaN what the formulas make NaN.
 * Sums and outputs are fp32.  Rows with few finite logits or many alike, where
 * more than 1024 may be among the largest, and rows with NaN are read `top` times more:
 * 4096 rows of 131072 in bf16 with 10 finite logits each take 11 ms for 20
 * alternatives and 33 for 64, with 1 % of them finite 0.22 and 0.43.  A NULL output is left out (tokens may be NULL with
 * logprobs; top_ids and top_logprobs each where top is 0 or it is not wanted).
 * vocab: at least top, at most 2^24; top: 0 to 64.
 */
typedef struct lux_token_logprobs_args {
    uint32_t struct_size;
    int32_t rows, vocab, top;
    int32_t dtype; /* of logits: FLOAT32, FLOAT16 or BFLOAT16 */
    float scale;
    int64_t logits_offset, row_stride;
    LuxBackendBuffer* logits;       /* [rows, vocab] */
    LuxBackendBuffer* tokens;       /* int32[rows], or NULL */
    LuxBackendBuffer* logprobs;     /* f32[rows], or NULL */
    LuxBackendBuffer* entropy;      /* f32[rows], or NULL */
    LuxBackendBuffer* lse;          /* f32[rows], or NULL */
    LuxBackendBuffer* top_ids;      /* int32[rows, top], or NULL */
    LuxBackendBuffer* top_logprobs; /* f32[rows, top], or NULL */
} lux_token_logprobs_args;

typedef struct lux_gpu_prompt_vtbl {
    uint32_t ext_version; /* LUX_GPU_PROMPT_EXT_VERSION */
    uint32_t struct_size; /* sizeof(lux_gpu_prompt_vtbl) of the plugin */

    LuxBackendError (*op_paged_chunk_attention)(LuxBackendContext* ctx, const lux_paged_chunk_args* args);
    LuxBackendError (*op_paged_fork)(LuxBackendContext* ctx, const lux_paged_fork_args* args);
    LuxBackendError (*op_paged_release)(LuxBackendContext* ctx, const lux_paged_release_args* args);
    LuxBackendError (*op_paged_compact)(LuxBackendContext* ctx, const lux_paged_compact_args* args);
    LuxBackendError (*op_paged_copy)(LuxBackendContext* ctx, const lux_paged_copy_args* args);
    LuxBackendError (*op_token_logprobs)(LuxBackendContext* ctx, const lux_token_logprobs_args* args);

    void* _reserved[8];
} lux_gpu_prompt_vtbl;

/* layout pins: LP64 */
#if defined(__LP64__)
#ifdef __cplusplus
static_assert(sizeof(lux_paged_chunk_args) == 160, "chunk record");
static_assert(sizeof(lux_paged_fork_args) == 112, "fork record");
static_assert(sizeof(lux_paged_release_args) == 88, "release record");
static_assert(sizeof(lux_paged_compact_args) == 104, "compact record");
static_assert(sizeof(lux_paged_copy_args) == 72, "copy record");
static_assert(sizeof(lux_token_logprobs_args) == 96, "logprobs record");
static_assert(sizeof(lux_gpu_prompt_vtbl) == 120, "prompt table");
#else
_Static_assert(sizeof(lux_paged_chunk_args) == 160, "chunk record");
_Static_assert(sizeof(lux_paged_fork_args) == 112, "fork record");
_Static_assert(sizeof(lux_paged_release_args) == 88, "release record");
_Static_assert(sizeof(lux_paged_compact_args) == 104, "compact record");
_Static_assert(sizeof(lux_paged_copy_args) == 72, "copy record");
_Static_assert(sizeof(lux_token_logprobs_args) == 96, "logprobs record");
_Static_assert(sizeof(lux_gpu_prompt_vtbl) == 120, "prompt table");
#endif
#endif

#ifdef __cplusplus
}
#endif

#endif /* LUX_GPU_PROMPT_BACKEND_H */
