// prompt.h -- launchers of the kernels of prompts and of pages in use (chunk
// attention, fork, release, compaction and copy of pages, token log
// probabilities).  prompt_ops.hip validates sizes, buffers and overlaps before it
// calls these; every pointer is the first element used.
#pragma once
#include "serving.h"

namespace lxq {

// partial results of the chunk attention: two per range, one range per CU, each up
// to 256 rows of 192 channels (or of fewer, or 128 of 256) and their maxima and
// sums; and a record per range
constexpr int kChunkRanges = 256;
constexpr size_t kChunkPartBytes = (size_t)kChunkRanges * (2 * 256 * (192 + 2) * 4 + 32);

struct ChunkArgs {
    const void *q, *kc, *vc;
    const int32_t *table, *starts, *seq, *lens;
    void* out;
    float* lse;
    int R, T, H, Hk, G, D, page, pool, columns, window, dtype;
    float scale, softcap;
    int64_t q_row, out_row;
    DivBy div;
    char* ws;  // kChunkPartBytes
    int cus;
};
LuxStatus launch_paged_chunk(const ChunkArgs& a, hipStream_t st);

struct ForkArgs {
    const int32_t *src, *dst, *free_pages, *head;
    int32_t *lens, *table, *shares, *copy_src, *copy_dst, *counts;
    int F, R, columns, page, pool, free_count;
    DivBy div;
    int32_t* ws;  // 2 F words
    size_t ws_words;
};
LuxStatus launch_paged_fork(const ForkArgs& a, hipStream_t st);

struct ReleaseArgs {
    const int32_t *lens, *keep, *table, *head;
    int32_t *shares, *free_pages, *kv, *counts;
    int R, columns, page, pool, free_count;
    DivBy div;
    int32_t* ws;  // 512 words, and one per 4096 pages
    size_t ws_words;
};
LuxStatus launch_paged_release(const ReleaseArgs& a, hipStream_t st);

struct CompactArgs {
    const int32_t *lens, *table, *shares;
    int32_t *table_out, *shares_out, *free_pages, *copy_src, *copy_dst, *counts;
    int R, columns, page, pool, free_count, limit, max_moves;
    DivBy div, by_columns;
    int32_t* ws;  // a bit and a word per page
    size_t ws_words;
};
LuxStatus launch_paged_compact(const CompactArgs& a, hipStream_t st);

struct CopyArgs {
    const int32_t *src, *dst;
    void *kc, *vc;
    int n, layers, pool;
    int64_t page_bytes, layer_bytes;
    int esz;
};
LuxStatus launch_paged_copy(const CopyArgs& a, hipStream_t st);

struct LogprobArgs {
    const void* logits;
    const int32_t* tokens;
    float *logprobs, *entropy, *lse, *top_lp;
    int32_t* top_ids;
    int T, V, top, dtype;
    float scale;
    int64_t row;
    char* ws;
    size_t ws_bytes;
    uint32_t* count;  // `counts` counters, zero between launches
    int counts;
    int cus;
};
LuxStatus launch_token_logprobs(const LogprobArgs& a, hipStream_t st);

}  // namespace lxq
