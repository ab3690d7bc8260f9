// serving.h -- launchers of the decoding step's kernels (paged plan, append,
// attention, block norm).  serving_ops.hip validates sizes, buffers and
// overlaps before it calls these; every pointer is the first element used.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kernels.h"

namespace lxq {

// the words of a context's workspace that the GEMMs keep between launches
// (qsplit.h); what lies behind them holds nothing from one launch to the next
constexpr size_t kWorkspaceWords = 4096;

// t / d for 0 <= t < 2^31 as (t * mul) >> (31 + sh): sh = ceil(log2 d), mul =
// ceil(2^(31 + sh) / d) < 2^33 exceeds the quotient's factor by less than
// 2^-31 / d per unit of t
struct DivBy {
    uint64_t mul;
    int sh, d;
    DivBy(int by = 1) : sh(0), d(by) {
        while ((1ll << sh) < by) sh++;
        mul = ((1ull << (31 + sh)) + (uint64_t)by - 1) / (uint64_t)by;
    }
};

// A launch has fewer than 2^32 threads (with more, those past a multiple of it run
// and no error is reported): more blocks of `threads` go in several, launch(first,
// blocks) each
template <class F>
void launch_blocks(int64_t blocks, int threads, F launch) {
    const int64_t most = (1ll << 31) / threads;
    for (int64_t first = 0; first < blocks; first += most)
        launch((int)first, (unsigned)(blocks - first < most ? blocks - first : most));
}

struct PlanArgs {
    const int32_t *seq, *fresh, *free_pages, *head;
    int32_t *table, *slots, *positions, *request, *starts, *lens, *counts;
    int R, T, columns, page, pool, F;
    DivBy div;
    int32_t* ws;  // R words, for the two-launch form
    size_t ws_words;
};
LuxStatus launch_paged_plan(const PlanArgs& a, hipStream_t st);

struct AppendArgs {
    const void *k, *v;
    const int32_t* slots;
    void *kc, *vc;
    int T, Hk, D, page, pool, in_dt, cache_dt;
    int64_t k_row, v_row;
    DivBy div;
};
LuxStatus launch_paged_append(const AppendArgs& a, hipStream_t st);

struct AttnArgs {
    const void *q, *kc, *vc;
    const int32_t *table, *lens;
    void* out;
    float* lse;
    int R, H, Hk, G, D, page, pool, columns, window, dtype;
    float scale, softcap;
    int64_t q_row, out_row;
    DivBy div;
    float* ws;  // partial results
    size_t ws_bytes;
    uint32_t* count;  // `counts` words, zero between launches
    int counts;
    int cus;
};
LuxStatus launch_paged_attention(const AttnArgs& a, hipStream_t st);

struct NormArgs {
    const void *x, *r, *pw, *pb, *gate, *nw, *nb;
    void *h, *out;
    int T, D, post, pre, gate_mode, x_dt, r_dt, w_dt;
    float rscale, eps;
    int64_t x_row, r_row, g_row, h_row, o_row;
};
LuxStatus launch_block_norm(const NormArgs& a, hipStream_t st);

}  // namespace lxq
