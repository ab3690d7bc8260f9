// paged_plan.hip -- the pages and slots of a step's new tokens, from the
// requests' lengths.
//
// need_r = min(ceil((seq_r + new_r) / P), columns) - ceil(seq_r / P) pages and
// new_r tokens per request; two exclusive sums over the requests give each
// request's first page in the free list and its first token.  Then one thread
// per token finds its request (the last one that starts at or before it) and
// writes its slot; the token at the start of a page that its request did not
// hold writes the page's table entry: a new page's first token is new itself.
//
// All latency.  Up to kMost requests every block sums them all by itself, into
// LDS, and goes on to its tokens: one launch and two trips to memory (64 requests
// with a token each 3.9 us, 3.2 of them the kernel; 1000 with 16384 tokens 5.1).
// More are summed by a launch of their own.
#include "serving_device.h"

namespace lxq {
namespace {

// where the first new token's page is in the list: 0 before the list
__device__ __forceinline__ int head_of(const PlanArgs& a) { return a.head[0] < 0 ? 0 : a.head[0]; }

struct Request {
    int seq, fresh, have, need;
};
__device__ __forceinline__ Request request_of(const PlanArgs& a, int s, int n) {
    Request q;
    const int cap = a.columns * a.page;  // below 2^31
    q.seq = s < 0 ? 0 : s > cap ? cap : s;
    q.fresh = n < 0 ? 0 : n;
    q.have = div_by(q.seq, a.div);
    if (q.have * a.page < q.seq) q.have++;
    // pages for the tokens that the table has room for
    const int end = q.fresh < cap - q.seq ? q.seq + q.fresh : cap;
    int want = div_by(end, a.div);
    if (want * a.page < end) want++;
    q.need = want - q.have;
    return q;
}

__device__ __forceinline__ Request request_at(const PlanArgs& a, int r) { return request_of(a, a.seq[r], a.fresh[r]); }

// inclusive sums of two values over a block of NW waves; `total`: the block's
template <int NW>
__device__ __forceinline__ void block_scan(int& x, int& y, int& tx, int& ty, int (*part)[2]) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    x = wave_scan(x);
    y = wave_scan(y);
    __syncthreads();  // the last round's readers
    if (lane == 63) { part[w][0] = x; part[w][1] = y; }
    __syncthreads();
    tx = ty = 0;
#pragma unroll
    for (int i = 0; i < NW; i++) {
        if (i < w) { x += part[i][0]; y += part[i][1]; }
        tx += part[i][0];
        ty += part[i][1];
    }
}

// the pages of `need` from list entry `first` on that are there
__device__ __forceinline__ int pages_there(int64_t first, int need, int F) {
    const int64_t left = (int64_t)F - first;
    return left <= 0 ? 0 : left < need ? (int)left : need;
}

__device__ __forceinline__ void write_request(const PlanArgs& a, int r, const Request& q, int start, int64_t first, int& got, int& past) {
    got = pages_there(first, q.need, a.F);
    const int64_t end = (int64_t)q.seq + q.fresh, held = (int64_t)(q.have + got) * a.page;
    const int kv = (int)(end < held ? end : held);
    past = (int)(end - kv);
    a.starts[r] = start;
    a.lens[r] = kv;
}

// token t of request r, whose tokens start at `start` and pages at `first`
__device__ __forceinline__ void write_token(const PlanArgs& a, int t, int r, const Request& q, int start, int64_t first) {
    const int64_t p64 = (int64_t)q.seq + (t - start);
    const int pos = (int)p64;
    const int got = pages_there(first, q.need, a.F);
    int slot = -1;
    if (p64 < (int64_t)(q.have + q.need) * a.page) {
        const int i = div_by(pos, a.div), at = pos - i * a.page;
        int page;
        if (i < q.have) {
            page = a.table[(int64_t)r * a.columns + i];
        } else {
            page = i - q.have < got ? a.free_pages[first + (i - q.have)] : -1;
            if (at == 0) a.table[(int64_t)r * a.columns + i] = page;
        }
        if ((uint32_t)page < (uint32_t)a.pool) slot = page * a.page + at;
    }
    if (t < a.T) {
        a.slots[t] = slot;
        if (a.positions) a.positions[t] = pos;
        if (a.request) a.request[t] = r;
    }
}

__device__ __forceinline__ void write_no_token(const PlanArgs& a, int t) {
    a.slots[t] = -1;
    if (a.positions) a.positions[t] = 0;
    if (a.request) a.request[t] = -1;
}

// one launch for up to kMost requests; thread i sums a stretch of them.  With one
// and with two launches, a token each (32768 tokens take as long): 600 requests 4.7
// and 8.9 us, 1000 5.2 and 8.8, 2048 7.8 and 10.2, 3000 8.0 and 12.1, 4096 11.7 and
// 12.9.  Beyond that the block's LDS (48 KB) and the stretches per thread grow on.
constexpr int kMost = 4096;
__global__ __launch_bounds__(256) void plan_kernel(PlanArgs a) {
    __shared__ int part[4][2];
    __shared__ int starts[kMost + 1], firsts[kMost], seqs[kMost];
    constexpr int kEach = kMost / 256;
    const int each = (a.R + 255) / 256, r0 = (int)threadIdx.x * each;
    const int head = head_of(a);
    int s[kEach], n[kEach];
    auto load = [&](int i) {
        const int r = r0 + i;
        s[i] = r < a.R ? a.seq[r] : 0;
        n[i] = r < a.R ? a.fresh[r] : 0;
    };
    load(0);
    if (each > 1) {  // no branch between them: one trip for all
#pragma unroll
        for (int i = 1; i < kEach; i++) {
            s[i] = n[i] = 0;
            if (i < each) load(i);
        }
    }
    int tokens = 0, pages = 0;
#pragma unroll
    for (int i = 0; i < kEach; i++) {
        if (i >= each) break;
        const Request q = request_of(a, s[i], n[i]);
        tokens += q.fresh;
        pages += q.need;
    }
    int x = tokens, y = pages, all_tokens, all_pages;
    block_scan<4>(x, y, all_tokens, all_pages, part);
    int start = x - tokens, first = y - pages, past_all = 0;
#pragma unroll
    for (int i = 0; i < kEach; i++) {
        if (i >= each) break;
        const int r = r0 + i;
        if (r < a.R) {
            const Request q = request_of(a, s[i], n[i]);
            starts[r] = start;
            firsts[r] = first;
            seqs[r] = q.seq;
            if (blockIdx.x == 0) {
                int got, past;
                write_request(a, r, q, start, (int64_t)head + first, got, past);
                past_all += past;
            }
            start += q.fresh;
            first += q.need;
        }
    }
    if (threadIdx.x == 0) starts[a.R] = all_tokens;
    if (blockIdx.x == 0) {
        int none = 0, tp, tn;
        block_scan<4>(past_all, none, tp, tn, part);
        if (threadIdx.x == 0) {
            const int got = pages_there(head, all_pages, a.F);
            a.starts[a.R] = all_tokens;
            a.counts[0] = head + got;
            a.counts[1] = all_tokens;
            a.counts[2] = all_pages - got;
            a.counts[3] = tp;
        }
    }
    __syncthreads();
    const int64_t most = all_tokens > a.T ? all_tokens : a.T, step = (int64_t)gridDim.x * 256;
    for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < most; t += step) {
        if (t >= all_tokens) {
            write_no_token(a, (int)t);
            continue;
        }
        int lo = 0, hi = a.R - 1;  // the last request that starts at or before t: none after it is empty
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (starts[mid] <= (int)t) lo = mid;
            else hi = mid - 1;
        }
        write_token(a, (int)t, lo, request_of(a, seqs[lo], starts[lo + 1] - starts[lo]), starts[lo], (int64_t)head + firsts[lo]);
    }
}

// more requests, first launch: one block walks the requests
__global__ __launch_bounds__(1024) void plan_requests_kernel(PlanArgs a) {
    __shared__ int part[16][2];
    const int head = head_of(a);
    int tokens = 0;
    int64_t pages = 0;
    int got_all = 0, past_all = 0;
    for (int r0 = 0; r0 < a.R; r0 += 1024) {
        const int r = r0 + (int)threadIdx.x;
        Request q = {0, 0, 0, 0};
        if (r < a.R) q = request_at(a, r);
        int x = q.fresh, y = q.need, tx, ty;
        block_scan<16>(x, y, tx, ty, part);
        if (r < a.R) {
            const int64_t first = head + pages + (y - q.need);
            int got, past;
            write_request(a, r, q, tokens + x - q.fresh, first, got, past);
            a.ws[r] = (int)(pages + (y - q.need));
            got_all += got;
            past_all += past;
        }
        tokens += tx;
        pages += ty;
    }
    int tg, tp;
    block_scan<16>(got_all, past_all, tg, tp, part);
    if (threadIdx.x == 0) {
        a.starts[a.R] = tokens;
        a.counts[0] = head + tg;
        a.counts[1] = tokens;
        a.counts[2] = (int)(pages - tg);
        a.counts[3] = tp;
    }
}

// second launch: a thread per token
__global__ __launch_bounds__(256) void plan_tokens_kernel(PlanArgs a) {
    const int head = head_of(a);
    const int total = a.starts[a.R];
    const int64_t most = total > a.T ? total : a.T, step = (int64_t)gridDim.x * 256;
    for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < most; t += step) {
        if (t >= total) {
            write_no_token(a, (int)t);
            continue;
        }
        int lo = 0, hi = a.R - 1;  // the last request that starts at or before t: none after it is empty
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (a.starts[mid] <= (int)t) lo = mid;
            else hi = mid - 1;
        }
        write_token(a, (int)t, lo, request_at(a, lo), a.starts[lo], (int64_t)head + a.ws[lo]);
    }
}

}  // namespace

LuxStatus launch_paged_plan(const PlanArgs& a, hipStream_t st) {
    const int blocks = a.T < 256 * 1024 ? (a.T + 255) / 256 : 1024;
    const dim3 g(blocks < 1 ? 1 : blocks);
    if (a.R <= kMost) {
        hipLaunchKernelGGL(plan_kernel, g, dim3(256), 0, st, a);
    } else {
        if ((size_t)a.R > a.ws_words) return LuxStatus::NotSupported;
        hipLaunchKernelGGL(plan_requests_kernel, dim3(1), dim3(1024), 0, st, a);
        hipLaunchKernelGGL(plan_tokens_kernel, g, dim3(256), 0, st, a);
    }
    return hipGetLastError() == hipSuccess ? LuxStatus::Ok : LuxStatus::Internal;
}

}  // namespace lxq
