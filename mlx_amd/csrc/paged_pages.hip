// paged_pages.hip -- pages in use: forks that share them, pages given back,
// compaction of a pool, and copies of their contents.
//
// All but the copies is whole numbers and latency.  What decides an order (which
// fork takes which page, where a page goes back to in the list) is a sum over
// forks or pages in their own order, never the order in which threads arrive: equal
// calls give equal results.  What bounds them is the number of launches and of trips
// to memory in a row, so that each loads as much as it can before it waits: 64
// requests of up to 256 pages given back in 10.4 us (three launches), 2048 of up to
// 128 in 12.4, 24 forks with their copies and a release in 18.4, 37 requests of up to
// 42 pages compacted in 5.0 and the pages copied in 6.5.  The one block that numbers a
// larger pool's moves goes through its bits in order: 72 us of 88 for 164450 pages,
// 65000 of them live.  The copies are bound by HBM: 0.87 GB read and written in 336 us,
// 5.2 TB/s.
#include "serving_device.h"
#include "prompt.h"

namespace lxq {
namespace {

typedef uint32_t u4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ int load_now(const int32_t* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ void store_now(int32_t* p, int v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ int add_now(int32_t* p, int v) { return __hip_atomic_fetch_add(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

__device__ __forceinline__ int cut(int n, int cap) { return n < 0 ? 0 : n > cap ? cap : n; }
__device__ __forceinline__ int pages_of(int n, const DivBy& div) {
    const int full = div_by(n, div);
    return full * div.d < n ? full + 1 : full;
}

// exclusive sum of v over the block's NW waves; `all`: the block's sum
template <int NW>
__device__ __forceinline__ int block_sum(int v, int& all, int* part) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int through = wave_scan(v);
    __syncthreads();  // the last round's readers
    if (lane == 63) part[w] = through;
    __syncthreads();
    int before = through - v;
    all = 0;
#pragma unroll
    for (int i = 0; i < NW; i++) {
        if (i < w) before += part[i];
        all += part[i];
    }
    return before;
}

// the same of N values at once: v becomes the sums before
template <int NW, int N>
__device__ __forceinline__ void block_sums(int (&v)[N], int (&all)[N], int (*part)[N]) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; k++) {
        const int through = wave_scan(v[k]);
        if (lane == 63) part[w][k] = through;
        v[k] = through - v[k];
        all[k] = 0;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NW; i++)
#pragma unroll
        for (int k = 0; k < N; k++) {
            const int x = part[i][k];
            if (i < w) v[k] += x;
            all[k] += x;
        }
}

// --- fork -----------------------------------------------------------------------------

// A wave: the table's entries of a fork that shares `full` pages of row s, four
// columns a lane at a time
__device__ __forceinline__ void fork_columns(const ForkArgs& a, int s, int d, int full) {
    const int32_t* from = a.table + (int64_t)s * a.columns;
    int32_t* to = a.table + (int64_t)d * a.columns;
    const int lane = threadIdx.x & 63;
    for (int c = lane; c < full; c += 256) {
        int id[4];
#pragma unroll
        for (int i = 0; i < 4; i++) id[i] = c + 64 * i < full ? from[c + 64 * i] : -1;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (c + 64 * i < full) to[c + 64 * i] = id[i];
            if ((uint32_t)id[i] < (uint32_t)a.pool) add_now(a.shares + id[i], 1);
        }
    }
}

// a fork of n tokens (below 0: not made) of which the last are not a whole page: the
// page for them, of which the forks before took those up to `at`.  `last`: the
// source's entry
struct Taken {
    int entry;   // after the full pages' ones, any number
    bool rest;   // there is one
    int n;       // tokens that it holds
    bool there;  // a page was needed and there
};
__device__ __forceinline__ Taken take_page(const ForkArgs& a, int f, int n, int full, int last, int at, int& all, int* part) {
    const bool rest = n > full * a.page;
    const bool take = rest && (uint32_t)last < (uint32_t)a.pool;
    at += block_sum<16>(take ? 1 : 0, all, part);
    const bool there = take && at < a.free_count;
    const int page = there ? a.free_pages[at] : -1;
    if (f < a.F) {
        a.copy_src[f] = there ? last : -1;
        a.copy_dst[f] = page;
    }
    return Taken{take ? page : last, rest, take && !there ? full * a.page : n, there};
}
__device__ __forceinline__ void fork_counts(const ForkArgs& a, int head, int taken, int shared, int out, int needed) {
    a.counts[0] = head + taken;
    a.counts[1] = shared;
    a.counts[2] = needed - taken;
    a.counts[3] = out;
}

// One block, a thread per fork: which forks are made (the first one of its dst is),
// and the pages they take.  ALL: the table too, in the same launch.
template <bool ALL>
__global__ __launch_bounds__(1024) void fork_few_kernel(ForkArgs a) {
    __shared__ __attribute__((aligned(16))) int dsts[1024];
    __shared__ int part[16], parts[16][3], rows[ALL ? 1024 : 1][3];
    const int cap = a.columns * a.page, f = threadIdx.x, head = cut(a.head[0], a.free_count);
    const int s = f < a.F ? a.src[f] : -1, d = f < a.F ? a.dst[f] : -1;
    bool made = (uint32_t)s < (uint32_t)a.R && (uint32_t)d < (uint32_t)a.R && s != d;
    const int held = made ? a.lens[s] : 0, has = made ? a.lens[d] : 0;
    made = made && has <= 0;
    dsts[f] = made ? d : -1;
    __syncthreads();
    // the forks before the wave's last one, without branches (which took 20 us for 224 forks)
    const int end = __builtin_amdgcn_readfirstlane(f < a.F ? f + 64 : 0);
    int twice = 0;
#pragma unroll 4
    for (int g = 0; g < end; g += 4) {
        const u4 x = *reinterpret_cast<const u4*>(dsts + g);
#pragma unroll
        for (int i = 0; i < 4; i++) twice |= (g + i < f) & ((int)x[i] == d);
    }
    made = made && !twice;
    const int n = made ? cut(held, cap) : -1, full = made ? div_by(n, a.div) : 0;
    const int last = n > full * a.page ? a.table[(int64_t)s * a.columns + full] : -1;
    if constexpr (ALL) {
        rows[f][0] = s;
        rows[f][1] = d;
        rows[f][2] = full;
        __syncthreads();
        for (int g = f >> 6; g < a.F; g += 16) fork_columns(a, rows[g][0], rows[g][1], rows[g][2]);
    }
    int needed;
    const Taken t = take_page(a, f, n, full, last, head, needed, part);
    int v[3] = {t.there, full, f < a.F && !made}, all[3];
    block_sums<16, 3>(v, all, parts);
    if (made) a.lens[d] = t.n;
    if (f == 0) fork_counts(a, head, all[0], all[1], all[2], needed);
    if constexpr (ALL) {
        if (t.rest) a.table[(int64_t)d * a.columns + full] = t.entry;
    } else if (f < a.F) {
        a.ws[f] = t.rest ? ~full : full;
        a.ws[a.F + f] = t.entry;
    }
}

// One block, for more forks than threads: each writes its number, below 0, as its
// dst's length, and the lowest stays.
__global__ __launch_bounds__(1024) void fork_kernel(ForkArgs a) {
    __shared__ int part[16], parts[16][3];
    const int cap = a.columns * a.page, tid = threadIdx.x, head = cut(a.head[0], a.free_count);
    for (int f = tid; f < a.F; f += 1024) {
        const int s = a.src[f], d = a.dst[f];
        const bool ok = (uint32_t)s < (uint32_t)a.R && (uint32_t)d < (uint32_t)a.R && s != d && load_now(a.lens + d) <= 0;
        a.ws[f] = ok ? cut(load_now(a.lens + s), cap) : -1;
    }
    __syncthreads();
    for (int f = tid; f < a.F; f += 1024)
        if (a.ws[f] >= 0) store_now(a.lens + a.dst[f], 0);
    __syncthreads();
    for (int f = tid; f < a.F; f += 1024)
        if (a.ws[f] >= 0) __hip_atomic_fetch_min(a.lens + a.dst[f], f - a.F, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    int v[3] = {0, 0, 0}, all[3], needed = 0;
    for (int f0 = 0; f0 < a.F; f0 += 1024) {
        const int f = f0 + tid;
        const int n = f < a.F ? a.ws[f] : -1;
        const int d = n >= 0 ? a.dst[f] : 0;
        const bool made = n >= 0 && load_now(a.lens + d) == f - a.F;
        int round;
        const int full = made ? div_by(n, a.div) : 0;
        const int last = made && n > full * a.page ? a.table[(int64_t)a.src[f] * a.columns + full] : -1;
        const Taken t = take_page(a, f, made ? n : -1, full, last, head + needed, round, part);
        needed += round;
        if (f < a.F) {
            a.ws[f] = t.rest ? ~full : full;
            a.ws[a.F + f] = t.entry;
        }
        if (made) store_now(a.lens + d, t.n);
        v[0] += t.there;
        v[1] += full;
        v[2] += f < a.F && !made;
    }
    block_sums<16, 3>(v, all, parts);
    if (tid == 0) fork_counts(a, head, all[0], all[1], all[2], needed);
}

// a wave per fork: ws holds its full pages, below 0 (~full) where an entry follows them
__global__ __launch_bounds__(256) void fork_table_kernel(ForkArgs a) {
    for (int64_t f = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); f < a.F; f += (int64_t)gridDim.x * 4) {
        const int is = a.ws[f], entry = a.ws[a.F + f], full = is < 0 ? ~is : is;
        if (full > 0) fork_columns(a, a.src[f], a.dst[f], full);
        if (is < 0 && (threadIdx.x & 63) == 0) a.table[(int64_t)a.dst[f] * a.columns + full] = entry;
    }
}

// --- release --------------------------------------------------------------------------

constexpr int kDropBlocks = 512, kRun = 4096;  // blocks that drop entries; pages of a run

// A wave: request r's pages behind what it keeps lose a holder, and a page that had
// one alone counts -1 until the list has it.  Four columns a lane, so that a trip to
// the table and one to the counts serve 256.  `back`: pages that go back; returns
// the entries
__device__ __forceinline__ int drop(const ReleaseArgs& a, int r, int& back) {
    const int n = cut(a.lens[r], a.columns * a.page), k = a.keep[r];
    const int kept = k < 0 ? 0 : k < n ? k : n;
    const int c1 = pages_of(n, a.div);
    const int32_t* row = a.table + (int64_t)r * a.columns;
    int entries = 0;
    for (int c = pages_of(kept, a.div) + ((int)threadIdx.x & 63); c < c1; c += 256) {
        int id[4], had[4];
#pragma unroll
        for (int i = 0; i < 4; i++) id[i] = c + 64 * i < c1 ? row[c + 64 * i] : -1;
#pragma unroll
        for (int i = 0; i < 4; i++) had[i] = (uint32_t)id[i] < (uint32_t)a.pool ? add_now(a.shares + id[i], -1) : 1;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            entries += (uint32_t)id[i] < (uint32_t)a.pool;
            back += had[i] == 0;
        }
    }
    return entries;
}
__device__ __forceinline__ void write_kept(const ReleaseArgs& a, int r) {
    const int n = cut(a.lens[r], a.columns * a.page), k = a.keep[r];
    a.kv[r] = k < 0 ? 0 : k < n ? k : n;
}

// four pages of a thread: their counts, how many of them go back (a count below 0),
// and their entries of the list from `to` on (below 0: lost; none from `head` on,
// whatever counts the caller had)
struct Four {
    int p, v[4];
    __device__ __forceinline__ Four(const ReleaseArgs& a, int run) : p(run * kRun + 4 * (int)threadIdx.x) {
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = p + i < a.pool ? load_now(a.shares + p + i) : 0;
    }
    __device__ __forceinline__ int back() const { return (v[0] < 0) + (v[1] < 0) + (v[2] < 0) + (v[3] < 0); }
    __device__ __forceinline__ void give(const ReleaseArgs& a, int to, int head) const {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (v[i] < 0) {
                if (to >= 0 && to < head) a.free_pages[to] = p + i;
                to++;
                a.shares[p + i] = 0;
            }
    }
};
__device__ __forceinline__ void release_counts(const ReleaseArgs& a, int head, int back, int entries) {
    a.counts[0] = head > back ? head - back : 0;
    a.counts[1] = back;
    a.counts[2] = entries - back;
    a.counts[3] = back > head ? back - head : 0;
}

// one block for small pools
__global__ __launch_bounds__(1024) void release_kernel(ReleaseArgs a) {
    __shared__ int part[16], parts[16][2];
    const int tid = threadIdx.x, head = cut(a.head[0], a.free_count);
    int v[2] = {0, 0}, all[2];
    for (int r = tid >> 6; r < a.R; r += 16) v[1] += drop(a, r, v[0]);
    block_sums<16, 2>(v, all, parts);
    for (int r = tid; r < a.R; r += 1024) write_kept(a, r);  // kv may be lens: all have read them
    int at = head - all[0];
    for (int run = 0; run * kRun < a.pool; run++) {
        const Four pages(a, run);
        int back;
        const int to = at + block_sum<16>(pages.back(), back, part);
        pages.give(a, to, head);
        at += back;
    }
    if (tid == 0) release_counts(a, head, all[0], all[1]);
}

// three launches: entries per block into ws, pages that go back per run into ws
// behind them, the list
__global__ __launch_bounds__(256) void release_drop_kernel(ReleaseArgs a) {
    __shared__ int part[4];
    int back = 0, entries = 0, all;
    for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < a.R; r += (int64_t)gridDim.x * 4) {
        entries += drop(a, (int)r, back);
        if ((threadIdx.x & 63) == 0) write_kept(a, (int)r);
    }
    block_sum<4>(entries, all, part);
    if (threadIdx.x == 0) a.ws[blockIdx.x] = all;
}
__global__ __launch_bounds__(1024) void release_count_kernel(ReleaseArgs a) {
    __shared__ int part[16];
    int all;
    block_sum<16>(Four(a, blockIdx.x).back(), all, part);
    if (threadIdx.x == 0) a.ws[kDropBlocks + blockIdx.x] = all;
}
__global__ __launch_bounds__(1024) void release_list_kernel(ReleaseArgs a, int drops, int runs) {
    __shared__ int parts[16][4];
    const int tid = threadIdx.x, head = cut(a.head[0], a.free_count);
    const Four pages(a, blockIdx.x);
    // pages that go back in this run; in all, and before this run; entries
    int v[4] = {pages.back(), 0, 0, tid < drops ? a.ws[tid] : 0}, all[4];
    for (int i = tid; i < runs; i += 1024) {
        const int n = a.ws[kDropBlocks + i];
        v[1] += n;
        v[2] += i < (int)blockIdx.x ? n : 0;
    }
    block_sums<16, 4>(v, all, parts);
    pages.give(a, head - all[1] + all[2] + v[0], head);
    if (blockIdx.x == 0 && tid == 0) release_counts(a, head, all[1], all[3]);
}

// --- compaction -----------------------------------------------------------------------

// ws: a bit per page (live), then a word per page (the new name of a live page from
// the limit on, -1 where it stays)
__device__ __forceinline__ int words_of(int pool) { return (pool + 31) / 32; }

__global__ __launch_bounds__(256) void compact_clear_kernel(CompactArgs a) {
    const int64_t n = a.pool, step = (int64_t)gridDim.x * 256;
    for (int64_t p = (int64_t)blockIdx.x * 256 + threadIdx.x; p < n; p += step) {
        if (p < words_of(a.pool)) a.ws[p] = 0;
        if (a.shares_out != a.shares) a.shares_out[p] = a.shares[p];
    }
}
// a wave per request
__global__ __launch_bounds__(256) void compact_mark_kernel(CompactArgs a) {
    for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < a.R; r += (int64_t)gridDim.x * 4) {
        const int held = pages_of(cut(a.lens[r], a.columns * a.page), a.div);
        for (int c = threadIdx.x & 63; c < held; c += 64) {
            const int id = a.table[r * a.columns + c];
            if ((uint32_t)id < (uint32_t)a.pool)
                __hip_atomic_fetch_or(reinterpret_cast<uint32_t*>(a.ws) + (id >> 5), 1u << (id & 31), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    }
}
// one block: a thread takes a stretch of words
__global__ __launch_bounds__(1024) void compact_moves_kernel(CompactArgs a) {
    __shared__ int part[16];
    const int tid = threadIdx.x, words = words_of(a.pool), each = (words + 1023) / 1024;
    const int w0 = tid * each, w1 = w0 + each < words ? w0 + each : words;
    const uint32_t* bits = reinterpret_cast<const uint32_t*>(a.ws);
    int32_t* name = a.ws + words;
    // bits of word w that stand for pages below the limit
    auto low = [&](int w) { return 32 * w + 32 <= a.limit ? ~0u : 32 * w >= a.limit ? 0u : (1u << (a.limit & 31)) - 1u; };
    int high_mine = 0, room_mine = 0, live_mine = 0;
    for (int w = w0; w < w1; w++) {
        const uint32_t b = bits[w], l = low(w);
        live_mine += __popc(b);
        high_mine += __popc(b & ~l);
        room_mine += __popc(~b & l);
    }
    int high, room, live;
    int hi = block_sum<16>(high_mine, high, part), lo = block_sum<16>(room_mine, room, part);
    block_sum<16>(live_mine, live, part);
    int moves = high < room ? high : room;
    moves = moves < a.max_moves ? moves : a.max_moves;
    const int left = room - moves, first = a.free_count - left;
    for (int w = w0; w < w1; w++) {
        const uint32_t b = bits[w], l = low(w);
        for (uint32_t x = b & ~l; x; x &= x - 1, hi++) {
            const int id = 32 * w + __builtin_ctz(x);
            if (hi < moves) a.copy_src[hi] = id;
            else name[id] = -1;
        }
        for (uint32_t x = ~b & l; x; x &= x - 1, lo++) {
            const int id = 32 * w + __builtin_ctz(x);
            if (lo < moves) a.copy_dst[lo] = id;
            else if (first + lo - moves >= 0) a.free_pages[first + lo - moves] = id;
        }
    }
    for (int i = moves + tid; i < a.max_moves; i += 1024) a.copy_src[i] = a.copy_dst[i] = -1;
    __syncthreads();
    for (int i = tid; i < moves; i += 1024) {
        const int from = a.copy_src[i], to = a.copy_dst[i];
        name[from] = to;
        a.shares_out[to] = a.shares[from];
        a.shares_out[from] = 0;
    }
    if (tid == 0) {
        a.counts[0] = first > 0 ? first : 0;
        a.counts[1] = moves;
        a.counts[2] = high - moves;
        a.counts[3] = live;
    }
}
__global__ __launch_bounds__(256) void compact_table_kernel(CompactArgs a) {
    const int32_t* name = a.ws + words_of(a.pool);
    for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < a.R; r += (int64_t)gridDim.x * 4) {
        const int held = pages_of(cut(a.lens[r], a.columns * a.page), a.div);
        const int n = a.table_out == a.table ? held : a.columns;
        for (int c = threadIdx.x & 63; c < n; c += 64) {
            int id = a.table[r * a.columns + c];
            if (c < held && id >= a.limit && id < a.pool && name[id] >= 0) id = name[id];
            a.table_out[r * a.columns + c] = id;
        }
    }
}

// The same in one block, for pools of up to kFewPages and tables of up to kFewEntries:
// the bits, the ranks before each word and the new names stay in LDS, the table's
// entries in registers.
constexpr int kFewPages = 8192, kFewEntries = 16384;
__global__ __launch_bounds__(1024) void compact_few_kernel(CompactArgs a) {
    constexpr int W = kFewPages / 32, EACH = kFewEntries / 1024;
    __shared__ uint32_t bits[W];
    __shared__ int before[W][2], to[kFewPages], parts[16][3];
    const int tid = threadIdx.x, entries = a.R * a.columns, cap = a.columns * a.page;
    if (tid < W) bits[tid] = 0;
    if (a.shares_out != a.shares)
        for (int p = tid; p < a.pool; p += 1024) a.shares_out[p] = a.shares[p];
    __syncthreads();
    int id[EACH];
    uint32_t held = 0;
#pragma unroll
    for (int k = 0; k < EACH; k++) {
        const int x = tid + 1024 * k;
        id[k] = x < entries ? a.table[x] : -1;
    }
#pragma unroll
    for (int k = 0; k < EACH; k++) {
        const int x = tid + 1024 * k;
        if (x >= entries) break;
        const int r = div_by(x, a.by_columns), c = x - r * a.columns;
        const bool in = c < pages_of(cut(a.lens[r], cap), a.div);
        held |= (uint32_t)in << k;
        if (in && (uint32_t)id[k] < (uint32_t)a.pool) atomicOr(bits + (id[k] >> 5), 1u << (id[k] & 31));
    }
    __syncthreads();
    // of word w: live pages from the limit on, and places below it
    auto low = [&](int w) { return 32 * w + 32 <= a.limit ? ~0u : 32 * w >= a.limit ? 0u : (1u << (a.limit & 31)) - 1u; };
    int v[3] = {0, 0, 0}, all[3];
    if (tid < W) {
        const uint32_t b = bits[tid], l = low(tid);
        v[0] = __popc(b & ~l);
        v[1] = __popc(~b & l);
        v[2] = __popc(b);
    }
    block_sums<16, 3>(v, all, parts);
    if (tid < W) {
        before[tid][0] = v[0];
        before[tid][1] = v[1];
    }
    const int high = all[0], room = all[1];
    int moves = high < room ? high : room;
    moves = moves < a.max_moves ? moves : a.max_moves;
    const int first = a.free_count - (room - moves);
    __syncthreads();
    auto rank_high = [&](int p) { return before[p >> 5][0] + __popc(bits[p >> 5] & ~low(p >> 5) & ((1u << (p & 31)) - 1u)); };
    for (int p = tid; p < a.limit; p += 1024) {
        const uint32_t b = bits[p >> 5];
        if ((b >> (p & 31)) & 1) continue;
        const int at = before[p >> 5][1] + __popc(~b & ((1u << (p & 31)) - 1u));
        if (at < moves) {
            a.copy_dst[at] = p;
            to[at] = p;
        } else if (first + at - moves >= 0) {
            a.free_pages[first + at - moves] = p;
        }
    }
    for (int i = moves + tid; i < a.max_moves; i += 1024) a.copy_src[i] = a.copy_dst[i] = -1;
    __syncthreads();
    for (int p = a.limit + tid; p < a.pool; p += 1024) {
        if (!((bits[p >> 5] >> (p & 31)) & 1)) continue;
        const int at = rank_high(p);
        if (at >= moves) continue;
        a.copy_src[at] = p;
        a.shares_out[to[at]] = a.shares[p];
        a.shares_out[p] = 0;
    }
#pragma unroll
    for (int k = 0; k < EACH; k++) {
        const int x = tid + 1024 * k;
        if (x >= entries) break;
        const bool in = (held >> k) & 1;
        int now = id[k];
        if (in && now >= a.limit && now < a.pool) {
            const int at = rank_high(now);
            if (at < moves) now = to[at];
        }
        if (now != id[k] || a.table_out != a.table) a.table_out[x] = now;
    }
    if (tid == 0) {
        a.counts[0] = first > 0 ? first : 0;
        a.counts[1] = moves;
        a.counts[2] = high - moves;
        a.counts[3] = all[2];
    }
}

// --- copy -----------------------------------------------------------------------------

constexpr int kPiece = 16384;  // bytes of a block

// Pieces of a page, pages, then matrices (keys and values of each layer): blocks that
// run together stay within a matrix, whose pages lie close (4096 pages' contents in
// 16 layers: 342 us against 369 with the matrices of a page one after the other)
template <class V>
__global__ __launch_bounds__(256) void copy_kernel(CopyArgs a, int first, int pieces) {
    const uint32_t b = (uint32_t)first + blockIdx.x, pair = b / (uint32_t)pieces, piece = b - pair * (uint32_t)pieces;
    const uint32_t m = pair / (uint32_t)a.n, i = pair - m * (uint32_t)a.n;
    const int from = a.src[i], to = a.dst[i];
    if ((uint32_t)from >= (uint32_t)a.pool || (uint32_t)to >= (uint32_t)a.pool || from == to) return;
    char* base = static_cast<char*>(m & 1 ? a.vc : a.kc) + (int64_t)(m >> 1) * a.layer_bytes;
    const int64_t at = (int64_t)piece * kPiece, left = a.page_bytes - at;
    const int n = (int)(left < kPiece ? left : kPiece);
    const char* s = base + from * a.page_bytes + at;
    char* d = base + to * a.page_bytes + at;
    constexpr int kEach = sizeof(V) == 16 ? kPiece / (256 * 16) : 8;
    for (int x0 = threadIdx.x * (int)sizeof(V); x0 < n; x0 += kEach * 256 * (int)sizeof(V)) {
        V v[kEach];
#pragma unroll
        for (int k = 0; k < kEach; k++) {
            const int x = x0 + k * 256 * (int)sizeof(V);
            if (x < n) v[k] = *reinterpret_cast<const V*>(s + x);
        }
#pragma unroll
        for (int k = 0; k < kEach; k++) {
            const int x = x0 + k * 256 * (int)sizeof(V);
            if (x < n) *reinterpret_cast<V*>(d + x) = v[k];
        }
    }
}

LuxStatus status() { return hipGetLastError() == hipSuccess ? LuxStatus::Ok : LuxStatus::Internal; }
unsigned blocks_of(int64_t items, int per, int most) {
    const int64_t b = (items + per - 1) / per;
    return (unsigned)(b < 1 ? 1 : b < most ? b : most);
}

}  // namespace

LuxStatus launch_paged_fork(const ForkArgs& a, hipStream_t st) {
    if (!a.ws || (size_t)a.F * 2 > a.ws_words) return LuxStatus::NotSupported;
    // A wave of the one block takes its forks one after the other, in rounds of 256
    // columns; a second launch costs 2 to 3 us and has a wave for each.  Rows that are full,
    // one launch against two: 16 forks of 64 columns 5.6 us, 8.6; 16 of 256 8.0, 9.0; 24 of 257
    // 11.1, 9.4; 32 of 256 14.5, 9.2; 64 of 256 28, 9.3; 64 of 32 7.5, 8.0; 128 of 32 12, 9.1.  A
    // table is wider than most of its rows are long: half full on average, with the copies
    // and the release behind, 24 of 257 take 20.9 us, 21.7; 32 of 257 22.0 both; 48 of 257
    // 24.2, 22.3; 64 of 129 22.4, 22.8; 16 of 1025 31.8, 28.3.
    if (a.F <= 64 && (int64_t)a.F * a.columns <= 8192) {
        hipLaunchKernelGGL(fork_few_kernel<true>, dim3(1), dim3(1024), 0, st, a);
        return status();
    }
    if (a.F <= 1024) hipLaunchKernelGGL(fork_few_kernel<false>, dim3(1), dim3(1024), 0, st, a);
    else hipLaunchKernelGGL(fork_kernel, dim3(1), dim3(1024), 0, st, a);
    hipLaunchKernelGGL(fork_table_kernel, dim3(blocks_of(a.F, 4, 4096)), dim3(256), 0, st, a);
    return status();
}

LuxStatus launch_paged_release(const ReleaseArgs& a, hipStream_t st) {
    const int runs = a.pool > 0 ? (a.pool + kRun - 1) / kRun : 1;
    // A round of the one block's sixteen waves over requests, or over a run of pages,
    // takes about as long as another launch.
    if (a.pool <= kRun && a.R <= 16) {
        hipLaunchKernelGGL(release_kernel, dim3(1), dim3(1024), 0, st, a);
        return status();
    }
    if (!a.ws || (size_t)runs + kDropBlocks > a.ws_words) return LuxStatus::NotSupported;
    const unsigned drops = blocks_of(a.R, 4, kDropBlocks);
    hipLaunchKernelGGL(release_drop_kernel, dim3(drops), dim3(256), 0, st, a);
    hipLaunchKernelGGL(release_count_kernel, dim3(runs), dim3(1024), 0, st, a);
    hipLaunchKernelGGL(release_list_kernel, dim3(runs), dim3(1024), 0, st, a, (int)drops, runs);
    return status();
}

LuxStatus launch_paged_compact(const CompactArgs& a, hipStream_t st) {
    if (a.pool <= kFewPages && (int64_t)a.R * a.columns <= kFewEntries) {
        hipLaunchKernelGGL(compact_few_kernel, dim3(1), dim3(1024), 0, st, a);
        return status();
    }
    if (!a.ws || (size_t)a.pool + (size_t)(a.pool + 31) / 32 > a.ws_words) return LuxStatus::NotSupported;
    hipLaunchKernelGGL(compact_clear_kernel, dim3(blocks_of(a.pool, 256, 1024)), dim3(256), 0, st, a);
    hipLaunchKernelGGL(compact_mark_kernel, dim3(blocks_of(a.R, 4, 4096)), dim3(256), 0, st, a);
    hipLaunchKernelGGL(compact_moves_kernel, dim3(1), dim3(1024), 0, st, a);
    hipLaunchKernelGGL(compact_table_kernel, dim3(blocks_of(a.R, 4, 4096)), dim3(256), 0, st, a);
    return status();
}

LuxStatus launch_paged_copy(const CopyArgs& a, hipStream_t st) {
    const int64_t pieces = (a.page_bytes + kPiece - 1) / kPiece, blocks = pieces * 2 * a.layers * a.n;
    if (blocks >= (1ll << 31)) return LuxStatus::NotSupported;
    const bool wide = (((uintptr_t)a.kc | (uintptr_t)a.vc | (uint64_t)a.page_bytes | (uint64_t)a.layer_bytes) & 15) == 0;
    launch_blocks(blocks, 256, [&](int first, unsigned n) {
        if (wide) hipLaunchKernelGGL(copy_kernel<u4>, dim3(n), dim3(256), 0, st, a, first, (int)pieces);
        else if (a.esz == 4) hipLaunchKernelGGL(copy_kernel<uint32_t>, dim3(n), dim3(256), 0, st, a, first, (int)pieces);
        else hipLaunchKernelGGL(copy_kernel<uint16_t>, dim3(n), dim3(256), 0, st, a, first, (int)pieces);
    });
    return status();
}

}  // namespace lxq
