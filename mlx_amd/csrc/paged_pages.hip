// paged_pages.hip -- pages in use: forks that share them, pages given back,
// compaction of a pool, and copies of their contents.
//
// All but the copies is whole numbers and latency.  What decides an order (which
// fork takes which page, where a page goes back to in the list) is a sum over
// forks or pages in their own order, never the order in which threads arrive: equal
// calls give equal results.
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

// --- fork -----------------------------------------------------------------------------

// the table's entries of fork f: ws[f] full pages from src's row, then ws[F + f]
// where it is not kNoEntry
constexpr int kNoEntry = -0x7fffffff - 1;
__device__ __forceinline__ void fork_columns(const ForkArgs& a, int f, int first, int step) {
    const int full = a.ws[f];
    if (full < 0) return;
    const int32_t* from = a.table + (int64_t)a.src[f] * a.columns;
    int32_t* to = a.table + (int64_t)a.dst[f] * a.columns;
    for (int c = first; c < full; c += step) {
        const int id = from[c];
        to[c] = id;
        if ((uint32_t)id < (uint32_t)a.pool) add_now(a.shares + id, 1);
    }
    if (first == 0 && a.ws[a.F + f] != kNoEntry) to[full] = a.ws[a.F + f];
}

// One block: which forks are made, and the pages they take.  A fork is made if it is
// the first one of its dst: each writes its number, below 0, as dst's length, and
// the lowest stays.  ALL: the table too, in the same launch.
template <bool ALL>
__global__ __launch_bounds__(1024) void fork_kernel(ForkArgs a) {
    __shared__ int part[16];
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
    int taken = 0, shared = 0, out = 0;
    int needed = 0;
    for (int f0 = 0; f0 < a.F; f0 += 1024) {
        const int f = f0 + tid;
        const int n = f < a.F ? a.ws[f] : -1;
        const int d = n >= 0 ? a.dst[f] : 0;
        const bool made = n >= 0 && load_now(a.lens + d) == f - a.F;
        const int full = made ? div_by(n, a.div) : 0;
        int last = -1;
        const bool rest = made && n > full * a.page;
        if (rest) last = a.table[(int64_t)a.src[f] * a.columns + full];
        const bool take = rest && (uint32_t)last < (uint32_t)a.pool;
        int all;
        const int at = head + needed + block_sum<16>(take ? 1 : 0, all, part);
        needed += all;
        if (f < a.F) {
            const bool there = take && at < a.free_count;
            const int page = there ? a.free_pages[at] : -1;
            a.copy_src[f] = there ? last : -1;
            a.copy_dst[f] = page;
            a.ws[f] = made ? full : -1;
            a.ws[a.F + f] = rest ? (take ? page : last) : kNoEntry;
            if (made) store_now(a.lens + d, take && !there ? full * a.page : n);
            taken += there;
            shared += full;
            out += !made;
        }
    }
    int all_taken, all_shared, all_out;
    block_sum<16>(taken, all_taken, part);
    block_sum<16>(shared, all_shared, part);
    block_sum<16>(out, all_out, part);
    if (tid == 0) {
        a.counts[0] = head + all_taken;
        a.counts[1] = all_shared;
        a.counts[2] = needed - all_taken;
        a.counts[3] = all_out;
    }
    if constexpr (ALL) {
        __syncthreads();
        for (int f = tid >> 6; f < a.F; f += 16) fork_columns(a, f, tid & 63, 64);
    }
}

// a wave per fork
__global__ __launch_bounds__(256) void fork_table_kernel(ForkArgs a) {
    for (int64_t f = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); f < a.F; f += (int64_t)gridDim.x * 4)
        fork_columns(a, (int)f, threadIdx.x & 63, 64);
}

// --- release --------------------------------------------------------------------------

constexpr int kDropBlocks = 512, kRun = 4096;  // blocks that drop entries; pages of a run

// request r's pages behind what it keeps lose a holder; a page that had one alone
// counts -1 until the list has it.  `back`: pages that go back; returns the entries
__device__ __forceinline__ int drop(const ReleaseArgs& a, int r, int first, int step, int& back) {
    const int n = cut(a.lens[r], a.columns * a.page), k = a.keep[r];
    const int kept = k < 0 ? 0 : k < n ? k : n;
    const int c1 = pages_of(n, a.div);
    int entries = 0;
    for (int c = pages_of(kept, a.div) + first; c < c1; c += step) {
        const int id = a.table[(int64_t)r * a.columns + c];
        if ((uint32_t)id >= (uint32_t)a.pool) continue;
        entries++;
        back += add_now(a.shares + id, -1) == 0;
    }
    return entries;
}
__device__ __forceinline__ void write_kept(const ReleaseArgs& a, int r) {
    const int n = cut(a.lens[r], a.columns * a.page), k = a.keep[r];
    a.kv[r] = k < 0 ? 0 : k < n ? k : n;
}

// the pages from p0 on, four to a thread: those that go back take the list's entries
// from `at` on (below 0: lost)
template <int NT>
__device__ __forceinline__ int give_back(const ReleaseArgs& a, int p0, int at, int* part) {
    const int p = p0 + 4 * (int)threadIdx.x;
    int v[4], mine = 0, all;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        v[i] = p + i < a.pool ? load_now(a.shares + p + i) : 0;
        mine += v[i] < 0;
    }
    int to = at + block_sum<NT / 64>(mine, all, part);
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (v[i] < 0) {
            if (to >= 0) a.free_pages[to] = p + i;
            to++;
            a.shares[p + i] = 0;
        }
    return all;
}
__device__ __forceinline__ void release_counts(const ReleaseArgs& a, int head, int back, int entries) {
    a.counts[0] = head > back ? head - back : 0;
    a.counts[1] = back;
    a.counts[2] = entries - back;
    a.counts[3] = back > head ? back - head : 0;
}

// one block for small pools
__global__ __launch_bounds__(1024) void release_kernel(ReleaseArgs a) {
    __shared__ int part[16];
    const int tid = threadIdx.x, head = cut(a.head[0], a.free_count);
    int back = 0, entries = 0, all_back, all_entries;
    for (int r = tid >> 6; r < a.R; r += 16) entries += drop(a, r, tid & 63, 64, back);
    block_sum<16>(back, all_back, part);
    block_sum<16>(entries, all_entries, part);
    for (int r = tid; r < a.R; r += 1024) write_kept(a, r);  // kv may be lens: all have read them
    int at = head - all_back;
    for (int p0 = 0; p0 < a.pool; p0 += kRun) at += give_back<1024>(a, p0, at, part);
    if (tid == 0) release_counts(a, head, all_back, all_entries);
}

// three launches: entries per block into ws, pages that go back per run into ws
// behind them, the list
__global__ __launch_bounds__(256) void release_drop_kernel(ReleaseArgs a) {
    __shared__ int part[4];
    int back = 0, entries = 0, all;
    for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < a.R; r += kDropBlocks * 4) {
        entries += drop(a, (int)r, threadIdx.x & 63, 64, back);
        if ((threadIdx.x & 63) == 0) write_kept(a, (int)r);
    }
    block_sum<4>(entries, all, part);
    if (threadIdx.x == 0) a.ws[blockIdx.x] = all;
}
__global__ __launch_bounds__(1024) void release_count_kernel(ReleaseArgs a) {
    __shared__ int part[16];
    const int p = blockIdx.x * kRun + 4 * (int)threadIdx.x;
    int mine = 0, all;
#pragma unroll
    for (int i = 0; i < 4; i++) mine += p + i < a.pool && a.shares[p + i] < 0;
    block_sum<16>(mine, all, part);
    if (threadIdx.x == 0) a.ws[kDropBlocks + blockIdx.x] = all;
}
__global__ __launch_bounds__(1024) void release_list_kernel(ReleaseArgs a, int runs) {
    __shared__ int part[16];
    const int tid = threadIdx.x, head = cut(a.head[0], a.free_count);
    int mine = 0, before = 0, back, first;
    for (int i = tid; i < runs; i += 1024) {
        const int n = a.ws[kDropBlocks + i];
        mine += n;
        before += i < (int)blockIdx.x ? n : 0;
    }
    block_sum<16>(mine, back, part);
    block_sum<16>(before, first, part);
    give_back<1024>(a, blockIdx.x * kRun, head - back + first, part);
    if (blockIdx.x == 0) {
        int entries;
        block_sum<16>(tid < kDropBlocks ? a.ws[tid] : 0, entries, part);
        if (tid == 0) release_counts(a, head, back, entries);
    }
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

// --- copy -----------------------------------------------------------------------------

constexpr int kPiece = 16384;  // bytes of a block

// pieces of `pieces` per page of a matrix; matrices: keys and values of each layer
template <class V>
__global__ __launch_bounds__(256) void copy_kernel(CopyArgs a, int first, int pieces) {
    const uint32_t b = (uint32_t)first + blockIdx.x, pair = b / (uint32_t)pieces, piece = b - pair * (uint32_t)pieces;
    const uint32_t i = pair / (uint32_t)(2 * a.layers), m = pair - i * (uint32_t)(2 * a.layers);
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
    if ((int64_t)a.F * a.columns <= 16384) {
        hipLaunchKernelGGL(fork_kernel<true>, dim3(1), dim3(1024), 0, st, a);
    } else {
        hipLaunchKernelGGL(fork_kernel<false>, dim3(1), dim3(1024), 0, st, a);
        hipLaunchKernelGGL(fork_table_kernel, dim3(blocks_of(a.F, 4, 4096)), dim3(256), 0, st, a);
    }
    return status();
}

LuxStatus launch_paged_release(const ReleaseArgs& a, hipStream_t st) {
    const int runs = (a.pool + kRun - 1) / kRun;
    if (a.pool <= 8 * kRun && (int64_t)a.R * a.columns <= 65536) {
        hipLaunchKernelGGL(release_kernel, dim3(1), dim3(1024), 0, st, a);
        return status();
    }
    if (!a.ws || (size_t)runs + kDropBlocks > a.ws_words) return LuxStatus::NotSupported;
    hipLaunchKernelGGL(release_drop_kernel, dim3(kDropBlocks), dim3(256), 0, st, a);
    hipLaunchKernelGGL(release_count_kernel, dim3(runs < 1 ? 1 : runs), dim3(1024), 0, st, a);
    hipLaunchKernelGGL(release_list_kernel, dim3(runs < 1 ? 1 : runs), dim3(1024), 0, st, a, runs);
    return status();
}

LuxStatus launch_paged_compact(const CompactArgs& a, hipStream_t st) {
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
