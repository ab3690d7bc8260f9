// token_logprobs.hip -- log probabilities of given tokens, entropy and the top
// alternatives of rows of logits, in one pass over them.
//
// With y = (x - r) c, c = scale log2 e and r near the row's maximum M:
//   S = sum exp2(y), E = sum exp2(y) y, moved from r to M at the end
//   lse = scale M + ln 2 (log2 S + d E / S),  H = ln 2 (log2 S - E / S)
// where c is d of itself below scale log2 e, by its rounding: a mean of y times d.
// A thread keeps its own r, S and E and its largest logit.  Of 64 groups of threads
// the k-th largest maximum is at most the row's k-th largest logit, so that the top
// k lie in the few threads with a maximum from there on (24 logits on average for k
// = 20): these are read again, out of the cache, and ranked by counting.
//
// Few rows are cut into parts, a block each; the last block of a row joins them.
// 4096 rows of 131072 bf16 logits: 194 us, 5.5 TB/s of the one read (a large copy
// moves 4.7); 8 rows of f32: 11.4 us, of which the read is 1.3, the launch 2.5, and the rest
// reductions over the block and trips to the counter and to the other parts' results.
//
// Rows in which that goes wrong (more logits from the bound on than are ranked, as
// where most are -infinity, or NaN) are finished by a search, one largest logit
// after the other, a reading of the row each: those 4096 rows with 10 finite logits take
// 11.1 ms for the 20 largest (0.22 with 1 % finite), 33.5 for 64 (0.43); the 8 rows 51
// us and 955.
#include "prompt.h"
#include "serving_device.h"

namespace lxq {
namespace {

typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4h __attribute__((ext_vector_type(4), aligned(2)));

constexpr int NT = 512, NW = NT / 64;
constexpr int kGroups = 64;     // groups of threads
constexpr int kRoom = 1024;     // logits that are ranked
constexpr int kMostParts = 64;
// r c up to which (x - r) c is taken as x c - r c: the rounding of r c is at most 4
constexpr float kFar = 0x1p27f;
constexpr float kBehind = 8.f;  // by which a thread's maximum passes its r c
constexpr float kNear = 4096.f;  // 2^-kNear is 0, and that of a few less: products by c are off by up to 8 there
constexpr float kLn2 = 0.69314718055994531f;

// order of logits: NaN above all, -0 as 0; 0 stands for no logit
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);
    return x != x ? ~0u : b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) {
    return k == ~0u ? __uint_as_float(0x7fc00000u) : __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
// the larger logit first, then the lower place
__device__ __forceinline__ uint64_t entry_of(uint32_t key, int at) { return (uint64_t)key << 32 | (uint32_t)~at; }
__device__ __forceinline__ int place_of(uint64_t e) { return (int)~(uint32_t)e; }

// sums of a part of a row, about its largest logit `top` (-infinity: none)
struct Sums {
    float top, s, e;  // NaN where there is one; s and e mean nothing where it is not finite
};

// s and e about r (in units of c) to those about another one
__device__ __forceinline__ void move(float& s, float& e, float by) {  // by = (r - new r) c
    by = fmaxf(by, -1e4f);  // where 2^by is 0, its product with e is, too
    const float f = __builtin_amdgcn_exp2f(by);
    e = f * fmaf(s, by, e);
    s *= f;
}

struct Params {
    LogprobArgs a;
    int parts, len;  // of a row, logits of a part (a multiple of 8)
    float c, d;
    Sums* sums;      // [rows, parts]
    uint64_t* tops;  // [rows, parts, top]
};

template <int T>
__device__ __forceinline__ float logit(const void* row, int i) {
    if constexpr (T == DT_F32) return static_cast<const float*>(row)[i];
    const uint32_t h = static_cast<const uint16_t*>(row)[i];
    return T == DT_F16 ? f16_to_f32(h) : bf16_to_f32(h);
}
template <int T>
__device__ __forceinline__ void unpack(const u4& v, float* x) {
    if constexpr (T == DT_F32) {
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] = __uint_as_float(v[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            x[2 * j] = T == DT_F16 ? f16_to_f32(v[j] & 0xffffu) : __uint_as_float(v[j] << 16);
            x[2 * j + 1] = T == DT_F16 ? f16_to_f32(v[j] >> 16) : __uint_as_float(v[j] & 0xffff0000u);
        }
    }
}

__device__ __forceinline__ uint64_t wave_most(uint64_t v) {
#pragma unroll
    for (int k = 1; k < 64; k *= 2) {
        const uint64_t o = __shfl_xor(v, k);
        v = v > o ? v : o;
    }
    return v;
}

struct Shared {
    uint64_t list[kRoom];
    uint64_t most[NW];
    uint64_t lows[kMostParts];
    uint64_t bound;
    uint32_t groups[kGroups];
    float part[NW][3];
    int count, odd, threads, last;
    uint16_t who[NT];
};

// The block: at(i, rank) for each of the n entries of v (in LDS), rank: how many
// come before it, the larger first, then the lower place.  Eight threads share an
// entry's comparisons, which would be a chain of reads for one.
template <class V, class F>
__device__ __forceinline__ void ranks(const V* v, int n, F at) {
    const int part = threadIdx.x & 7;
    for (int i0 = 0; i0 < n; i0 += NT / 8) {
        const int i = i0 + (int)(threadIdx.x >> 3);
        const V mine = v[i < n ? i : 0];
        int rank = 0;
#pragma unroll 8
        for (int j = part; j < n; j += 8) {
            const V o = v[j];
            rank += o > mine || (o == mine && j < i);
        }
#pragma unroll
        for (int k = 1; k < 8; k *= 2) rank += __shfl_xor(rank, k);
        if (part == 0 && i < n) at(i, rank);
    }
}

// lse - scale M
__device__ __forceinline__ float log_of(const Params& p, const Sums& t) {
    if (t.top == -INFINITY || t.top == INFINITY) return 0.f;
    return fmaf(p.d, t.e / t.s, log2f(t.s)) * kLn2;
}
// the row's scores, from its sums and its top entries
__device__ __forceinline__ void write_sums(const Params& p, int r, const Sums& t, float x_tok, bool has_tok, float log_sum) {
    const LogprobArgs& a = p.a;
    // NaN in the row, +infinity, nothing but -infinity, or as it should be
    const bool nan = t.top != t.top, none = t.top == -INFINITY, high = t.top == INFINITY;
    if (nan) log_sum = t.top;
    const float lse = fmaf(a.scale, t.top, log_sum);
    if (a.lse) a.lse[r] = lse;
    if (a.entropy) a.entropy[r] = none ? 0.f : high || nan ? __uint_as_float(0x7fc00000u) : fmaf(-kLn2, t.e / t.s, log_sum);
    if (a.logprobs) a.logprobs[r] = !has_tok || none ? -INFINITY : high || nan ? fmaf(a.scale, x_tok, -lse) : (x_tok - t.top) * a.scale - log_sum;
}
__device__ __forceinline__ float top_logprob(const LogprobArgs& a, const Sums& t, float x, float log_sum) {
    if (t.top == -INFINITY) return -INFINITY;
    if (t.top != t.top || t.top == INFINITY) return a.scale * x - a.scale * t.top;
    return (x - t.top) * a.scale - log_sum;
}

// what other blocks read: written through, read from beyond the block's own caches
template <class V>
__device__ __forceinline__ void put_out(V* p, V v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
template <class V>
__device__ __forceinline__ V look(const V* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// a block, behind the last part: the row's scores from its parts' sums and entries
__device__ __forceinline__ void join_parts(const Params& p, int r, float x_tok, bool has, Shared& sh) {
    uint64_t* list = sh.list;
    int& count = sh.count;
    const LogprobArgs& a = p.a;
    const int tid = threadIdx.x, lane = tid & 63;
    const uint64_t* tops = p.tops + (int64_t)r * p.parts * a.top;
    if (tid == 0) count = 0;
    const int entries = p.parts * a.top;
    const uint64_t first_entry = tid < entries ? look(tops + tid) : 0, second_entry = tid + NT < entries ? look(tops + tid + NT) : 0;
    // a bound: the m-th largest of the parts' d-th entries, where m d is top or more
    const int d = (a.top + p.parts - 1) / p.parts, m = d ? (a.top + d - 1) / d : 0;
    const uint64_t low_mine = a.top > 0 && tid < p.parts ? look(tops + tid * a.top + d - 1) : 0;
    // each wave for itself
    const Sums* its = p.sums + (int64_t)r * p.parts + lane;
    const Sums mine = lane < p.parts ? Sums{look(&its->top), look(&its->s), look(&its->e)} : Sums{-INFINITY, 0.f, 0.f};
    uint32_t k = lane < p.parts ? key_of(mine.top) : 0u;
    uint32_t most = k;
#pragma unroll
    for (int i = 1; i < 64; i *= 2) {
        const uint32_t o = (uint32_t)__shfl_xor((int)most, i);
        most = most > o ? most : o;
    }
    Sums t = {value_of(most), 0.f, 0.f};
    float s = mine.s, e = mine.e;
    if (!(fabsf(mine.top) < INFINITY) || !(fabsf(t.top) < INFINITY)) s = e = 0.f;
    else move(s, e, (mine.top - t.top) * p.c);
    t.s = wave_sum(s);
    t.e = wave_sum(e);
    const float log_sum = log_of(p, t);
    if (tid == 0) write_sums(p, r, t, x_tok, has, log_sum);
    if (a.top == 0) return;
    if (tid < p.parts) sh.lows[tid] = low_mine;
    __syncthreads();
    ranks(sh.lows, p.parts, [&](int i, int rank) {
        if (rank == m - 1) sh.bound = sh.lows[i];
    });
    __syncthreads();
    const uint64_t low = sh.bound;
    for (int i = tid; i < entries; i += NT) {
        const uint64_t x = i == tid ? first_entry : i == tid + NT ? second_entry : look(tops + i);
        if (x >= low && x != 0) {
            const int at = atomicAdd(&count, 1);
            if (at < kRoom) list[at] = x;
        }
    }
    __syncthreads();
    const int found = count;
    auto write = [&](int rank, uint64_t x) {
        if (rank >= a.top) return;
        if (a.top_ids) a.top_ids[(int64_t)r * a.top + rank] = place_of(x);
        if (a.top_lp) a.top_lp[(int64_t)r * a.top + rank] = top_logprob(a, t, value_of((uint32_t)(x >> 32)), log_sum);
    };
    if (found <= kRoom) {
        ranks(list, found, [&](int i, int rank) { write(rank, list[i]); });
        return;
    }
    for (int i = tid; i < entries; i += NT) {
        const uint64_t x = look(tops + i);
        int rank = 0;
        for (int j = 0; j < entries; j++) rank += look(tops + j) > x;
        if (x != 0) write(rank, x);
    }
}

// one block: part blockIdx of row; SPLIT: its results go to the workspace, and the
// last block of the row joins them
template <int T, bool SPLIT>
__global__ __launch_bounds__(NT) void logprobs_kernel(Params p, int first) {
    constexpr int E = T == DT_F32 ? 4 : 8;
    __shared__ Shared sh;
    const LogprobArgs& a = p.a;
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int block = first + (int)blockIdx.x, r = SPLIT ? block / p.parts : block, part = SPLIT ? block - r * p.parts : 0;
    const int from = part * p.len, to = SPLIT && from + p.len < a.V ? from + p.len : a.V, n = to > from ? to - from : 0;
    const char* base = static_cast<const char*>(a.logits) + ((int64_t)r * a.row + from) * (T == DT_F32 ? 4 : 2);
    const int vectors = n >= NT * E ? n / E : 0;  // fewer logits: one by one, so that all threads have some
    const int token = a.tokens && a.logprobs ? a.tokens[r] : -1;
    const bool has = (uint32_t)token < (uint32_t)a.V;
    const float x_tok = has ? logit<T>(static_cast<const char*>(a.logits) + (int64_t)r * a.row * (T == DT_F32 ? 4 : 2), token) : 0.f;
    if (tid == 0) sh.count = sh.odd = sh.threads = 0;

    // the thread's vectors tid, tid + NT, ..., and logits behind the vectors likewise
    float top = -INFINITY, ref = 0.f, s = 0.f, e = 0.f;  // ref: r c, as the loop subtracts it
    bool fresh = true;
    auto take = [&](const float* x, int m) {
        float mx = x[0];
#pragma unroll
        for (int j = 1; j < m; j++) mx = fmaxf(mx, x[j]);
        top = fmaxf(top, mx);
        // A new r only where the maximum passes it by kBehind: what E / S leaves of the
        // entropy when both are moved to the maximum is off by the roundings of that
        // distance (with 60 bf16 rows were off by 2.4e-7 of it, with 8 by 6e-8, as with 2)
        if (__any(fresh || fmaf(mx, p.c, -ref) > kBehind)) {
            const float to = mx * p.c;
            if ((fresh || to - ref > kBehind) && fabsf(to) < kFar) {
                if (!fresh) move(s, e, ref - to);
                ref = to;
                fresh = false;
            }
        }
        float vs = 0.f, ve = 0.f;  // the vector's sums by themselves: fewer roundings at the size of all
#pragma unroll
        for (int j = 0; j < m; j++) {
            const float y = fmaf(x[j], p.c, -ref), q = __builtin_amdgcn_exp2f(y);
            vs += q;
            ve = fmaf(q, fmaxf(y, -1000.f), ve);  // not 0 times -infinity
        }
        s += vs;
        e += ve;
    };
    constexpr int kU = 4;
    int v = tid;
    for (; v + (kU - 1) * NT < vectors; v += kU * NT) {
        u4 d[kU];
#pragma unroll
        for (int k = 0; k < kU; k++) d[k] = *reinterpret_cast<const u4h*>(base + (int64_t)(v + k * NT) * 16);
#pragma unroll
        for (int k = 0; k < kU; k++) {
            float x[E];
            unpack<T>(d[k], x);
            take(x, E);
        }
    }
    u4 rest[kU - 1];
#pragma unroll
    for (int k = 0; k < kU - 1; k++)
        if (v + k * NT < vectors) rest[k] = *reinterpret_cast<const u4h*>(base + (int64_t)(v + k * NT) * 16);
#pragma unroll
    for (int k = 0; k < kU - 1; k++) {
        if (v + k * NT >= vectors) break;
        float x[E];
        unpack<T>(rest[k], x);
        take(x, E);
    }
    const int behind = vectors * E;
    for (int i = behind + tid; i < n; i += NT) {
        float x[1] = {logit<T>(base, i)};
        take(x, 1);
    }

    // the block's sums, about its largest logit
    const bool odd = !(s < INFINITY);
    float wtop = top;
#pragma unroll
    for (int k = 1; k < 64; k *= 2) wtop = fmaxf(wtop, __shfl_xor(wtop, k));
    // groups of 8 threads
    float gtop = top;
#pragma unroll
    for (int k = 1; k < 8; k *= 2) gtop = fmaxf(gtop, __shfl_xor(gtop, k));
    const bool any = tid < vectors || behind + tid < n;
    uint32_t gkey = any ? key_of(gtop) : 0u;
#pragma unroll
    for (int k = 1; k < 8; k *= 2) {
        const uint32_t o = (uint32_t)__shfl_xor((int)gkey, k);
        gkey = gkey > o ? gkey : o;
    }
    if ((lane & 7) == 0) sh.groups[tid >> 3] = gkey;
    if (lane == 0) sh.part[w][0] = wtop;
    __syncthreads();
    if (odd) sh.odd = 1;
    float all = sh.part[0][0];
#pragma unroll
    for (int i = 1; i < NW; i++) all = fmaxf(all, sh.part[i][0]);
    if (fresh || all == -INFINITY) s = e = 0.f;
    else move(s, e, fmaf(-all, p.c, ref));
    s = wave_sum(s);
    e = wave_sum(e);
    if (lane == 0) {
        sh.part[w][1] = s;
        sh.part[w][2] = e;
    }
    // the bound: the k-th largest of the groups' maxima
    if (a.top > 0)
        ranks(sh.groups, kGroups, [&](int i, int rank) {
            if (rank == a.top - 1) sh.bound = sh.groups[i];
        });
    __syncthreads();
    const uint32_t bound = (uint32_t)sh.bound;
    Sums t = {all, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NW; i++) {
        t.s += sh.part[i][1];
        t.e += sh.part[i][2];
    }
    // NaN, infinite and far logits, and rows whose largest is far below 0, or so near
    // to there that logits a thread left out as far ones (fresh) count beside it: the
    // sums once more
    bool nan = false;
    if (sh.odd || (all > -INFINITY && all * p.c <= kNear - kFar)) {
        s = e = 0.f;
        for (int i = tid; i < n; i += NT) {
            const float x = logit<T>(base, i), y = fmaxf((x - all) * p.c, -1000.f), q = __builtin_amdgcn_exp2f(y);
            nan |= x != x;
            s += q;
            e = fmaf(q, y, e);
        }
        nan = __syncthreads_or(nan);
        s = wave_sum(s);
        e = wave_sum(e);
        if (lane == 0) {
            sh.part[w][1] = s;
            sh.part[w][2] = e;
        }
        __syncthreads();
        t.s = t.e = 0.f;
#pragma unroll
        for (int i = 0; i < NW; i++) {
            t.s += sh.part[i][1];
            t.e += sh.part[i][2];
        }
        if (nan) t.top = __uint_as_float(0x7fc00000u);
    }

    int found = 0;
    if (a.top > 0 && !nan) {
        auto list = [&](const u4& v, int i) {
            float x[E];
            unpack<T>(v, x);
            int some = 0;
#pragma unroll
            for (int j = 0; j < E; j++) some += key_of(x[j]) >= bound;
            if (some == 0) return;
            int at = atomicAdd(&sh.count, some);
#pragma unroll
            for (int j = 0; j < E; j++) {
                const uint32_t k = key_of(x[j]);
                if (k >= bound && at < kRoom) sh.list[at] = entry_of(k, from + i * E + j);
                at += k >= bound;
            }
        };
        const bool mine = any && key_of(top) >= bound;
        if (vectors <= (kU - 1) * NT) {  // they are still in registers
#pragma unroll
            for (int k = 0; k < kU - 1; k++)
                if (mine && tid + k * NT < vectors) list(rest[k], tid + k * NT);
        } else {
            // the threads that have logits from the bound on, then those logits: a
            // thread reads one vector of one of them
            if (mine) sh.who[atomicAdd(&sh.threads, 1)] = (uint16_t)tid;
            __syncthreads();
            const int each = (vectors + NT - 1) / NT, items = sh.threads * each;
            for (int x0 = tid; x0 < items; x0 += NT) {
                const int which = (int)((uint32_t)x0 / (uint32_t)each), i = sh.who[which] + (x0 - which * each) * NT;
                if (i < vectors) list(u4(*reinterpret_cast<const u4h*>(base + (int64_t)i * 16)), i);
            }
        }
        for (int i = behind + tid; i < n; i += NT) {
            const uint32_t k = key_of(logit<T>(base, i));
            if (k >= bound) {
                const int at = atomicAdd(&sh.count, 1);
                if (at < kRoom) sh.list[at] = entry_of(k, from + i);
            }
        }
        __syncthreads();
        found = sh.count;
    }
    const float log_sum = SPLIT ? 0.f : log_of(p, t);
    if (!SPLIT) {
        if (tid == 0) write_sums(p, r, t, x_tok, has, log_sum);
    } else if (tid == 0) {
        Sums* its = p.sums + (int64_t)r * p.parts + part;
        put_out(&its->top, t.top);
        put_out(&its->s, t.s);
        put_out(&its->e, t.e);
    }
    auto put = [&](int rank, uint64_t entry) {
        if (SPLIT) {
            put_out(p.tops + ((int64_t)r * p.parts + part) * a.top + rank, entry);
        } else {
            if (a.top_ids) a.top_ids[(int64_t)r * a.top + rank] = place_of(entry);
            if (a.top_lp) a.top_lp[(int64_t)r * a.top + rank] = top_logprob(a, t, value_of((uint32_t)(entry >> 32)), log_sum);
        }
    };
    if (a.top > 0 && !nan && found <= kRoom) {
        ranks(sh.list, found, [&](int i, int rank) {
            if (rank < a.top) put(rank, sh.list[i]);
        });
        // a part with fewer logits than that
        if (SPLIT && tid >= found && tid < a.top) put(tid, 0);
    } else if (a.top > 0) {
        // one after the other: the largest entry below the last one
        uint64_t last = ~0ull;
        for (int k = 0; k < a.top; k++) {
            uint64_t best = 0;
            for (int i = tid; i < n; i += NT) {
                const uint64_t x = entry_of(key_of(logit<T>(base, i)), from + i);
                if ((x < last || k == 0) && x > best) best = x;  // NaN in place 0 is all ones
            }
            best = wave_most(best);
            if (lane == 0) sh.most[w] = best;
            __syncthreads();
            last = sh.most[0];
#pragma unroll
            for (int i = 1; i < NW; i++) last = sh.most[i] > last ? sh.most[i] : last;
            if (tid == 0) put(k, last);
            __syncthreads();
        }
    }
    if constexpr (SPLIT) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the wave's part of the results is out
        __syncthreads();
        if (tid == 0) {
            // the last block of the row leaves the counter at 0
            uint32_t* c = p.a.count + r;
            sh.last = __hip_atomic_fetch_add(c, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)(p.parts - 1);
            if (sh.last) __hip_atomic_store(c, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (sh.last) join_parts(p, r, x_tok, has, sh);
    }
}

template <int T>
LuxStatus launch_t(const LogprobArgs& a, hipStream_t st) {
    Params p = {};
    p.a = a;
    const double c = (double)a.scale * 1.4426950408889634;
    p.c = c < 0x1.fffffep127 ? (float)c : 0x1.fffffep127f;  // finite: 0 times it is 0
    p.d = p.c > 0x1p-126f ? (float)(c / p.c - 1.) : 0.f;
    // two blocks per CU; parts of at least 4096 logits
    int parts = a.T > 0 ? 2 * a.cus / a.T : 1;
    if (parts > a.V / 4096) parts = a.V / 4096;
    if (parts > kMostParts) parts = kMostParts;
    const size_t one = sizeof(Sums) + (size_t)a.top * 8;
    if (parts > 1 && (!a.ws || (size_t)a.T * parts * one > a.ws_bytes || a.T > a.counts)) parts = 1;
    if (parts <= 1) {
        p.parts = 1;
        p.len = a.V;
        launch_blocks(a.T, NT, [&](int first, unsigned n) {
            hipLaunchKernelGGL((logprobs_kernel<T, false>), dim3(n), dim3(NT), 0, st, p, first);
        });
    } else {
        p.len = ((a.V + parts - 1) / parts + 7) & ~7;
        p.parts = (a.V + p.len - 1) / p.len;
        p.tops = reinterpret_cast<uint64_t*>(a.ws);
        p.sums = reinterpret_cast<Sums*>(a.ws + (size_t)a.T * p.parts * a.top * 8);
        hipLaunchKernelGGL((logprobs_kernel<T, true>), dim3(a.T * p.parts), dim3(NT), 0, st, p, 0);
    }
    return hipGetLastError() == hipSuccess ? LuxStatus::Ok : LuxStatus::Internal;
}

}  // namespace

LuxStatus launch_token_logprobs(const LogprobArgs& a, hipStream_t st) {
    if (a.dtype == DT_F32) return launch_t<DT_F32>(a, st);
    return a.dtype == DT_F16 ? launch_t<DT_F16>(a, st) : launch_t<DT_BF16>(a, st);
}

}  // namespace lxq
