// paged_attn.h -- attention of one new token per request over a paged cache.
//
// For each request and head of keys, the queries of its group (up to 16: the
// columns of a matrix tile; larger groups take several) meet every cached
// token once.  A wave takes tiles of kTile tokens:
//   S^T[token, query] = K . Q^T      A = K rows, straight from the cache
//   P^T = exp2(S^T - m)              running maximum m and sum l per query
//   O^T[channel, query] += V^T . P^T
// A 16x16 result has its column (the query) in the lane and its rows (tokens
// 4g .. 4g + 3 for lane group g = lane / 16) in the lane's registers, which is
// the B operand of the second product with those tokens as its k: P never
// leaves its lane, m and l are the lane's own, and no LDS is touched.  k may be
// numbered in any order as long as A agrees: V's rows are loaded 16 bytes per
// lane and token and their 16-bit halves paired by token with one byte permute
// per pair.
//
// A block's NW waves share a stretch of one request's tokens, tile by tile in
// turn; at its end they meet in LDS.  Where pairs of request and head are too
// few or too uneven for the card, the tokens of all pairs are laid end to end
// in units of NW tiles and cut into P equal ranges, one per block: a pair that
// a cut goes through leaves partial (m, l, O) in the workspace, which a second
// launch joins.  Bound by HBM.
#pragma once
#include "qcommon.h"
#include "serving.h"

namespace lxq {
namespace attn {

typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4h __attribute__((ext_vector_type(4), aligned(2)));  // rows of q start anywhere
typedef float f4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr float kLowest = -3.0e38f;  // the maximum of no score
constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.69314718055994531f;

struct Params {
    AttnArgs a;
    int HQ;            // heads of keys times query tiles of a group
    int QT, rows;      // query tiles of a group; rows of a tile kept in partial results
    int P;             // ranges; 0: one block per pair
    float* part_o;     // [2 P, rows, D]
    float* part_ml;    // [2 P, rows, 2]
    int64_t* meta;     // [P, 4]
};

// what a boundary between two ranges needs to know to join the pair it cuts
struct Cut {
    int r, hq;  // r < 0: nothing to join here
    int u0, n;  // units of the pair before the cut, and in all
    int64_t units;
    int64_t pad;
};

// of `units` units, range w of P starts at first(w): the first units % P
// ranges are one unit longer
struct Ranges {
    int64_t base, rem;
    __device__ Ranges(int64_t units, int P) : base(units / P), rem(units - units / P * P) {}
    __device__ int64_t first(int w) const { return w * base + (w < rem ? w : rem); }
    __device__ int of(int64_t u) const {
        const int64_t long_ones = rem * (base + 1);
        return (int)(u < long_ones ? u / (base + 1) : rem + (u - long_ones) / base);
    }
};

__device__ __forceinline__ int div_by(int t, const DivBy& d) { return (int)(((uint64_t)(uint32_t)t * d.mul) >> (31 + d.sh)); }

// the tokens of request r that count: [start, end), and where tiles begin
struct Extent {
    int start, end, base;
};
__device__ __forceinline__ Extent extent_of(const AttnArgs& a, int r) {
    const int cap = a.pool > 0 ? a.columns * a.page : 0;
    int n = a.lens[r];
    n = n < 0 ? 0 : n > cap ? cap : n;
    const int s = a.window > 0 && n > a.window ? n - a.window : 0;
    return Extent{s, n, s & ~31};
}
// units of `tokens` tokens; a request with none has one, which writes its zeros
__device__ __forceinline__ int units_of(const Extent& e, int tokens) {
    const int n = (int)(((int64_t)e.end - e.base + tokens - 1) / tokens);
    return n < 1 ? 1 : n;
}

template <int T>
__device__ __forceinline__ f4 mfma_qk(const u4& k, const u4& q, f4 c) {
    if constexpr (T == DT_F16) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, k), __builtin_bit_cast(f16x8, q), c, 0, 0, 0);
    } else if constexpr (T == DT_BF16) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, k), __builtin_bit_cast(bf16x8, q), c, 0, 0, 0);
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++)
            c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k[j]), __uint_as_float(q[j]), c, 0, 0, 0);
        return c;
    }
}

// max / sum over the four lanes that hold one query's tokens
__device__ __forceinline__ float group_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float group_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// T: type of q, cache and out; DP: head_dim rounded up to 64, 128 or 256;
// FULL: head_dim is DP
template <int T, int DP, bool FULL, int NW>
struct Attn {
    static constexpr int ES = T == DT_F32 ? 4 : 2, E = 16 / ES;  // bytes; elements per 16 bytes
    static constexpr int SUB = T == DT_F32 ? 1 : 2, kTile = 16 * SUB;
    static constexpr int NC = DP / (4 * E);                  // 16-byte chunks of a key row per lane
    static constexpr int VE = E < DP / 16 ? E : DP / 16;     // channels of a value row per lane and load
    static constexpr int NV = DP / (16 * VE);                // loads per value row
    static constexpr int VW = VE * ES / 4;                   // their words
    static constexpr int kUnit = kTile * NW;
    static constexpr int LS = DP + 4;                        // LDS row of a query, in floats
    typedef uint32_t uv __attribute__((ext_vector_type(VW)));

    static constexpr size_t lds_bytes(int rows) { return (size_t)NW * (rows * LS + 32) * 4; }

    u4 q[NC], k[SUB][NC];
    uv v[4 * SUB][NV];
    f4 o[NV][VE];
    float m, l;

    // lane's token of a tile: its row of the cache, or -1
    __device__ __forceinline__ static int page_at(const AttnArgs& a, const Extent& e, int r, int t) {
        return t >= e.start && t < e.end ? a.table[(int64_t)r * a.columns + div_by(t, a.div)] : -1;
    }
    __device__ __forceinline__ static int row_at(const AttnArgs& a, int h, int t, int page) {
        const int at = t - div_by(t, a.div) * a.page;
        return (uint32_t)page < (uint32_t)a.pool ? (page * a.Hk + h) * a.page + at : -1;
    }

    __device__ __forceinline__ void load_q(const AttnArgs& a, int r, int h, int qt) {
        const int lane = threadIdx.x & 63, i = qt * 16 + (lane & 15);
#pragma unroll
        for (int c = 0; c < NC; c++) {
            const int d = (4 * c + (lane >> 4)) * E;
            q[c] = u4{0, 0, 0, 0};
            if (i < a.G && (FULL || d < a.D)) {
                const char* p = static_cast<const char*>(a.q) + (r * a.q_row + (int64_t)(h * a.G + i) * a.D + d) * ES;
                q[c] = *reinterpret_cast<const u4h*>(p);
            }
        }
    }
    // rows of masked tokens read row 0; channels past head_dim stay zero
    __device__ __forceinline__ void load_k(const AttnArgs& a, int row) {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int s = 0; s < SUB; s++) {
            const int rw = __shfl(row, 16 * s + (lane & 15));
            const char* p = static_cast<const char*>(a.kc) + (uint64_t)(uint32_t)(rw < 0 ? 0 : rw) * (uint32_t)(a.D * ES) + (lane >> 4) * 16;
#pragma unroll
            for (int c = 0; c < NC; c++)
                if (FULL || (4 * c + (lane >> 4)) * E < a.D) k[s][c] = *reinterpret_cast<const u4*>(p + c * 64);
        }
    }
    __device__ __forceinline__ void load_v(const AttnArgs& a, int row) {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int t = 0; t < 4 * SUB; t++) {
            const int rw = __shfl(row, 16 * (t / 4) + 4 * (lane >> 4) + t % 4);
            const char* p = static_cast<const char*>(a.vc) + (uint64_t)(uint32_t)(rw < 0 ? 0 : rw) * (uint32_t)(a.D * ES);
#pragma unroll
            for (int c = 0; c < NV; c++) {
                const int d = (16 * c + (lane & 15)) * VE;  // past head_dim: channels that are not stored
                v[t][c] = *reinterpret_cast<const uv*>(p + (FULL || d < a.D ? d * ES : 0));
            }
        }
    }

    __device__ __forceinline__ void scores(f4* s) const {
#pragma unroll
        for (int i = 0; i < SUB; i++) s[i] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int i = 0; i < SUB; i++) s[i] = mfma_qk<T>(k[i][c], q[c], s[i]);
    }

    // s (scores) to exp2 of their distance to the running maximum; bits: the
    // tile's tokens that count
    __device__ __forceinline__ void soften(const AttnArgs& a, f4* s, uint64_t bits) {
        const int g = (threadIdx.x & 63) >> 4;
        const float scale = a.scale * kLog2e;
        float mx = kLowest;
#pragma unroll
        for (int i = 0; i < SUB; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                float x = s[i][j];
                if (a.softcap > 0.f) x = a.softcap * kLog2e * tanhf(x * a.scale / a.softcap);
                else x *= scale;
                x = (bits >> (16 * i + 4 * g + j)) & 1 ? x : -INFINITY;
                s[i][j] = x;
                mx = fmaxf(mx, x);
            }
        mx = fmaxf(group_max(mx), m);
        if (__any(mx > m)) {
            const float f = __builtin_amdgcn_exp2f(m - mx);
            m = mx;
            l *= f;
#pragma unroll
            for (int c = 0; c < NV; c++)
#pragma unroll
                for (int e = 0; e < VE; e++) o[c][e] *= f;
        }
#pragma unroll
        for (int i = 0; i < SUB; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                s[i][j] = __builtin_amdgcn_exp2f(s[i][j] - m);
                l += s[i][j];
            }
    }

    // values of tokens that do not count are anything, NaN included: 0 instead
    __device__ __forceinline__ void drop_values(uint64_t bits) {
        const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
        for (int t = 0; t < 4 * SUB; t++) {
            const bool on = (bits >> (16 * (t / 4) + 4 * g + t % 4)) & 1;
#pragma unroll
            for (int c = 0; c < NV; c++)
#pragma unroll
                for (int w = 0; w < VW; w++) v[t][c][w] = on ? v[t][c][w] : 0u;
        }
    }

    __device__ __forceinline__ void gather(const f4* s) {
        if constexpr (T == DT_F32) {
#pragma unroll
            for (int c = 0; c < NV; c++)
#pragma unroll
                for (int e = 0; e < VE; e++)
#pragma unroll
                    for (int t = 0; t < 4; t++)
                        o[c][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(v[t][c][e]), s[0][t], o[c][e], 0, 0, 0);
        } else {
            // exp2(s - m) is at most 1: 2^-9 (bf16) or 2^-11 (f16) of each
            // term, as good as the output's own rounding
            const u4 p = {pack2<T>(s[0][0], s[0][1]), pack2<T>(s[0][2], s[0][3]), pack2<T>(s[1][0], s[1][1]),
                          pack2<T>(s[1][2], s[1][3])};
#pragma unroll
            for (int c = 0; c < NV; c++)
#pragma unroll
                for (int e = 0; e < VE; e++) {
                    const uint32_t sel = e % 2 ? 0x07060302u : 0x05040100u;
                    u4 x;
#pragma unroll
                    for (int t = 0; t < 4; t++) x[t] = __builtin_amdgcn_perm(v[2 * t + 1][c][e / 2], v[2 * t][c][e / 2], sel);
                    o[c][e] = mfma_qk<T>(x, p, o[c][e]);
                }
        }
    }

    // tiles first, first + NW, ... below last of one pair
    __device__ __forceinline__ void run(const AttnArgs& a, const Extent& ex, int r, int h, int qt, int first, int last) {
        const int lane = threadIdx.x & 63, in_tile = lane & (kTile - 1);
        m = kLowest;
        l = 0.f;
#pragma unroll
        for (int c = 0; c < NV; c++)
#pragma unroll
            for (int e = 0; e < VE; e++) o[c][e] = f4{0.f, 0.f, 0.f, 0.f};
        if (first >= last) return;
        if constexpr (!FULL) {
#pragma unroll
            for (int i = 0; i < SUB; i++)
#pragma unroll
                for (int c = 0; c < NC; c++) k[i][c] = u4{0, 0, 0, 0};
        }
        int t = ex.base + first * kTile + in_tile;
        int row = row_at(a, h, t, page_at(a, ex, r, t));
        load_q(a, r, h, qt);
        load_k(a, row);
        int page = page_at(a, ex, r, t + kUnit);
        load_v(a, row);
        for (int j = first; j < last; j += NW) {
            const bool more = j + NW < last;
            const uint64_t bits = __ballot(row >= 0);
            f4 s[SUB];
            scores(s);
            int next = 0;
            t += kUnit;
            if (more) {
                next = row_at(a, h, t, page);
                load_k(a, next);
                page = page_at(a, ex, r, t + kUnit);
            }
            soften(a, s, bits);
            if (bits != ~0ull) drop_values(bits);
            gather(s);
            if (more) {
                load_v(a, next);
                row = next;
            }
        }
        l = group_sum(l);
    }

    // the waves' results of one pair: out and lse, or (slot >= 0) a partial result
    __device__ __forceinline__ void join(const Params& p, int r, int h, int qt, int slot, float* lds) {
        const AttnArgs& a = p.a;
        const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, qi = lane & 15, g = lane >> 4;
        float* ml = lds + NW * p.rows * LS;  // [NW][16][2]
        const int rows = a.G - qt * 16 < 16 ? a.G - qt * 16 : 16;
        if (lane < 16) {
            ml[(w * 16 + lane) * 2] = m;
            ml[(w * 16 + lane) * 2 + 1] = l;
        }
        if (qi < rows) {
#pragma unroll
            for (int c = 0; c < NV; c++)
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int e = 0; e < VE; e += 4)
                        *reinterpret_cast<f4*>(lds + (w * p.rows + qi) * LS + (16 * c + 4 * g + i) * VE + e) =
                            f4{o[c][e][i], o[c][e + 1][i], o[c][e + 2][i], o[c][e + 3][i]};
        }
        __syncthreads();
        const int per = a.D / 4;
        for (int x = threadIdx.x; x < rows * per; x += NW * 64) {
            const int i = x / per, d = (x - i * per) * 4;
            float top = kLowest;
#pragma unroll
            for (int y = 0; y < NW; y++) top = fmaxf(top, ml[(y * 16 + i) * 2]);
            float sum = 0.f;
            f4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int y = 0; y < NW; y++) {
                const float f = __builtin_amdgcn_exp2f(ml[(y * 16 + i) * 2] - top);
                sum += ml[(y * 16 + i) * 2 + 1] * f;
                acc += *reinterpret_cast<const f4*>(lds + (y * p.rows + i) * LS + d) * f;
            }
            if (slot >= 0) {
                const int64_t at = (int64_t)slot * p.rows + i;
                *reinterpret_cast<f4*>(p.part_o + at * a.D + d) = acc;
                if (d == 0) {
                    p.part_ml[at * 2] = top;
                    p.part_ml[at * 2 + 1] = sum;
                }
            } else {
                store_row(a, r, h * a.G + qt * 16 + i, d, acc, top, sum);
            }
        }
        __syncthreads();
    }

    // four channels of a head's result; no token counted: 0 and -infinity
    __device__ __forceinline__ static void store_row(const AttnArgs& a, int r, int head, int d, f4 acc, float top, float sum) {
        const float f = sum == 0.f ? 0.f : 1.f / sum;
        const int64_t at = r * a.out_row + (int64_t)head * a.D + d;
        if (sum == 0.f) acc = f4{0.f, 0.f, 0.f, 0.f};
        if constexpr (T == DT_F32) {
            typedef float f4s __attribute__((ext_vector_type(4), aligned(4)));
            *reinterpret_cast<f4s*>(static_cast<float*>(a.out) + at) = acc * f;
        } else {
            typedef uint32_t u2s __attribute__((ext_vector_type(2), aligned(2)));
            *reinterpret_cast<u2s*>(static_cast<uint16_t*>(a.out) + at) =
                u2s{pack2<T>(acc[0] * f, acc[1] * f), pack2<T>(acc[2] * f, acc[3] * f)};
        }
        if (d == 0 && a.lse) a.lse[(int64_t)r * a.H + head] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
    }
};

extern __shared__ __attribute__((aligned(16))) float attn_lds[];

// one block per pair
template <int T, int DP, bool FULL, int NW>
__global__ __launch_bounds__(64 * NW) void attn_pair_kernel(Params p) {
    using A = Attn<T, DP, FULL, NW>;
    A x;
    const int w = threadIdx.x >> 6;
    const int r = blockIdx.x / p.HQ, hq = blockIdx.x - r * p.HQ, h = hq / p.QT, qt = hq - h * p.QT;
    const Extent ex = extent_of(p.a, r);
    x.run(p.a, ex, r, h, qt, w, (ex.end - ex.base + A::kTile - 1) / A::kTile);
    x.join(p, r, h, qt, -1, attn_lds);
}

// range blockIdx.x of P
template <int T, int DP, bool FULL, int NW>
__global__ __launch_bounds__(64 * NW) void attn_range_kernel(Params p) {
    using A = Attn<T, DP, FULL, NW>;
    constexpr int NT = 64 * NW;
    const AttnArgs& a = p.a;
    const int w = threadIdx.x >> 6, me = blockIdx.x;
    // units of the requests: thread i sums a stretch of them
    __shared__ int64_t sums[NT], found[2];
    const int each = (a.R + NT - 1) / NT, r0 = (int)threadIdx.x * each;
    const int r1 = r0 + each < a.R ? r0 + each : a.R;
    int64_t mine = 0;
    for (int r = r0; r < r1; r++) mine += units_of(extent_of(a, r), A::kUnit);
    sums[threadIdx.x] = mine;
    __syncthreads();
    int64_t before = 0, total = 0;
    for (int i = 0; i < NT; i++) {
        if (i < (int)threadIdx.x) before += sums[i];
        total += sums[i];
    }
    const int64_t units = total * p.HQ;
    const Ranges ranges(units, p.P);
    int64_t pos = ranges.first(me);
    const int64_t end = ranges.first(me + 1);
    if (threadIdx.x == 0) reinterpret_cast<Cut*>(p.meta)[me].r = -1;
    if (pos >= end) return;
    if (r0 < r1 && pos >= before * p.HQ && pos < (before + mine) * p.HQ) {
        int r = r0;
        for (;; r++) {
            const int n = units_of(extent_of(a, r), A::kUnit);
            if (pos < (before + n) * p.HQ) break;
            before += n;
        }
        found[0] = r;
        found[1] = before * p.HQ;
    }
    __syncthreads();
    int r = (int)found[0];
    Extent ex = extent_of(a, r);
    int n = units_of(ex, A::kUnit);
    int hq = (int)((pos - found[1]) / n), u = (int)(pos - found[1] - (int64_t)hq * n);
    if (threadIdx.x == 0 && u > 0 && pos - u >= ranges.first(me - 1))
        reinterpret_cast<Cut*>(p.meta)[me] = Cut{r, hq, u, n, units, 0};
    bool at_start = true;
    A x;
    while (pos < end) {
        if (hq == p.HQ) {
            hq = 0;
            ex = extent_of(a, ++r);
            n = units_of(ex, A::kUnit);
        }
        const int64_t left = end - pos;
        const int u1 = left < n - u ? u + (int)left : n;
        const int h = hq / p.QT, qt = hq - h * p.QT;
        const int tiles = (ex.end - ex.base + A::kTile - 1) / A::kTile;
        x.run(a, ex, r, h, qt, u * NW + w, u1 * NW < tiles ? u1 * NW : tiles);
        x.join(p, r, h, qt, u == 0 && u1 == n ? -1 : 2 * me + (at_start ? 0 : 1), attn_lds);
        at_start = false;
        pos += u1 - u;
        u = 0;
        hq++;
    }
}

// joins the partial results of the pair that the cut at range blockIdx.x's
// start goes through first; block (x, y) takes query row y
template <int T, int DP>
__global__ __launch_bounds__(256) void attn_join_kernel(Params p) {
    const AttnArgs& a = p.a;
    const int me = blockIdx.x, i = blockIdx.y;
    const Cut c = reinterpret_cast<const Cut*>(p.meta)[me];
    if (c.r < 0) return;
    const int h = c.hq / p.QT, qt = c.hq - h * p.QT;
    if (qt * 16 + i >= a.G) return;
    const Ranges ranges(c.units, p.P);
    const int64_t from = ranges.first(me) - c.u0;
    const int parts = ranges.of(from + c.n - 1) - (me - 1) + 1;
    const int slot0 = 2 * (me - 1) + (ranges.first(me - 1) == from ? 0 : 1);
    auto slot = [&](int s) { return (int64_t)(s == 0 ? slot0 : 2 * (me - 1 + s)) * p.rows + i; };
    __shared__ float red[256];
    __shared__ f4 sum_o[256];
    float top = kLowest;
    for (int s = threadIdx.x; s < parts; s += 256) top = fmaxf(top, p.part_ml[slot(s) * 2]);
    red[threadIdx.x] = top;
    __syncthreads();
    for (int k = 128; k > 0; k >>= 1) {
        if ((int)threadIdx.x < k) red[threadIdx.x] = fmaxf(red[threadIdx.x], red[threadIdx.x + k]);
        __syncthreads();
    }
    top = red[0];
    __syncthreads();
    // DP / 4 threads across a row, 1024 / DP of them in turn over the parts
    constexpr int across = DP / 4, turns = 256 / across;
    const int d = (int)threadIdx.x % across * 4, turn = (int)threadIdx.x / across;
    float sum = 0.f;
    f4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int s = turn; s < parts; s += turns) {
        const int64_t at = slot(s);
        const float f = __builtin_amdgcn_exp2f(p.part_ml[at * 2] - top);
        sum += p.part_ml[at * 2 + 1] * f;
        if (d < a.D) acc += *reinterpret_cast<const f4*>(p.part_o + at * a.D + d) * f;
    }
    red[threadIdx.x] = sum;
    sum_o[threadIdx.x] = acc;
    __syncthreads();
    if (turn == 0 && d < a.D) {
#pragma unroll
        for (int y = 1; y < turns; y++) {
            sum += red[y * across + threadIdx.x];
            acc += sum_o[y * across + threadIdx.x];
        }
        Attn<T, DP, true, 1>::store_row(a, c.r, h * a.G + qt * 16 + i, d, acc, top, sum);
    }
}

template <int T, int DP, bool FULL>
LuxStatus launch_d(Params& p, hipStream_t st) {
    constexpr int NW = 4;
    using A = Attn<T, DP, FULL, NW>;
    const size_t lds = A::lds_bytes(p.rows);
    const int64_t pairs = (int64_t)p.a.R * p.HQ;
    static const hipError_t attr_p = hipFuncSetAttribute(reinterpret_cast<const void*>(attn_pair_kernel<T, DP, FULL, NW>),
                                                         hipFuncAttributeMaxDynamicSharedMemorySize, (int)A::lds_bytes(16));
    static const hipError_t attr_r = hipFuncSetAttribute(reinterpret_cast<const void*>(attn_range_kernel<T, DP, FULL, NW>),
                                                         hipFuncAttributeMaxDynamicSharedMemorySize, (int)A::lds_bytes(16));
    if (attr_p != hipSuccess || attr_r != hipSuccess) return LuxStatus::Internal;
    // ranges: two blocks per CU, as many as the workspace has room for
    int P = 2 * p.a.cus;
    const size_t one = (size_t)p.rows * (p.a.D + 2) * 2 * 4 + sizeof(Cut);
    if ((size_t)P * one > p.a.ws_bytes) P = (int)(p.a.ws_bytes / one);
    const bool whole = P < 2 || p.a.columns * (int64_t)p.a.page <= A::kUnit;
    if (whole) {
        hipLaunchKernelGGL((attn_pair_kernel<T, DP, FULL, NW>), dim3((unsigned)pairs), dim3(64 * NW), lds, st, p);
    } else {
        p.P = P;
        p.meta = reinterpret_cast<int64_t*>(p.a.ws);
        p.part_ml = p.a.ws + (size_t)P * sizeof(Cut) / 4;
        p.part_o = p.part_ml + (size_t)P * 4 * p.rows;
        hipLaunchKernelGGL((attn_range_kernel<T, DP, FULL, NW>), dim3(P), dim3(64 * NW), lds, st, p);
        hipLaunchKernelGGL((attn_join_kernel<T, DP>), dim3(P, p.rows), dim3(256), 0, st, p);
    }
    return hipGetLastError() == hipSuccess ? LuxStatus::Ok : LuxStatus::Internal;
}

template <int T>
LuxStatus launch_t(const AttnArgs& a, hipStream_t st) {
    Params p = {};
    p.a = a;
    p.QT = (a.G + 15) / 16;
    p.HQ = a.Hk * p.QT;
    p.rows = a.G < 16 ? a.G : 16;
    if (a.D <= 64) return a.D == 64 ? launch_d<T, 64, true>(p, st) : launch_d<T, 64, false>(p, st);
    if (a.D <= 128) return a.D == 128 ? launch_d<T, 128, true>(p, st) : launch_d<T, 128, false>(p, st);
    return a.D == 256 ? launch_d<T, 256, true>(p, st) : launch_d<T, 256, false>(p, st);
}

extern template LuxStatus launch_t<DT_F32>(const AttnArgs&, hipStream_t);
extern template LuxStatus launch_t<DT_F16>(const AttnArgs&, hipStream_t);
extern template LuxStatus launch_t<DT_BF16>(const AttnArgs&, hipStream_t);

}  // namespace attn
}  // namespace lxq
