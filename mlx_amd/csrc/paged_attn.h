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
// a cut goes through leaves partial (m, l, O) in the workspace, which the last of
// its blocks to arrive joins.  At its last tile of a pair a wave already loads
// the first of the next one (256 requests up to 1024 tokens 107.5 us without,
// 103 with).
//
// Bound by HBM where the cache is long: 8 requests of 131072 tokens, 8 heads of
// 128 bf16 (4.3 GB) in 624 us, 6.9 TB/s; 64 ragged ones up to 8192 (1.1 GB) 181
// us, 6.2 TB/s.  Short calls are a chain of trips to memory (lengths, table,
// keys, partial results, counter, their join): one request of 4096 tokens, 32
// heads on 8 of 128 f16 (17 MB) 9.6 us.
#pragma once
#include "serving_device.h"

namespace lxq {
namespace attn {

typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4h __attribute__((ext_vector_type(4), aligned(2)));  // rows of q start anywhere
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kDevice = 16;  // cache policy of the partial results: device scope (sc1)
constexpr float kLowest = -0x1.fffffep127f;  // the maximum of no score: no finite score is below
constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.69314718055994531f;

struct Params {
    // a.scale and a.softcap as the kernels take them: scores by log2 e are s *
    // scale, or softcap tanh(y) with 2 y = s * scale
    AttnArgs a;
    int HQ;           // heads of keys times query tiles of a group
    int QT, rows;     // query tiles of a group; rows of a tile kept in partial results
    DivBy P, by_hq;   // ranges; division by HQ
    float* part_o;    // [2 P, rows, D]
    float* part_ml;   // [2 P, rows, 2]
    uint32_t part_o_bytes, part_ml_bytes;
};

// of `units` units, range w of P starts at first(w): the first units % P
// ranges are one unit longer
struct Ranges {
    int base, rem;
    __device__ Ranges(int units, const DivBy& P) : base(div_by(units, P)), rem(units - base * P.d) {}
    __device__ int first(int w) const { return w * base + (w < rem ? w : rem); }
    __device__ int of(int u) const {
        const int long_ones = rem * (base + 1);
        return u < long_ones ? (int)((uint32_t)u / (uint32_t)(base + 1)) : rem + (int)((uint32_t)(u - long_ones) / (uint32_t)base);
    }
};

// the tokens of request r that count: [start, end), and where tiles begin
struct Extent {
    int start, end, base;
};
__device__ __forceinline__ Extent extent_of(const AttnArgs& a, int n) {
    const int cap = a.pool > 0 ? a.columns * a.page : 0;
    n = n < 0 ? 0 : n > cap ? cap : n;
    const int s = a.window > 0 && n > a.window ? n - a.window : 0;
    return Extent{s, n, s & ~31};
}
// values that all lanes share, kept in scalar registers
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ Extent extent_at(const AttnArgs& a, int r) { return extent_of(a, uniform(a.lens[r])); }
// runs of `tokens` tokens (without a sign: a request may end just below 2^31)
__device__ __forceinline__ int runs_of(const Extent& e, int tokens) {
    return (int)(((uint32_t)(e.end - e.base) + (uint32_t)tokens - 1) / (uint32_t)tokens);
}
// units of `tokens` tokens; a request with none has one, which writes its zeros
__device__ __forceinline__ int units_of(const Extent& e, int tokens) {
    const int n = runs_of(e, tokens);
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

// two values >= 0 of the type, of x and y without their last bits
template <int T>
__device__ __forceinline__ uint32_t cut2(float x, float y) {
    if constexpr (T == DT_F16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x, y));
    else return __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302u);
}
// the type's smallest value (bf16: its smallest normal one) where they are below it
template <int T>
__device__ __forceinline__ uint32_t least2(uint32_t v) {
    typedef uint16_t h2 __attribute__((ext_vector_type(2)));
    constexpr uint16_t least = T == DT_F16 ? 0x0001 : 0x0080;
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(h2, v), h2{least, least}));
}

// slot of the s-th part of a pair that starts in range w0: a range keeps the part
// that its first units continue in slot 2 w, the one that its last units start in
// slot 2 w + 1
__device__ __forceinline__ uint32_t slot(int w0, int s) { return (uint32_t)(2 * (w0 + s) + (s == 0)); }

// x / d for whole numbers below 2^15: the half keeps the quotient off the next one
__device__ __forceinline__ int small_div(int x, int d) {
    return (int)(((float)x + 0.5f) * __builtin_amdgcn_rcpf((float)d));
}

__device__ __forceinline__ float wave_max(float v) {
    v = fmaxf(v, dpp_f<0xB1>(v));
    v = fmaxf(v, dpp_f<0x4E>(v));
    v = fmaxf(v, dpp_f<0x141>(v));
    v = fmaxf(v, dpp_f<0x140>(v));
    return fmaxf(fmaxf(lane_f(v, 0), lane_f(v, 16)), fmaxf(lane_f(v, 32), lane_f(v, 48)));
}

// max / sum over the four lanes that hold one query's tokens: both halves of a
// row or wave swap are the pair's values, in either order
__device__ __forceinline__ float group_max(float v) {
    uint32_t x = __float_as_uint(v);
    auto p = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = __float_as_uint(fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1])));
    p = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
}
__device__ __forceinline__ float group_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// a wave's part of a pair
struct Piece {
    int r, h, qt;
    int first, last;  // tiles
    Extent ex;
};

// T: type of q, cache and out; DP: head_dim, or that rounded up to 64, 128, 192 or 256;
// FULL: head_dim is DP; WHOLE: pages hold whole runs of 16 tokens, so that a run
// has one page and its rows one scalar base (else each lane finds its token's
// row and the others take it from there); ONCE: cache loads that leave no copy
template <int T, int DP, bool FULL, bool WHOLE, bool ONCE, int NW>
struct Attn {
    static constexpr int ES = T == DT_F32 ? 4 : 2, E = 16 / ES;  // bytes; elements per 16 bytes
    static constexpr int SUB = T == DT_F32 ? 1 : 2, kTile = 16 * SUB;
    static constexpr int NC = DP / (4 * E);                  // 16-byte chunks of a key row per lane
    static constexpr int VE = DP == 192 ? 4 : E < DP / 16 ? E : DP / 16;  // channels of a value row per lane and load
    static constexpr int NV = DP / (16 * VE);                // loads per value row
    static constexpr int VW = VE * ES / 4;                   // their words
    static constexpr int kUnit = kTile * NW;
    static constexpr int LS = DP + 4;                        // LDS row of a query, in floats
    // the weights are 2^kLift exp2(s - m), here and in the partial results: f16
    // ends at 2^-24, and the weights below 2^-25 that a wave would lose beside a
    // large one may together be most of the result (16 heads of 256 on one, 37
    // requests up to 5000 tokens: 30.4 us so and without)
    static constexpr float kLift = T == DT_F16 ? 14.f : 0.f, kDown = T == DT_F16 ? 0x1p-14f : 1.f;
    typedef uint32_t uv __attribute__((ext_vector_type(VW)));

    static constexpr int NT = 64 * NW;
    static constexpr int kChunk = 64, kFinish = 16 * (kChunk + 4) + 4 * NT;
    // the waves' results, or what finish() keeps; a word
    static constexpr size_t lds_floats(int rows) {
        return (size_t)NW * (rows * LS + 32) > kFinish ? (size_t)NW * (rows * LS + 32) : kFinish;
    }
    static constexpr size_t lds_bytes(int rows) { return lds_floats(rows) * 4 + 16; }

    __device__ __forceinline__ static int dim(const AttnArgs& a) { return FULL ? DP : a.D; }
    // channel d of a row, in a run of channels that ends at `end`, is one of
    // head_dim's: below DP - 64 all are, smaller head dims take the next smaller form
    __device__ __forceinline__ static bool has(const AttnArgs& a, int d, int end) { return FULL || end <= DP - 64 || d < a.D; }

    u4 q[NC], k[SUB][NC];
    uv v[4 * SUB][NV];
    f4 o[NV][VE];
    float m, l;
    int page[SUB], row[SUB];  // pages of the next tile, rows of the one in k and v: per run of 16, or the lane's token's in [0]
    uint32_t bits;            // the tokens that count of the tile in k and v

    __device__ __forceinline__ Attn() {
        if constexpr (!FULL) {  // the channels past head_dim, which no load touches
#pragma unroll
            for (int i = 0; i < SUB; i++)
#pragma unroll
                for (int c = 0; c < NC; c++) k[i][c] = u4{0, 0, 0, 0};
        }
    }

    static constexpr uint32_t kAll = SUB == 2 ? 0xffffffffu : 0xffffu;

    // pages of the tile at token t0, which may be past the request's end and past 2^31
    __device__ __forceinline__ void look(const AttnArgs& a, const Extent& e, int r, uint32_t t0) {
        if constexpr (WHOLE) {
            // (address space 4: scalar loads)
            const auto* table = (const __attribute__((address_space(4))) int32_t*)a.table + (int64_t)r * a.columns;
#pragma unroll
            for (int s = 0; s < SUB; s++) {
                const uint32_t t = t0 + 16 * s;
                page[s] = t < (uint32_t)e.end && t + 16 > (uint32_t)e.start ? table[div_by((int)t, a.div)] : -1;
            }
        } else {
            const uint32_t t = t0 + (threadIdx.x & (kTile - 1));
            page[0] = t >= (uint32_t)e.start && t < (uint32_t)e.end ? a.table[(int64_t)r * a.columns + div_by((int)t, a.div)] : -1;
        }
    }
    // the rows they stand for; masked ones read row 0
    __device__ __forceinline__ void resolve(const AttnArgs& a, const Extent& e, int h, int t0) {
        if constexpr (WHOLE) {
            const int lo = e.start > t0 ? e.start - t0 : 0, n = e.end - t0;
            bits = (n >= kTile ? kAll : (1u << n) - 1u) & (kAll << lo);
#pragma unroll
            for (int s = 0; s < SUB; s++) {
                const int t = t0 + 16 * s, at = t - div_by(t, a.div) * a.page;
                const bool there = (uint32_t)page[s] < (uint32_t)a.pool;
                row[s] = there ? (page[s] * a.Hk + h) * a.page + at : 0;
                if (!there) bits &= ~(0xffffu << (16 * s));
            }
        } else {
            const int t = t0 + (int)(threadIdx.x & (kTile - 1)), at = t - div_by(t, a.div) * a.page;
            const bool there = (uint32_t)page[0] < (uint32_t)a.pool;
            row[0] = there ? (page[0] * a.Hk + h) * a.page + at : 0;
            bits = (uint32_t)__ballot(there) & kAll;
        }
    }
    // the row of token i (of lane's choice in [0, 16)) of run s, in bytes from the cache's start: scalar and lane part
    __device__ __forceinline__ const char* at_row(const AttnArgs& a, const void* cache, int s, int i) const {
        const char* p = static_cast<const char*>(cache);
        const uint32_t len = (uint32_t)(dim(a) * ES);
        if constexpr (WHOLE) return p + (uint64_t)(uint32_t)row[s] * len + (uint32_t)i * len;
        else return p + (uint64_t)(uint32_t)__shfl(row[0], 16 * s + i) * len;
    }

    // columns past the group's end take its first query: nobody reads their results
    __device__ __forceinline__ void load_q(const AttnArgs& a, int r, int h, int qt) {
        const int lane = threadIdx.x & 63, i = qt * 16 + (lane & 15);
        const char* p = static_cast<const char*>(a.q) + (r * a.q_row + (int64_t)(h * a.G + (i < a.G ? i : 0)) * dim(a)) * ES;
#pragma unroll
        for (int c = 0; c < NC; c++) {
            const int d = (4 * c + (lane >> 4)) * E;
            q[c] = *reinterpret_cast<const u4h*>(p + (has(a, d, 4 * (c + 1) * E) ? d * ES : 0));
            if (!has(a, d, 4 * (c + 1) * E)) q[c] = u4{0, 0, 0, 0};
        }
    }

    template <class V>
    __device__ __forceinline__ static V load(const char* p) {
        if constexpr (ONCE) return __builtin_nontemporal_load(reinterpret_cast<const V*>(p));
        else return *reinterpret_cast<const V*>(p);
    }
    // channels past head_dim stay zero
    __device__ __forceinline__ void load_k(const AttnArgs& a) {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int s = 0; s < SUB; s++) {
            const char* p = at_row(a, a.kc, s, lane & 15) + (lane >> 4) * 16;
#pragma unroll
            for (int c = 0; c < NC; c++)
                if (has(a, (4 * c + (lane >> 4)) * E, 4 * (c + 1) * E)) k[s][c] = load<u4>(p + c * 64);
        }
    }
    __device__ __forceinline__ void load_v(const AttnArgs& a) {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int t = 0; t < 4 * SUB; t++) {
            const char* p = at_row(a, a.vc, t / 4, 4 * (lane >> 4) + t % 4);
#pragma unroll
            for (int c = 0; c < NV; c++) {
                const int d = (16 * c + (lane & 15)) * VE;  // past head_dim: channels that are not stored
                v[t][c] = load<uv>(p + (has(a, d, 16 * (c + 1) * VE) ? d * ES : 0));
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

    // s (scores) to exp2 of their distance to the running maximum, lifted; bits: the
    // tile's tokens that count
    __device__ __forceinline__ void soften(const AttnArgs& a, f4* s, uint32_t bits) {
        const int g = (threadIdx.x & 63) >> 4;
        if (a.softcap > 0.f) {
#pragma unroll
            for (int i = 0; i < SUB; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) s[i][j] = a.softcap * tanh_of(s[i][j] * a.scale);
        } else {
#pragma unroll
            for (int i = 0; i < SUB; i++) s[i] *= a.scale;
        }
        if (bits != kAll) {
#pragma unroll
            for (int i = 0; i < SUB; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) s[i][j] = (bits >> (16 * i + 4 * g + j)) & 1 ? s[i][j] : -INFINITY;
        }
        float mx = kLowest;
#pragma unroll
        for (int i = 0; i < SUB; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) mx = fmaxf(mx, s[i][j]);
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
        const float from = m - kLift;
#pragma unroll
        for (int i = 0; i < SUB; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                s[i][j] = __builtin_amdgcn_exp2f(s[i][j] - from);
                l += s[i][j];
            }
    }

    // values of tokens that do not count are anything, NaN included: 0 instead
    __device__ __forceinline__ void drop_values(uint32_t bits) {
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
            // The weights as the sum of two values of the type (one alone is off
            // by as much as the output's own rounding: 8 requests of 131072
            // tokens bf16 2.3e-3 off in 64 bits, 1.7e-3 so, 621.8 and 622.8 us).
            // Both are above 0, so that an infinite value of v stays one: the
            // first is cut, not rounded, and neither is below the type's smallest
            // (bf16: normal) value, a weight of 2^-38 in f16 and 2^-126 in bf16.
            u4 p[2];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float x = s[i / 2][i % 2 * 2], y = s[i / 2][i % 2 * 2 + 1];
                const uint32_t high = cut2<T>(x, y);
                p[0][i] = least2<T>(high);
                const float hx = T == DT_F16 ? f16_to_f32(high & 0xffffu) : __uint_as_float(high << 16);
                const float hy = T == DT_F16 ? f16_to_f32(high >> 16) : __uint_as_float(high & 0xffff0000u);
                p[1][i] = least2<T>(pack2<T>(x - hx, y - hy));
            }
#pragma unroll
            for (int c = 0; c < NV; c++)
#pragma unroll
                for (int e = 0; e < VE; e++) {
                    const uint32_t sel = e % 2 ? 0x07060302u : 0x05040100u;
                    u4 x;
#pragma unroll
                    for (int t = 0; t < 4; t++) x[t] = __builtin_amdgcn_perm(v[2 * t + 1][c][e / 2], v[2 * t][c][e / 2], sel);
                    o[c][e] = mfma_qk<T>(x, p[0], o[c][e]);
                    o[c][e] = mfma_qk<T>(x, p[1], o[c][e]);
                }
        }
    }

    // a tile's scores into the running maximum, sum and result
    __device__ __forceinline__ void take(const AttnArgs& a, f4* s, uint32_t now) {
        soften(a, s, now);
        if (now != kAll) drop_values(now);
        gather(s);
    }

    // One wave's tiles of a piece: first, first + NW, ... below last.  At its
    // last tile it loads the first tile of `next`, so that the card does not
    // wait between pieces; `primed`: so did the piece before this one.
    __device__ __forceinline__ void run(const AttnArgs& a, const Piece& c, const Piece& next, bool& primed) {
        m = kLowest;
        l = 0.f;
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int e = 0; e < VE; e++) o[i][e] = f4{0.f, 0.f, 0.f, 0.f};
        if (c.first >= c.last) return;
        int t = c.ex.base + c.first * kTile;
        if (!primed) {
            look(a, c.ex, c.r, t);
            load_q(a, c.r, c.h, c.qt);
            resolve(a, c.ex, c.h, t);
            load_k(a);
            look(a, c.ex, c.r, (uint32_t)t + kUnit);
            load_v(a);
        }
        f4 s[SUB];
        for (int j = c.first + NW; j < c.last; j += NW) {
            const uint32_t now = bits;
            scores(s);
            t += kUnit;
            resolve(a, c.ex, c.h, t);
            load_k(a);
            look(a, c.ex, c.r, (uint32_t)t + kUnit);
            take(a, s, now);
            load_v(a);
        }
        // the last tile: no branch between its scores and the loads of the loop
        // above, which would have the scores wait for the values too
        const uint32_t now = bits;
        scores(s);
        primed = next.first < next.last;
        if (primed) {
            t = next.ex.base + next.first * kTile;
            look(a, next.ex, next.r, t);
            load_q(a, next.r, next.h, next.qt);
            resolve(a, next.ex, next.h, t);
            load_k(a);
            look(a, next.ex, next.r, (uint32_t)t + kUnit);
        }
        take(a, s, now);
        if (primed) load_v(a);
        l = group_sum(l);
    }

    // the waves' results of one pair: out and lse, or (slot >= 0) a partial result
    __device__ __forceinline__ void join(const Params& p, int r, int h, int qt, int slot, float* lds) {
        const AttnArgs& a = p.a;
        const int lane = threadIdx.x & 63, w = uniform(threadIdx.x >> 6), qi = lane & 15, g = lane >> 4;
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
        const int per = dim(a) / 4;
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
                store_part(p, slot, i, d, acc, top, sum);
            } else {
                store_row(a, r, h * a.G + qt * 16 + i, d, acc, top, sum);
            }
        }
        __syncthreads();
    }

    __device__ __forceinline__ static __amdgpu_buffer_rsrc_t o_rsrc(const Params& p) {
        return __builtin_amdgcn_make_buffer_rsrc(p.part_o, 0, (int)p.part_o_bytes, 0x00020000);
    }
    __device__ __forceinline__ static __amdgpu_buffer_rsrc_t ml_rsrc(const Params& p) {
        return __builtin_amdgcn_make_buffer_rsrc(p.part_ml, 0, (int)p.part_ml_bytes, 0x00020000);
    }

    // four channels of a row of a partial result, at device scope: the block that
    // joins it may be on another die
    __device__ __forceinline__ static void store_part(const Params& p, int slot, int i, int d, f4 acc, float top, float sum) {
        const uint32_t at = (uint32_t)(slot * p.rows + i);
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4, acc), o_rsrc(p), (at * dim(p.a) + d) * 4, 0, kDevice);
        if (d == 0) __builtin_amdgcn_raw_buffer_store_b64(u2{__float_as_uint(top), __float_as_uint(sum)}, ml_rsrc(p), at * 8, 0, kDevice);
    }

    // Joins parts at, at + hop, ... (`parts` of them) of the pair that starts in
    // range w0 into the result, or (to >= 0) into the partial result in slot
    // `to`, which may be the first one's.  An item is four channels of a row.  A
    // wave takes whole rows of (m, l), a part per lane, and leaves the parts'
    // weights in LDS; then a thread adds up its item, and where the items are
    // fewer than the threads, several threads share an item's parts and meet in
    // LDS.  Items past NT come with at most kChunk parts.
    __device__ __forceinline__ static void finish(const Params& p, int r, int h, int qt, int w0, int at, int hop, int parts, int to,
                                                  float* lds) {
        const AttnArgs& a = p.a;
        const int lane = threadIdx.x & 63, w = uniform(threadIdx.x >> 6);
        const int rows = a.G - qt * 16 < 16 ? a.G - qt * 16 : 16, per = dim(a) / 4, items = rows * per;
        const int turns = items < NT ? small_div(NT, items) : 1;
        const int turn = turns > 1 ? small_div(threadIdx.x, items) : 0;
        const __amdgpu_buffer_rsrc_t ro = o_rsrc(p), rm = ml_rsrc(p);
        float* weight = lds;                                       // [16][kChunk]
        float* of_row = lds + 16 * kChunk;                         // [16][4]: maximum, sum, rescaling
        f4* all = reinterpret_cast<f4*>(lds + 16 * (kChunk + 4));  // [NT]
        for (int x0 = 0; x0 < items; x0 += NT) {
            const int x = x0 + (int)threadIdx.x - turn * items;
            const bool on = x < items && turn < turns;
            const int i = on ? small_div(x, per) : 0, d = on ? (x - i * per) * 4 : 0;
            f4 acc = {0.f, 0.f, 0.f, 0.f};
            for (int c0 = 0; c0 < parts; c0 += kChunk) {
                const int n = parts - c0 < kChunk ? parts - c0 : kChunk;
                const bool weigh = c0 > 0 || x0 == 0;
                u2 ml[16 / NW];
                if (weigh)
#pragma unroll
                    for (int k = 0; k < 16 / NW; k++) {
                        const int y = w + k * NW;
                        if (y >= rows) break;
                        ml[k] = __builtin_amdgcn_raw_buffer_load_b64(
                            rm, lane < n ? (slot(w0, at + (c0 + lane) * hop) * p.rows + y) * 8 : 0x80000000u, 0, kDevice);
                    }
                // up to kBatch of the thread's parts in flight together, in
                // groups of 8 as far as there are any
                constexpr int kBatch = 16;
                u4 o[kBatch];
                const uint32_t step = (uint32_t)(p.rows * dim(a)) * 4, stride = 2 * turns * hop * step;
                auto load_o = [&](int s0) {
                    int s = s0 + turn;
                    uint32_t from = (uint32_t)(i * dim(a) + d) * 4 + slot(w0, at + (c0 + s) * hop) * step;
#pragma unroll
                    for (int q = 0; q < kBatch; q += 8) {
                        if (s0 + q * turns >= n) break;
#pragma unroll
                        for (int k = q; k < q + 8; k++) {
                            // past the last: an offset past the end, which reads zeros
                            o[k] = __builtin_amdgcn_raw_buffer_load_b128(ro, s < n ? from : 0x80000000u, 0, kDevice);
                            from += stride - (k == 0 && at + (c0 + s) * hop == 0 ? step : 0);
                            s += turns;
                        }
                    }
                };
                load_o(0);
                if (weigh)
#pragma unroll
                    for (int k = 0; k < 16 / NW; k++) {
                        const int y = w + k * NW;
                        if (y >= rows) break;
                        float* mine = of_row + 4 * y;
                        const float m = lane < n ? __uint_as_float(ml[k][0]) : kLowest, was = c0 ? mine[0] : kLowest;
                        const float top = fmaxf(was, wave_max(m)), f = lane < n ? __builtin_amdgcn_exp2f(m - top) : 0.f;
                        const float sum = wave_sum(f * __uint_as_float(ml[k][1])), f0 = __builtin_amdgcn_exp2f(was - top);
                        weight[y * kChunk + lane] = f;
                        if (lane == 0) {
                            mine[1] = (c0 ? mine[1] * f0 : 0.f) + sum;
                            mine[0] = top;
                            mine[2] = f0;
                        }
                    }
                __syncthreads();
                acc *= of_row[4 * i + 2];
                for (int s0 = 0; s0 < n; s0 += kBatch * turns) {
                    if (s0) load_o(s0);
#pragma unroll
                    for (int q = 0; q < kBatch; q += 8) {
                        if (s0 + q * turns >= n) break;
#pragma unroll
                        for (int k = q; k < q + 8; k++) {
                            const int s = s0 + turn + k * turns;
                            acc += __builtin_bit_cast(f4, o[k]) * weight[i * kChunk + (s < kChunk ? s : kChunk - 1)];
                        }
                    }
                }
                __syncthreads();
            }
            if (turns > 1) {
                all[threadIdx.x] = acc;
                __syncthreads();
                if (on && turn == 0)
                    for (int k = 1; k < turns; k++) acc += all[threadIdx.x + k * items];
                __syncthreads();
            }
            if (on && turn == 0) {
                if (to >= 0) store_part(p, to, i, d, acc, of_row[4 * i], of_row[4 * i + 1]);
                else store_row(a, r, h * a.G + qt * 16 + i, d, acc, of_row[4 * i], of_row[4 * i + 1]);
            }
        }
        __syncthreads();
    }

    // four channels of a head's result; no token counted: 0 and -infinity
    __device__ __forceinline__ static void store_row(const AttnArgs& a, int r, int head, int d, f4 acc, float top, float sum) {
        const float f = sum == 0.f ? 0.f : 1.f / sum;
        const int64_t at = r * a.out_row + (int64_t)head * dim(a) + d;
        if (sum == 0.f) acc = f4{0.f, 0.f, 0.f, 0.f};
        if constexpr (T == DT_F32) {
            typedef float f4s __attribute__((ext_vector_type(4), aligned(4)));
            *reinterpret_cast<f4s*>(static_cast<float*>(a.out) + at) = acc * f;
        } else {
            typedef uint32_t u2s __attribute__((ext_vector_type(2), aligned(2)));
            *reinterpret_cast<u2s*>(static_cast<uint16_t*>(a.out) + at) =
                u2s{pack2<T>(acc[0] * f, acc[1] * f), pack2<T>(acc[2] * f, acc[3] * f)};
        }
        if (d == 0 && a.lse) a.lse[(int64_t)r * a.H + head] = sum == 0.f ? -INFINITY : (top + log2f(sum * kDown)) * kLn2;
    }
};

extern __shared__ __attribute__((aligned(16))) float attn_lds[];

// waves per SIMD that the registers allow (three at 64 and 128 channels were as
// fast or slower: 64 heads on 4, up to 4096 tokens of 64 channels 60.6 us with
// two, 63.4 with three)
template <int DP>
constexpr int kWaves = DP == 256 ? 1 : 2;

// one block per pair
template <int T, int DP, bool FULL, bool WHOLE, bool ONCE, int NW>
__global__ __launch_bounds__(64 * NW, (kWaves<DP>)) void attn_pair_kernel(Params p, int first) {
    using A = Attn<T, DP, FULL, WHOLE, ONCE, NW>;
    A x;
    const int w = uniform(threadIdx.x >> 6);
    const int pair = first + (int)blockIdx.x, r = pair / p.HQ, hq = pair - r * p.HQ, h = hq / p.QT, qt = hq - h * p.QT;
    const Extent ex = extent_at(p.a, r);
    bool primed = false;
    x.run(p.a, Piece{r, h, qt, w, runs_of(ex, A::kTile), ex}, Piece{}, primed);
    x.join(p, r, h, qt, -1, attn_lds);
}

// requests in front of unit pos / HQ, found by each wave for itself: lane i sums
// the units of a stretch of requests
struct Requests {
    int all;      // units of all requests, for one of a request's pairs
    int each, through, mine;
    int len;      // of the lane's last request
    __device__ __forceinline__ Requests(const AttnArgs& a, int unit) : each((a.R + 63) / 64), mine(0), len(0) {
        const int lane = threadIdx.x & 63;
        for (int r = lane * each; r < (lane + 1) * each && r < a.R; r++) {
            len = a.lens[r];
            mine += units_of(extent_of(a, len), unit);
        }
        through = wave_scan(mine);
        all = __builtin_amdgcn_readlane(through, 63);
    }
    // the request with unit `at`, the units before it and its length
    __device__ __forceinline__ int find(const AttnArgs& a, int unit, int at, int& before, int& its) const {
        const int lane = threadIdx.x & 63;
        int s = __popcll(__ballot(through <= at)), r = s * each;
        before = __builtin_amdgcn_readlane(through - mine, s);
        its = __builtin_amdgcn_readlane(len, s);
        for (; each > 1; r += 64) {
            const int at_lane = r + lane < a.R ? a.lens[r + lane] : 0;
            const int n = r + lane < a.R ? units_of(extent_of(a, at_lane), unit) : 0;
            const int sum = before + wave_scan(n);
            s = __popcll(__ballot(sum <= at));
            if (s < 64) {
                before = __builtin_amdgcn_readlane(sum - n, s);
                its = __builtin_amdgcn_readlane(at_lane, s);
                r += s;
                break;
            }
            before = __builtin_amdgcn_readlane(sum, 63);
        }
        return r;
    }
};

// The ranges that hold a pair's units [from, from + n).  Parts of up to 256 KB are
// joined at once; more in groups of about their square root, each by the last of
// its ranges to arrive, and the groups by the last group.  16 heads of 256 f16 on
// one, parts of 16 KB: a request of 65536 tokens beside 63 of 20 (some 250 parts)
// 92 us at once, 35 in groups; 4 of 16384 (64 parts) 32.8 and 26.3; 10 (26 parts)
// 47.1 and 48.1; 16 (16 parts) 53.4 and 57.2.
struct Parts {
    int w0, count;
    __device__ __forceinline__ Parts(const Ranges& ranges, int from, int n) : w0(ranges.of(from)) {
        count = ranges.of(from + n - 1) - w0 + 1;
    }
};
// parts of a group: all, or a power of two
__device__ __forceinline__ int group_of(const Params& p, int count) {
    if (count * (int64_t)(p.rows * p.a.D * 4) <= 256 * 1024) return count;
    int n = 8;
    while (n * n < count) n *= 2;
    return n;
}

// thread 0 counts one in; true for all threads of the last of `all`, which
// leaves the counter at 0
__device__ __forceinline__ bool count_in(uint32_t* c, int all, int* word) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this thread's partial results are out
    __syncthreads();
    if (threadIdx.x == 0) {
        const bool last = __hip_atomic_fetch_add(c, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)(all - 1);
        if (last) __hip_atomic_store(c, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *word = last;
    }
    __syncthreads();
    return uniform(*word);
}

// range blockIdx.x of P
template <int T, int DP, bool FULL, bool WHOLE, bool ONCE, int NW>
__global__ __launch_bounds__(64 * NW, (kWaves<DP>)) void attn_range_kernel(Params p) {
    using A = Attn<T, DP, FULL, WHOLE, ONCE, NW>;
    const AttnArgs& a = p.a;
    const int w = uniform(threadIdx.x >> 6), me = blockIdx.x;
    const Requests requests(a, A::kUnit);
    const Ranges ranges(requests.all * p.HQ, p.P);
    int pos = ranges.first(me);
    const int end = ranges.first(me + 1);
    if (pos >= end) return;
    int before, len;
    int r = requests.find(a, A::kUnit, div_by(pos, p.by_hq), before, len);
    Extent ex = extent_of(a, len);
    int n = units_of(ex, A::kUnit);
    int hq = (int)((uint32_t)(pos - before * p.HQ) / (uint32_t)n), u = pos - before * p.HQ - hq * n;
    bool primed = false;
    A x;
    // the piece of pair (r, hq) from unit u on, as far as the range goes
    auto piece = [&] {
        const int h = p.QT == 1 ? hq : hq / p.QT, tiles = runs_of(ex, A::kTile);
        const int last = (u + (end - pos) < n ? u + (end - pos) : n) * NW;
        return Piece{r, h, hq - h * p.QT, u * NW + w, last < tiles ? last : tiles, ex};
    };
    Piece c = piece();
    int r0 = 0, h0 = 0, qt0 = 0, w0 = 0, n0 = 0, r1 = 0, h1 = 0, qt1 = 0, w1 = 0, n1 = 0;  // the pairs to join, of n parts
    int* word = reinterpret_cast<int*>(attn_lds + A::lds_floats(p.rows));
    while (pos < end) {
        const int from = pos - u, all = n, u0 = u, u1 = u + (end - pos) < n ? u + (end - pos) : n;
        const bool part = u0 > 0 || u1 < n;
        pos += u1 - u0;
        u = 0;
        if (pos < end && ++hq == p.HQ) {
            hq = 0;
            ex = extent_at(a, ++r);
            n = units_of(ex, A::kUnit);
        }
        const Piece next = piece();  // at the range's end: no tiles
        x.run(a, c, next, primed);
        x.join(p, c.r, c.h, c.qt, !part ? -1 : 2 * me + (u0 == 0), attn_lds);
        if (part) {
            // counters: P for the pairs that start in a range and go past its
            // end (only one does) and its first group, P for the group that
            // starts in a range behind that one, P for the pairs' groups
            const Parts parts(ranges, from, all);
            const int group = group_of(p, parts.count);
            int g = 0, in_group = parts.count;
            if (group < parts.count) {
                g = (me - parts.w0) & -group;
                in_group = parts.count - g < group ? parts.count - g : group;
            }
            if (count_in(a.count + (g ? p.P.d + parts.w0 + g : parts.w0), in_group, word)) {
                // joined at the end of the range, when the tiles' registers
                // are free; a range has at most two cut pairs
                if (u0 > 0) r0 = c.r, h0 = c.h, qt0 = c.qt, w0 = parts.w0, n0 = parts.count;
                else r1 = c.r, h1 = c.h, qt1 = c.qt, w1 = parts.w0, n1 = parts.count;
            }
            __syncthreads();
        }
        c = next;
    }
#pragma unroll 1
    for (int i = 0; i < 2; i++) {
        if (n0) {
            const int group = group_of(p, n0);
            int parts = n0, hop = 1;
            if (group < n0) {
                const int g = (me - w0) & -group, groups = (n0 + group - 1) / group;
                A::finish(p, r0, h0, qt0, w0, g, 1, n0 - g < group ? n0 - g : group, (int)slot(w0, g), attn_lds);
                parts = count_in(a.count + 2 * p.P.d + w0, groups, word) ? groups : 0;
                hop = group;
            }
            if (parts) A::finish(p, r0, h0, qt0, w0, 0, hop, parts, -1, attn_lds);
        }
        r0 = r1, h0 = h1, qt0 = qt1, w0 = w1, n0 = n1;
        n1 = 0;
    }
}

template <int T, int DP, bool FULL, bool WHOLE, bool ONCE>
LuxStatus launch_d(Params& p, hipStream_t st) {
    constexpr int NW = 4;
    using A = Attn<T, DP, FULL, WHOLE, ONCE, NW>;
    const size_t lds = A::lds_bytes(p.rows);
    const int64_t pairs = (int64_t)p.a.R * p.HQ;
    auto pair = attn_pair_kernel<T, DP, FULL, WHOLE, ONCE, NW>;
    auto range = attn_range_kernel<T, DP, FULL, WHOLE, ONCE, NW>;
    static const bool attr = [&] {
        for (const void* k : {(const void*)pair, (const void*)range})
            if (hipFuncSetAttribute(k, hipFuncAttributeMaxDynamicSharedMemorySize, (int)A::lds_bytes(16)) != hipSuccess) return false;
        return true;
    }();
    if (!attr) return LuxStatus::Internal;
    // ranges: as many blocks as run at once, and the workspace has room for
    int P = kWaves<DP> * p.a.cus;
    const size_t one = (size_t)p.rows * (p.a.D + 2) * 2 * 4;
    if ((size_t)P * one > p.a.ws_bytes) P = (int)(p.a.ws_bytes / one);
    if (P > p.a.counts / 3) P = p.a.counts / 3;
    const int64_t longest = ((int64_t)p.a.columns * p.a.page + A::kUnit - 1) / A::kUnit + 1;  // units of a pair
    // Tables of up to two units: a block per pair.  Longer ones may belong to short
    // or uneven requests, and are cut: 512 requests up to 2000 tokens, 8 heads on 2
    // of 64, 53.8 us (64.2 whole), 1024 100.3 (102.7); but up to 300 tokens, 8 heads
    // on one of 128, 1024 take 27.2 (19.7)
    const bool whole = P < 2 || longest <= 2 || longest * pairs >= (1ll << 31);
    if (whole) {
        launch_blocks(pairs, 64 * NW, [&](int first, unsigned n) {
            hipLaunchKernelGGL(pair, dim3(n), dim3(64 * NW), lds, st, p, first);
        });
        return hipGetLastError() == hipSuccess ? LuxStatus::Ok : LuxStatus::Internal;
    }
    p.P = DivBy(P);
    p.by_hq = DivBy(p.HQ);
    p.part_ml = p.a.ws;
    p.part_ml_bytes = (uint32_t)P * 2 * p.rows * 8;
    p.part_o = p.part_ml + p.part_ml_bytes / 4;
    p.part_o_bytes = (uint32_t)P * 2 * p.rows * p.a.D * 4;
    hipLaunchKernelGGL(range, dim3(P), dim3(64 * NW), lds, st, p);
    return hipGetLastError() == hipSuccess ? LuxStatus::Ok : LuxStatus::Internal;
}

template <int T, int DP, bool FULL>
LuxStatus launch_full(Params& p, hipStream_t st) {
    if (p.a.page % 16) return launch_d<T, DP, FULL, false, false>(p, st);
    // Rows that end on cache lines, of a pool that the last-level cache (256 MB)
    // cannot hold: loads that leave no copy (8 requests of 131072 tokens 701 ->
    // 625 us, 64 ragged ones up to 8192 203 -> 180).  A smaller pool may still
    // be there from the call before (256 requests up to 128 tokens 18.5 us with
    // such loads, 16.4 without; out of HBM 19.6 and 20.2), and a line that two
    // rows share is wanted twice (head_dim 80, 64 requests up to 2048 tokens
    // 46.1 and 41.1).
    const int64_t row = (int64_t)p.a.D * (T == DT_F32 ? 4 : 2);
    const bool once = row % 128 == 0 && 2 * row * p.a.pool * p.a.page * p.a.Hk >= (256ll << 20);
    return once ? launch_d<T, DP, FULL, true, true>(p, st) : launch_d<T, DP, FULL, true, false>(p, st);
}
template <int T, int DP>
LuxStatus launch_dp(Params& p, hipStream_t st) {
    return p.a.D == DP ? launch_full<T, DP, true>(p, st) : launch_full<T, DP, false>(p, st);
}

template <int T>
LuxStatus launch_t(const AttnArgs& a, hipStream_t st) {
    Params p = {};
    p.a = a;
    p.QT = (a.G + 15) / 16;
    p.HQ = a.Hk * p.QT;
    p.rows = a.G < 16 ? a.G : 16;
    p.a.scale = a.softcap > 0.f ? 2.f * kLog2e * a.scale / a.softcap : kLog2e * a.scale;
    p.a.softcap = a.softcap * kLog2e;
    if (a.D <= 64) return launch_dp<T, 64>(p, st);
    if (a.D <= 128) return launch_dp<T, 128>(p, st);
    // Padded to 192 channels instead of 256: two blocks per CU.  64 requests up to
    // 4096 tokens, 32 heads on 8, bf16 / f32: 136 channels 117.1 / 220.0 us instead of
    // 125.2 / 251.0, 160 135.1 / 244.3 (138.5 / 275.5), 184 150.6 / 285.0 (156.4 /
    // 310.2); 16 of 2048 with a head each f32 160 67.2 (88.4).  Slower at 184 with
    // one head of keys (37 up to 5000, 16 heads on it: 28.5 / 47.1, 26.7 / 44.8).
    return a.D <= 192 ? launch_dp<T, 192>(p, st) : launch_dp<T, 256>(p, st);
}

extern template LuxStatus launch_t<DT_F32>(const AttnArgs&, hipStream_t);
extern template LuxStatus launch_t<DT_F16>(const AttnArgs&, hipStream_t);
extern template LuxStatus launch_t<DT_BF16>(const AttnArgs&, hipStream_t);

}  // namespace attn
}  // namespace lxq
