// paged_chunk.h -- attention of chunks of new tokens over a paged cache.
//
// A tile is the queries of up to TB consecutive new tokens of one request for
// the heads that share one head of keys: RG x 32 rows, a row per token and head.
// A wave holds 32 rows and meets its cached tokens 32 at a time:
//   S^T[token, row] = K . Q^T      A = K rows from LDS, B = Q in registers
//   P^T = exp2(S^T - m)            running maximum m and sum l per row
//   O^T[channel, row] += V^T . P^T A = V^T, read from LDS transposed
// A 32x32 result has its column (the row of queries) in the lane and its rows
// (tokens (i % 4) + 8 (i / 4) + 4 (lane / 32)) in the lane's registers, which is
// the B operand of the second product if its k is numbered that way: P never
// leaves its lane, and the rescaling of O by a new maximum is the lane's own
// factor.  In 16 bits V's operand with that numbering is two transposed reads of
// four tokens each; in f32 a plain read per token.
//
// K and V reach LDS by global->LDS transfers, NS - 1 stages ahead, in 16-byte
// chunks whose place within a row is permuted by the row (the transfer takes the
// permuted chunk, LDS is filled in order), so that neither read meets itself in
// the banks.  KG groups of waves may share a tile's rows and take a part of each
// stage's tokens; they meet in LDS at the end.
//
// Work.  Tiles of all requests and heads are laid end to end, each as long as the
// stages that it sees, and cut into P equal ranges, one per block: causal, ragged
// and windowed batches and single requests fill the card alike.  A tile that a
// cut goes through leaves partial (m, l, O) in the workspace, which a second
// launch joins.  Ranges follow each other head by head, and an XCD takes a run
// of ranges, so that its L2 holds the keys that its blocks share.
#pragma once
#include "prompt.h"
#include "serving_device.h"

namespace lxq {
namespace chunk {

typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4h __attribute__((ext_vector_type(4), aligned(2)));  // rows of q start anywhere
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));

constexpr float kLowest = -0x1.fffffep127f;  // the maximum of no score: no finite score is below
constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.69314718055994531f;
constexpr float kLeast = 0x1p-126f;

// a tile that starts in a range and ends behind it: its parts, where it is
struct Cut {
    int32_t parts, r, tile, hq;
};

struct Params {
    ChunkArgs a;
    int GT, QT, HQ;   // heads of a tile; tiles of a group; heads of keys times those
    int TB;           // tokens of a tile
    int slots, each;  // places of tiles (some may be empty); places per thread
    DivBy by_tb, by_gt;
    int P;
    float c;          // scores by log2 e are s * c (or, capped, cap tanh(y) with 2 y log2 e = s * c)
    float cap;        // softcap log2 e
    uint32_t flip;    // sign bits of q: c is not negative
    float* part_o;    // [2 P, rows, DP]
    float* part_ml;   // [2 P, rows, 2]
    Cut* cuts;        // [P]
};

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
// (address space 4: scalar loads)
__device__ __forceinline__ int scalar_at(const int32_t* p, int64_t i) {
    return ((const __attribute__((address_space(4))) int32_t*)p)[i];
}
// The kernel's argument, read again from where it lies: a loop keeps the scalars
// that it uses, and those of the code around it are no burden to it
__device__ __forceinline__ const Params& argument() {
    auto p = (const __attribute__((address_space(4))) Params*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *(const Params*)p;
}
// the same value, for code that is to work out again what follows from it instead
// of keeping it in registers through other loops
__device__ __forceinline__ int afresh(int v) {
    asm volatile("" : "+v"(v));
    return v;
}
__device__ __forceinline__ int clamp(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }

// rows and tokens of a tile
struct Tile {
    int first, m;    // first new token (row of q), tokens
    int pos, n;      // position of the first one; tokens held
    int base, end;   // cached tokens that the tile sees lie in [base, end)
    int units;       // stages; a tile that sees nothing has one, which writes its zeros
};
template <int ST>
__device__ __forceinline__ Tile tile_of(const Params& p, int r, int tile) {
    const ChunkArgs& a = p.a;
    Tile t;
    const int cap = a.pool > 0 ? a.columns * a.page : 0;
    const int s0 = clamp(a.starts[r], 0, a.T), s1 = clamp(a.starts[r + 1], s0, a.T), i0 = tile * p.TB;
    t.first = s0 + i0;
    t.m = clamp(s1 - s0 - i0, 0, p.TB);
    t.pos = clamp(a.seq[r], 0, a.columns * a.page) + i0;
    t.n = clamp(a.lens[r], 0, cap);
    t.end = t.pos + t.m < t.n ? t.pos + t.m : t.n;
    t.base = a.window > 0 && t.pos + 1 > a.window ? (t.pos + 1 - a.window) & ~15 : 0;
    t.units = t.end > t.base ? (int)((uint32_t)(t.end - t.base + ST - 1) / ST) : 1;
    return t;
}

// Request r's tiles take places from starts[r] / TB + r on: as many as it has
// tiles, or one more.
__device__ __forceinline__ int place_of(const Params& p, int r) { return div_by(clamp(p.a.starts[r], 0, p.a.T), p.by_tb) + r; }
__device__ __forceinline__ int request_of_place(const Params& p, int place) {
    int lo = 0, hi = p.a.R - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (place_of(p, mid) <= place) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}
// the request of new token t: none after it starts there
__device__ __forceinline__ int request_of_token(const ChunkArgs& a, int t) {
    int lo = 0, hi = a.R - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (scalar_at(a.starts, mid) <= t) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// of `units` units, range w of P starts at first(w): the first units % P ranges
// are one unit longer
struct Ranges {
    uint64_t base, rem;
    __device__ Ranges(uint64_t units, int P) : base(units / (uint32_t)P), rem(units - base * (uint32_t)P) {}
    __device__ uint64_t first(int w) const { return (uint64_t)w * base + ((uint64_t)w < rem ? (uint64_t)w : rem); }
    __device__ int of(uint64_t u) const {
        const uint64_t long_ones = rem * (base + 1);
        return (int)(u < long_ones ? u / (base + 1) : rem + (u - long_ones) / base);
    }
};

// slot of the s-th part of a tile that starts in range w0: a range keeps the part
// that its first units continue in slot 2 w, the one that its last units start in
// slot 2 w + 1
__device__ __forceinline__ int slot(int w0, int s) { return 2 * (w0 + s) + (s == 0); }

template <int N>
__device__ __forceinline__ void wait_vm() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// the barrier behind which other waves read what this wave wrote to LDS, or
// overwrite what it reads
__device__ __forceinline__ void barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}
// global -> LDS: lane l copies 16 bytes to LDS m0 + 16 l
__device__ __forceinline__ void dma16(uint32_t m0v, const void* sbase, uint32_t voff) {
    asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(m0v), "v"(voff), "s"(sbase) : "memory", "m0");
}
__device__ __forceinline__ void dma16a(uint32_t m0v, const void* addr) {
    asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(m0v), "v"(addr) : "memory", "m0");
}

__device__ __forceinline__ float other_half(float v) {
    const uint32_t x = __float_as_uint(v);
    const auto q = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return __uint_as_float((threadIdx.x & 32) ? q[0] : q[1]);
}
__device__ __forceinline__ float half_max(float v) {
    const uint32_t x = __float_as_uint(v);
    const auto q = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return fmaxf(__uint_as_float(q[0]), __uint_as_float(q[1]));
}

// tanh(y) from z = 2 y log2 e: 1 - 2 / (1 + exp2(z)), off by 2^-22 at most.  Where y
// is small that is a large share of it, and times a large cap a large part of the
// score: there the series up to y^11, whose next term is below 2^-28 of y at 0.3.
__device__ __forceinline__ float tanh_of(float z) {
    const float far = fmaf(__builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z)), -2.f, 1.f);
    const float y = z * (0.5f * kLn2), q = y * y;
    float near = fmaf(q, -1382.f / 155925.f, 62.f / 2835.f);
    near = fmaf(q, near, -17.f / 315.f);
    near = fmaf(q, near, 2.f / 15.f);
    near = fmaf(q, near, -1.f / 3.f);
    return fabsf(y) < 0.3f ? fmaf(y * q, near, y) : far;
}

template <int T>
__device__ __forceinline__ f16v mfma(const u4& x, const u4& y, f16v c) {
    if constexpr (T == DT_F16) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, x), __builtin_bit_cast(f16x8, y), c, 0, 0, 0);
    } else if constexpr (T == DT_BF16) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), c, 0, 0, 0);
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++)
            c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(x[j]), __uint_as_float(y[j]), c, 0, 0, 0);
        return c;
    }
}

typedef const __attribute__((address_space(3))) char* lds_ptr;

// T: type of q, cache and out; DP: head_dim rounded up to 64, 128, 192 or 256; RG
// row groups times KG groups of tokens = waves; BT: tokens of a group's part of a
// stage; NS: stages in LDS; WHOLE: pages hold whole runs of the tokens that one
// transfer takes, so that a run has one scalar address (else each lane finds its
// token's)
template <int T, int DP, int RG, int KG, int BT, int NS, bool WHOLE>
struct Chunk {
    static constexpr int ES = T == DT_F32 ? 4 : 2, E = 16 / ES;  // bytes; elements per 16 bytes
    static constexpr int RS = (DP == 192 ? 256 : DP) * ES;       // LDS row of a token
    static constexpr int CPR = RS / 16, TI = 64 / CPR;           // its 16-byte chunks; tokens per transfer
    static constexpr int NW = RG * KG, NT = 64 * NW, ST = BT * KG, NI = ST / TI / NW;
    static_assert(NI * TI * NW == ST && TI <= 16, "every wave moves whole runs");
    static constexpr int kMat = ST * RS, kStage = 2 * kMat;
    static constexpr int NK = DP / (2 * E), ND = DP / 32, NB = BT / 32;
    static constexpr int KM = CPR < 16 ? 7 : 15;
    static constexpr int LS = DP + 4;  // row of the groups' meeting, in floats
    static constexpr int kMeet = KG > 1 ? NW * 32 * (LS + 2) * 4 : 0;
    static constexpr int kLds = NS * kStage > kMeet ? NS * kStage : kMeet;
    // the weights are 2^kLift exp2(s - m): f16 ends at 2^-24, and many weights
    // below 2^-25 beside a large one may together be most of the result
    static constexpr float kLift = T == DT_F16 ? 14.f : 0.f, kDown = T == DT_F16 ? 0x1p-14f : 1.f;
    // m may stay behind the maximum by this much (log2): O is rescaled less often,
    // and weights stay below 2^16 in f16
    static constexpr float kBehind = T == DT_F16 ? 1.f : 8.f;

    // where the registers are short, operands of so many steps ahead are loaded and
    // no more (0: as the compiler likes)
    static constexpr int kFence = T == DT_F32 && DP >= 128 ? 2 : DP == 256 || (DP == 128 && !WHOLE) ? 4 : 0;

    // permutations of a row's chunks
    __device__ __forceinline__ static int k_turn(int row) { return row & KM; }
    __device__ __forceinline__ static int v_turn(int row) {
        if constexpr (T == DT_F32) return ((row >> 2) & 1) << 3;
        else return CPR < 16 ? ((row >> 1) & 1) << 2 : (row & 3) << 2;
    }

    char* lds;
    int lane, w, rg, kg;
    uint32_t koff, voff;  // bytes of the lane's chunk in a run at a multiple of 16 tokens

    u4 q[NK];
    f16v o[ND];
    float m, l;
    int lo, len;  // the cached tokens that the lane's row sees

    __device__ __forceinline__ explicit Chunk(char* mem) : lds(mem) {
        lane = threadIdx.x & 63;
        w = uniform(threadIdx.x >> 6);
        rg = w % RG;
        kg = w / RG;
        const int ri = lane / CPR, c = lane % CPR;
        koff = (uint32_t)((c ^ k_turn(ri)) * 16);
        voff = (uint32_t)((c ^ v_turn(ri)) * 16);
    }

    // a stage's transfers into LDS stage `buf`: tokens from tb on, those past the
    // tile's last one from its row
    __device__ __forceinline__ void fill(const ChunkArgs& a, const Tile& t, int r, int hk, int tb, int buf) {
        const uint32_t dst = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds + (uint32_t)(buf * kStage);
        const uint32_t row_bytes = (uint32_t)(a.D * ES);
        const int ri = lane / CPR;
#pragma unroll
        for (int j = 0; j < NI; j++) {
            const int run = w * NI + j;
            const uint32_t at_lds = dst + (uint32_t)(run * 1024);
            const uint32_t kc = koff ^ (uint32_t)(k_turn(run * TI) * 16), vc = voff ^ (uint32_t)(v_turn(run * TI) * 16);
            const int t0 = tb + run * TI;
            if constexpr (WHOLE) {
                const int tr = t0 < t.end ? t0 : (t.end - 1) & ~(TI - 1);
                const int col = div_by(tr, a.div);
                int pg = scalar_at(a.table, (int64_t)r * a.columns + col);
                pg = (uint32_t)pg < (uint32_t)a.pool ? pg : 0;
                const uint64_t row = (uint64_t)(uint32_t)((pg * a.Hk + hk) * a.page + (tr - col * a.page));
                const char* kp = static_cast<const char*>(a.kc) + row * row_bytes;
                const char* vp = static_cast<const char*>(a.vc) + row * row_bytes;
                const int last = t.end - 1 - tr;  // rows behind the last one: the last one's
                const uint32_t at_row = (uint32_t)(ri < last ? ri : last) * row_bytes;
                if (a.D == RS / ES) {
                    dma16(at_lds, kp, kc + at_row);
                    dma16(at_lds + kMat, vp, vc + at_row);
                } else {
                    if (kc < row_bytes) dma16(at_lds, kp, kc + at_row);
                    if (vc < row_bytes) dma16(at_lds + kMat, vp, vc + at_row);
                }
            } else {
                int tok = t0 + ri;
                tok = tok < t.end ? tok : t.end - 1;
                const int col = div_by(tok, a.div);
                int pg = a.table[(int64_t)r * a.columns + col];
                pg = (uint32_t)pg < (uint32_t)a.pool ? pg : 0;
                const uint64_t row = (uint64_t)(uint32_t)((pg * a.Hk + hk) * a.page + (tok - col * a.page));
                if (kc < row_bytes) dma16a(at_lds, static_cast<const char*>(a.kc) + row * row_bytes + kc);
                if (vc < row_bytes) dma16a(at_lds + kMat, static_cast<const char*>(a.vc) + row * row_bytes + vc);
            }
        }
    }

    // row of the tile -> token of the tile, head; rows past the tile's take its last
    __device__ __forceinline__ static int token_of(const Params& p, const Tile& t, int row, int qt, int& head) {
        const int last = t.m * p.GT - 1;
        row = row < last ? row : last < 0 ? 0 : last;
        const int i = div_by(row, p.by_gt);
        head = qt * p.GT + row - i * p.GT;
        return i;
    }
    __device__ __forceinline__ static bool has_row(const Params& p, const Tile& t, int row, int qt) {
        if (row >= t.m * p.GT) return false;
        const int i = div_by(row, p.by_gt);
        return qt * p.GT + row - i * p.GT < p.a.G;
    }
    __device__ __forceinline__ static void sees(const ChunkArgs& a, const Tile& t, int i, int& from, int& to) {
        const int pos = t.pos + i;
        from = a.window > 0 && pos + 1 > a.window ? pos + 1 - a.window : 0;
        to = pos + 1 < t.n ? pos + 1 : t.n;
    }

    __device__ __forceinline__ void load_q(const Params& p, const Tile& t, int hk, int qt) {
        const ChunkArgs& a = p.a;
        int head;
        const int i = token_of(p, t, rg * 32 + (lane & 31), qt, head);
        head = head < a.G ? head : a.G - 1;
        const char* src = static_cast<const char*>(a.q) + ((int64_t)(t.first + i) * a.q_row + (int64_t)(hk * a.G + head) * a.D) * ES;
        const int h = afresh(lane >> 5);
#pragma unroll
        for (int k = 0; k < NK; k++) {
            const int d = (2 * k + h) * E;
            q[k] = *reinterpret_cast<const u4h*>(src + (d < a.D ? d * ES : 0));
            q[k] = d < a.D ? q[k] ^ p.flip : u4{0, 0, 0, 0};
            if (k % 16 == 15) __builtin_amdgcn_sched_barrier(0);
        }
        int from, to;
        sees(a, t, i, from, to);
        lo = from;
        len = to > from ? to - from : 0;
    }

    // which of the 32 NB tokens from tb on have a page
    __device__ __forceinline__ uint64_t pages_there(const ChunkArgs& a, const Tile& t, int r, int tb) const {
        const int tok = tb + lane;
        const bool in = lane < BT && tok < t.end;
        const int pg = in ? a.table[(int64_t)r * a.columns + div_by(tok, a.div)] : -1;
        return __ballot((uint32_t)pg < (uint32_t)a.pool);
    }

    // a group's BT tokens of a stage, from position tb on, into m, l and o
    __device__ __forceinline__ void take(const Params& p, const Tile& t, int r, int tb, int buf, bool masked, bool holes) {
        const ChunkArgs& a = p.a;
        const int h = lane >> 5, l31 = lane & 31;
        lds_ptr kb = (lds_ptr)lds + buf * kStage + kg * BT * RS, vb = kb + kMat;
        f16v s[NB];
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int i = 0; i < 16; i++) s[b][i] = 0.f;
        const uint32_t ka = (uint32_t)(l31 * RS) + (uint32_t)((h ^ k_turn(l31)) * 16);
#pragma unroll
        for (int k = 0; k < NK; k++) {
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const u4 x = *reinterpret_cast<const __attribute__((address_space(3))) u4*>(kb + (ka ^ (k * 32)) + b * 32 * RS);
                s[b] = mfma<T>(x, q[k], s[b]);
            }
            if (kFence > 0 && k % kFence == kFence - 1) __builtin_amdgcn_sched_barrier(0);
        }
        if (a.softcap > 0.f) {
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int i = 0; i < 16; i++) s[b][i] = p.cap * tanh_of(s[b][i] * p.c);
        }
        const float c = a.softcap > 0.f ? 1.f : p.c;
        if (masked) {
            const int from = lo - tb - 4 * h;  // against the token's number without the lane's 4 h
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    s[b][i] = (uint32_t)(32 * b + (i & 3) + 8 * (i >> 2) - from) < (uint32_t)len ? s[b][i] : -INFINITY;
                    if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);
                }
            if (holes) {
                const uint64_t there = pages_there(a, t, r, tb) >> (4 * h);
                uint32_t bits[2] = {(uint32_t)there, (uint32_t)(there >> 32)};
#pragma unroll
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        s[b][i] = (bits[b] >> ((i & 3) + 8 * (i >> 2))) & 1 ? s[b][i] : -INFINITY;
                        if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);
                    }
            }
        }
        float mx = kLowest;
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int i = 0; i < 16; i++) mx = fmaxf(mx, s[b][i]);
        mx = half_max(mx);
        if (__any((mx - m) * c > kBehind)) {
            const float to = fmaxf(m, mx), f = __builtin_amdgcn_exp2f((m - to) * c);
            m = to;
            l *= f;
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int i = 0; i < 16; i++) o[d][i] *= f;
        }
        // below every product of a maximum: a masked score's weight is 0 then, and
        // so is that of a row with no score yet
        const float from = fmaxf(m * c, -0x1p126f) - kLift;
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
                s[b][i] = __builtin_amdgcn_exp2f(fmaf(s[b][i], c, -from));
                l += s[b][i];
            }
        if constexpr (T == DT_F32) {
            const uint32_t va = (uint32_t)(4 * h * RS) + (uint32_t)(((l31 >> 2) ^ v_turn(4 * h)) * 16 + (lane & 3) * 4);
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    if (kFence > 0 && i % 2 == 0) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int d = 0; d < ND; d++) {
                        const float x = *reinterpret_cast<const __attribute__((address_space(3))) float*>(
                            vb + (va ^ (d * 128)) + (32 * b + (i & 3) + 8 * (i >> 2)) * RS);
                        o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(x, s[b][i], o[d], 0, 0, 0);
                    }
                }
        } else {
            // One value of the type per weight: off by half a step of it each, in
            // either direction, as the result itself is once
            const int i4 = (lane & 15) >> 2;
            const uint32_t va = (uint32_t)((4 * h + i4) * RS) +
                                (uint32_t)((((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ v_turn(4 * h + i4)) * 16) + (lane & 1) * 8);
#pragma unroll
            for (int kb16 = 0; kb16 < 2 * NB; kb16++) {
                if (kFence > 0) __builtin_amdgcn_sched_barrier(0);
                u4 x;
#pragma unroll
                for (int j = 0; j < 4; j++) x[j] = pack2<T>(s[kb16 / 2][8 * (kb16 & 1) + 2 * j], s[kb16 / 2][8 * (kb16 & 1) + 2 * j + 1]);
#pragma unroll
                for (int d = 0; d < ND; d++) {
                    typedef __attribute__((address_space(3))) s4* tr_ptr;
                    const s4 y0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)(vb + (va ^ (d * 64)) + 16 * kb16 * RS));
                    const s4 y1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)(vb + (va ^ (d * 64)) + (16 * kb16 + 8) * RS));
                    const u2 z0 = __builtin_bit_cast(u2, y0), z1 = __builtin_bit_cast(u2, y1);
                    o[d] = mfma<T>(u4{z0[0], z0[1], z1[0], z1[1]}, x, o[d]);
                }
            }
        }
    }

    // the maximum by log2 e that goes with l and o
    __device__ __forceinline__ static float top_of(const Params& p, float mm) { return fmaxf(mm * (p.a.softcap > 0.f ? 1.f : p.c), -0x1p126f); }

    // four channels of a row of the tile: into out, or a partial result
    __device__ __forceinline__ static void store4(const Params& p, const Tile& t, int hk, int qt, int to, int row, int d, f4 acc, float top, float sum) {
        if (to >= 0) {
            const int64_t at = (int64_t)to * (RG * 32) + row;
            *reinterpret_cast<f4*>(p.part_o + at * DP + d) = acc;
            if (d == 0) *reinterpret_cast<u2*>(p.part_ml + at * 2) = u2{__float_as_uint(top), __float_as_uint(sum)};
            return;
        }
        int head;
        const int i = token_of(p, t, row, qt, head);
        store_out(p.a, t.first + i, hk * p.a.G + head, d, acc, top, sum);
    }
    // no position counted: 0 and -infinity
    __device__ __forceinline__ static void store_out(const ChunkArgs& a, int tok, int head, int d, f4 acc, float top, float sum) {
        const float f = sum == 0.f ? 0.f : 1.f / sum;
        const int64_t at = (int64_t)tok * a.out_row + (int64_t)head * a.D + d;
        if (sum == 0.f) acc = f4{0.f, 0.f, 0.f, 0.f};
        if (d < a.D) {
            if constexpr (T == DT_F32) {
                typedef float f4s __attribute__((ext_vector_type(4), aligned(4)));
                *reinterpret_cast<f4s*>(static_cast<float*>(a.out) + at) = acc * f;
            } else {
                typedef uint32_t u2s __attribute__((ext_vector_type(2), aligned(2)));
                *reinterpret_cast<u2s*>(static_cast<uint16_t*>(a.out) + at) =
                    u2s{pack2<T>(acc[0] * f, acc[1] * f), pack2<T>(acc[2] * f, acc[3] * f)};
            }
        }
        if (d == 0 && a.lse) a.lse[(int64_t)tok * a.H + head] = sum == 0.f ? -INFINITY : (top + log2f(sum * kDown)) * kLn2;
    }

    __device__ __forceinline__ static float value(const void* base, int64_t i) {
        if constexpr (T == DT_F32) return static_cast<const float*>(base)[i];
        else return T == DT_F16 ? f16_to_f32(static_cast<const uint16_t*>(base)[i]) : bf16_to_f32(static_cast<const uint16_t*>(base)[i]);
    }

    // One row over the cached tokens of [from, to), by one wave and token by token:
    // for rows that a value which is not finite reached.  In the tile's products it
    // reaches rows that do not see it too (0 times infinity); here each row meets
    // its own tokens alone.  A weight never falls to 0 before an infinite value.
    __device__ __forceinline__ static void alone(const Params& p, int first, int pos, int n, int r, int hk, int head, int i, int from, int to,
                                              float* part_o, float* part_ml) {
        const ChunkArgs& a = p.a;
        constexpr int NV = DP / 64;
        const int lane = threadIdx.x & 63, at = pos + i;
        const int lo = a.window > 0 && at + 1 > a.window ? at + 1 - a.window : 0, hi = at + 1 < n ? at + 1 : n;
        const float c = a.softcap > 0.f ? 1.f : p.c;
        from = from > lo ? from : lo;
        to = to < hi ? to : hi;
        float q[NV], acc[NV], m = kLowest, l = 0.f;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int d = lane + 64 * j;
            const float x = d < a.D ? value(a.q, (int64_t)(first + i) * a.q_row + (int64_t)(hk * a.G + head) * a.D + d) : 0.f;
            q[j] = p.flip ? -x : x;
            acc[j] = 0.f;
        }
        for (int t = from; t < to; t++) {
            const int col = div_by(t, a.div), pg = scalar_at(a.table, (int64_t)r * a.columns + col);
            if ((uint32_t)pg >= (uint32_t)a.pool) continue;
            const int64_t row = (int64_t)((pg * a.Hk + hk) * a.page + (t - col * a.page)) * a.D;
            float s = 0.f, v[NV];
#pragma unroll
            for (int j = 0; j < NV; j++) {
                const int d = lane + 64 * j;
                s = fmaf(d < a.D ? value(a.kc, row + d) : 0.f, q[j], s);
                v[j] = d < a.D ? value(a.vc, row + d) : 0.f;
            }
            s = wave_sum(s);
            if (a.softcap > 0.f) s = p.cap * tanh_of(s * p.c);
            const float was = m;
            m = fmaxf(m, s);
            const float f = fmaxf(__builtin_amdgcn_exp2f((was - m) * c), kLeast);
            const float w = __builtin_amdgcn_exp2f(fmaf(s, c, -fmaxf(m * c, -0x1p126f)));
            l = fmaf(l, f, w);
#pragma unroll
            for (int j = 0; j < NV; j++) acc[j] = fmaf(fabsf(v[j]) == INFINITY ? fmaxf(w, kLeast) : w, v[j], acc[j] * f);
        }
        const float up = 1.f / kDown, top = fmaxf(m * c, -0x1p126f);
        const int tok = first + i, hd = hk * a.G + head;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int d = lane + 64 * j;
            if (part_o) {
                part_o[d] = acc[j] * up;
            } else if (d < a.D) {
                const float y = l == 0.f ? 0.f : acc[j] / l;
                store_f(a.out, (size_t)((int64_t)tok * a.out_row + (int64_t)hd * a.D + d), T, y);
            }
        }
        if (lane == 0) {
            if (part_o) {
                part_ml[0] = top;
                part_ml[1] = l * up;
            } else if (a.lse) {
                a.lse[(int64_t)tok * a.H + hd] = l == 0.f ? -INFINITY : (top + log2f(l)) * kLn2;
            }
        }
    }

    __device__ __forceinline__ void clear() {
        for (int i = threadIdx.x * 16; i < NS * kStage; i += NT * 16) *reinterpret_cast<u4*>(lds + i) = u4{0, 0, 0, 0};
    }

    // stages u0 .. u1 - 1 of a tile; to: the slot of a partial result, or -1
    __device__ __forceinline__ void piece(const Tile& t, int r, int hk, int qt, int u0, int u1, int to, uint32_t* bad) {
        const Params& p = argument();
        const ChunkArgs& a = p.a;
        const int first_tok = t.base + u0 * ST, last_tok = t.base + u1 * ST < t.end ? t.base + u1 * ST : t.end;
        const bool any = last_tok > first_tok;
        // are there pages that are none
        bool none = false;
        if (any) {
            const int c0 = div_by(first_tok, a.div), c1 = div_by(last_tok - 1, a.div);
            for (int c = c0 + (int)threadIdx.x; c <= c1; c += NT)
                none |= (uint32_t)a.table[(int64_t)r * a.columns + c] >= (uint32_t)a.pool;
        }
        if (threadIdx.x < RG) bad[threadIdx.x] = 0;
        const bool holes = __syncthreads_or(none);
        if (any) {
#pragma unroll
            for (int s = 0; s < NS - 1; s++)
                if (u0 + s < u1) fill(a, t, r, hk, first_tok + s * ST, s);
        }
        load_q(p, t, hk, qt);
        // what the compiler knows to be in flight ends here, not at its first use in the loop
        __builtin_amdgcn_s_waitcnt((0x7 << 4) | (0xF << 8));
        // the wave's rows: the first one's tokens and the last one's
        int head, lo0, hi0, lo1, hi1;
        sees(a, t, token_of(p, t, rg * 32, qt, head), lo0, hi0);
        sees(a, t, token_of(p, t, rg * 32 + 31, qt, head), lo1, hi1);
        const bool rows = rg * 32 < t.m * p.GT;
        m = kLowest;
        l = 0.f;
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[d][i] = 0.f;
        if (any) {
            int buf = 0;
            for (int u = u0; u < u1; u++) {
                if (NS > 2 && u1 - 1 - u >= NS - 2) wait_vm<WHOLE ? (NS - 2) * 2 * NI : 0>();
                else wait_vm<0>();
                barrier();
                const int ahead = u + NS - 1;
                if (ahead < u1) fill(a, t, r, hk, t.base + ahead * ST, buf == 0 ? NS - 1 : buf - 1);
                const int tb = t.base + u * ST + kg * BT;
                if (rows && tb < hi1 && tb + BT > lo0) take(p, t, r, tb, buf, holes || tb < lo1 || tb + BT > hi0, holes);
                buf = buf == NS - 1 ? 0 : buf + 1;
            }
        }
        l += other_half(l);
        const int h = afresh(lane >> 5), l31 = afresh(lane & 31);
        // 0 where all sums are finite, else NaN
        float z = 0.f;
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int i = 0; i < 16; i++) z = fmaf(o[d][i], 0.f, z);
        z += other_half(z);
        const uint32_t mine = (uint32_t)__ballot(z != z && fabsf(l) < INFINITY);
        if (lane == 0 && rows && mine) atomicOr(&bad[rg], mine);
        __syncthreads();
        const Params& e = argument();
        if constexpr (KG == 1) {
            const int row = rg * 32 + l31;
            if (has_row(e, t, row, qt) && !((bad[rg] >> l31) & 1)) {
                const float top = top_of(e, m);
#pragma unroll
                for (int d = 0; d < ND; d++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        store4(e, t, hk, qt, to, row, 32 * d + 8 * i + 4 * h, f4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]}, top, l);
            }
        } else {
            float* sums = reinterpret_cast<float*>(lds);
            float* ml = sums + NW * 32 * LS;
            float* mine_o = sums + (w * 32 + l31) * LS;
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    *reinterpret_cast<f4*>(mine_o + 32 * d + 8 * i + 4 * h) = f4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
            if (h == 0) {
                ml[(w * 32 + l31) * 2] = top_of(e, m);
                ml[(w * 32 + l31) * 2 + 1] = l;
            }
            __syncthreads();
            constexpr int per = DP / 4;
            for (int x = threadIdx.x; x < RG * 32 * per; x += NT) {
                const int row = x / per, d = (x - row * per) * 4;
                if (!has_row(e, t, row, qt) || ((bad[row >> 5] >> (row & 31)) & 1)) continue;
                float top = -0x1p126f;
#pragma unroll
                for (int g = 0; g < KG; g++) top = fmaxf(top, ml[(g * RG * 32 + row) * 2]);
                float sum = 0.f;
                f4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int g = 0; g < KG; g++) {
                    const float f = __builtin_amdgcn_exp2f(ml[(g * RG * 32 + row) * 2] - top);
                    sum += ml[(g * RG * 32 + row) * 2 + 1] * f;
                    acc += *reinterpret_cast<const f4*>(sums + (g * RG * 32 + row) * LS + d) * f;
                }
                store4(e, t, hk, qt, to, row, d, acc, top, sum);
            }
        }
        if (KG > 1 && e.a.D < RS / ES) {  // the meeting was where no transfer fills
            __syncthreads();
            clear();
        }
        for (int g = 0; g < RG; g++) {
            uint32_t rows_left = (uint32_t)uniform((int)bad[g]);
            for (int k = 0; rows_left; k++) {
                const int row = g * 32 + __builtin_ctz(rows_left);
                rows_left &= rows_left - 1;
                if (k % NW != w || !has_row(e, t, row, qt)) continue;
                int hd;
                const int i = token_of(e, t, row, qt, hd);
                const int64_t at = (int64_t)to * (RG * 32) + row;
                alone(e, t.first, t.pos, t.n, r, hk, hd, i, first_tok, last_tok, to >= 0 ? e.part_o + at * DP : nullptr, e.part_ml + at * 2);
            }
        }
    }
};

extern __shared__ __attribute__((aligned(16))) char chunk_lds[];

template <int T, int DP, int RG, int KG, int BT, int NS, bool WHOLE>
__global__ __launch_bounds__(64 * RG * KG, RG * KG / 4) void chunk_kernel(Params p) {
    using A = Chunk<T, DP, RG, KG, BT, NS, WHOLE>;
    constexpr int NW = A::NW, ST = A::ST;
    __shared__ int part[NW], own[3];
    __shared__ uint32_t bad[RG];
    const ChunkArgs& a = p.a;
    const int tid = threadIdx.x, lane = tid & 63;
    // an XCD takes every eighth block
    const int me = p.P % 8 == 0 ? (int)(blockIdx.x & 7) * (p.P / 8) + (int)(blockIdx.x >> 3) : (int)blockIdx.x;
    A x(chunk_lds);
    if (a.D < A::RS / A::ES) x.clear();  // chunks that no transfer fills
    // stages of the thread's places, and of all of them for one head
    const int s0 = tid * p.each, s1 = s0 + p.each < p.slots ? s0 + p.each : p.slots;
    int mine = 0;
    auto walk = [&](auto f) {
        if (s0 >= s1) return;
        int r = request_of_place(p, s0), from = place_of(p, r);
        for (int s = s0; s < s1; s++) {
            if (r + 1 < a.R) {
                const int next = place_of(p, r + 1);
                if (next <= s) {
                    r++;
                    from = next;
                }
            }
            const Tile t = tile_of<ST>(p, r, s - from);
            if (t.m > 0 && f(r, s - from, t.units)) return;
        }
    };
    walk([&](int, int, int units) {
        mine += units;
        return false;
    });
    int through = wave_scan(mine);
    if (lane == 63) part[tid >> 6] = through;
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int i = 0; i < NW; i++) {
        if (i < (tid >> 6)) through += part[i];
        all += part[i];
    }
    all = uniform(all);
    const Ranges ranges((uint64_t)(uint32_t)all * (uint32_t)p.HQ, p.P);
    uint64_t pos = ranges.first(me);
    int64_t left = (int64_t)(ranges.first(me + 1) - pos);
    Cut cut = {0, 0, 0, 0};
    if (left > 0) {
        int hq = (int)(pos / (uint32_t)all);
        const int at = (int)(pos - (uint64_t)hq * (uint32_t)all);
        if (at >= through - mine && at < through) {
            int before = through - mine;
            walk([&](int r, int tile, int units) {
                if (at >= before + units) {
                    before += units;
                    return false;
                }
                own[0] = r;
                own[1] = tile;
                own[2] = at - before;
                return true;
            });
        }
        __syncthreads();
        int r = uniform(own[0]), tile = uniform(own[1]), u = uniform(own[2]);
        while (true) {
            Tile t = tile_of<ST>(p, r, tile);
            t = Tile{uniform(t.first), uniform(t.m), uniform(t.pos), uniform(t.n), uniform(t.base), uniform(t.end), uniform(t.units)};
            const int64_t can = (int64_t)u + left;
            const int u1 = can < t.units ? (int)can : t.units;
            const int hk = p.QT == 1 ? hq : hq / p.QT, qt = hq - hk * p.QT;
            const bool whole = u == 0 && u1 == t.units;
            if (!whole && u == 0) cut = Cut{ranges.of(pos + t.units - 1) - me + 1, r, tile, hq};
            if (t.m > 0 && hq < p.HQ) x.piece(t, r, hk, qt, u, u1, whole ? -1 : 2 * me + (u == 0), bad);
            left -= u1 - u;
            pos += u1 - u;
            if (left <= 0) break;
            // the next tile: of the request, of the next one with new tokens, of the next head
            u = 0;
            tile++;
            int next = t.first + t.m;
            const int s1r = clamp(scalar_at(a.starts, r + 1), 0, a.T);
            if (next >= s1r) {
                if (next >= clamp(scalar_at(a.starts, a.R), 0, a.T)) {
                    hq++;
                    next = clamp(scalar_at(a.starts, 0), 0, a.T);
                    r = -1;
                }
                tile = 0;
                r++;
                if (r >= a.R || clamp(scalar_at(a.starts, r + 1), 0, a.T) <= next) r = request_of_token(a, next);
            }
            __syncthreads();  // the piece's last readers of LDS
        }
    }
    if (tid == 0 && p.cuts) p.cuts[me] = cut;
}

// The parts of the tile that range blockIdx.x started and others ended: a wave takes
// a row, a lane DP / 64 of its channels.
template <int T, int DP, int RG, int KG, int BT, int NS, bool WHOLE>
__global__ __launch_bounds__(256) void join_kernel(Params p) {
    using A = Chunk<T, DP, RG, KG, BT, NS, WHOLE>;
    constexpr int NV = DP / 64;
    const ChunkArgs& a = p.a;
    const Cut cut = p.cuts[blockIdx.x];
    if (cut.parts == 0) return;
    const int w0 = blockIdx.x, lane = threadIdx.x & 63;
    const Tile t = tile_of<A::ST>(p, cut.r, cut.tile);
    const int hk = cut.hq / p.QT, qt = cut.hq - hk * p.QT, rows = t.m * p.GT;
    for (int row = blockIdx.y * 4 + uniform(threadIdx.x >> 6); row < rows; row += gridDim.y * 4) {
        const int i = div_by(row, p.by_gt), head = qt * p.GT + row - i * p.GT;
        if (head >= a.G) continue;
        float top = -0x1p126f, sum = 0.f, acc[NV];
#pragma unroll
        for (int j = 0; j < NV; j++) acc[j] = 0.f;
        for (int s0 = 0; s0 < cut.parts; s0 += 64) {
            const int n = cut.parts - s0 < 64 ? cut.parts - s0 : 64;
            const u2 ml = lane < n ? *reinterpret_cast<const u2*>(p.part_ml + ((int64_t)slot(w0, s0 + lane) * (RG * 32) + row) * 2) : u2{0, 0};
            float tm = lane < n ? __uint_as_float(ml[0]) : -0x1p126f;
            float mx = tm;
#pragma unroll
            for (int k = 1; k < 64; k *= 2) mx = fmaxf(mx, __shfl_xor(mx, k));
            const float to = fmaxf(top, mx), f0 = __builtin_amdgcn_exp2f(top - to);
            top = to;
            // a part's weight never falls to 0: its sum may be infinite
            const float wgt = lane < n ? fmaxf(__builtin_amdgcn_exp2f(tm - to), kLeast) : 0.f;
            sum = sum * f0 + wave_sum(lane < n ? wgt * __uint_as_float(ml[1]) : 0.f);
#pragma unroll
            for (int j = 0; j < NV; j++) acc[j] *= fmaxf(f0, kLeast);
            constexpr int kB = 8;
            for (int s = 0; s < n; s += kB) {
                float v[kB][NV];
#pragma unroll
                for (int b = 0; b < kB; b++) {
                    const int at = s + b < n ? s + b : n - 1;
                    const float* src = p.part_o + ((int64_t)slot(w0, s0 + at) * (RG * 32) + row) * DP + lane;
#pragma unroll
                    for (int j = 0; j < NV; j++) v[b][j] = src[64 * j];
                }
#pragma unroll
                for (int b = 0; b < kB; b++) {
                    const float f = lane_f(wgt, s + b < n ? s + b : n - 1);
#pragma unroll
                    for (int j = 0; j < NV; j++) acc[j] = s + b < n ? fmaf(f, v[b][j], acc[j]) : acc[j];
                }
            }
        }
        const int tok = t.first + i, hd = hk * a.G + head;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int d = lane + 64 * j;
            if (d < a.D) store_f(a.out, (size_t)((int64_t)tok * a.out_row + (int64_t)hd * a.D + d), T, sum == 0.f ? 0.f : acc[j] / sum);
        }
        if (lane == 0 && a.lse) a.lse[(int64_t)tok * a.H + hd] = sum == 0.f ? -INFINITY : (top + log2f(sum * A::kDown)) * kLn2;
    }
}

template <int T, int DP, int RG, int KG, int BT, int NS, bool WHOLE>
LuxStatus launch_as(Params& p, hipStream_t st) {
    using A = Chunk<T, DP, RG, KG, BT, NS, WHOLE>;
    const ChunkArgs& a = p.a;
    constexpr int rows = RG * 32;
    p.GT = a.G < rows ? a.G : rows;
    p.QT = (a.G + p.GT - 1) / p.GT;
    p.HQ = a.Hk * p.QT;
    p.TB = rows / p.GT;
    p.by_tb = DivBy(p.TB);
    p.by_gt = DivBy(p.GT);
    p.slots = a.T / p.TB + a.R;
    p.each = (p.slots + A::NT - 1) / A::NT;
    auto main = chunk_kernel<T, DP, RG, KG, BT, NS, WHOLE>;
    auto join = join_kernel<T, DP, RG, KG, BT, NS, WHOLE>;
    static const bool attr = hipFuncSetAttribute((const void*)main, hipFuncAttributeMaxDynamicSharedMemorySize, A::kLds) == hipSuccess;
    if (!attr) return LuxStatus::Internal;
    p.P = a.cus < kChunkRanges ? a.cus : kChunkRanges;
    const size_t one = (size_t)rows * (DP + 2) * 2 * 4 + sizeof(Cut);
    if (!a.ws || (size_t)p.P * one > kChunkPartBytes) return LuxStatus::NotSupported;
    p.part_o = reinterpret_cast<float*>(a.ws);
    p.part_ml = p.part_o + (size_t)2 * p.P * rows * DP;
    p.cuts = reinterpret_cast<Cut*>(p.part_ml + (size_t)2 * p.P * rows * 2);
    hipLaunchKernelGGL(main, dim3(p.P), dim3(A::NT), A::kLds, st, p);
    hipLaunchKernelGGL(join, dim3(p.P, 8), dim3(256), 0, st, p);
    return hipGetLastError() == hipSuccess ? LuxStatus::Ok : LuxStatus::Internal;
}

template <int T>
LuxStatus launch_t(const ChunkArgs& a, hipStream_t st) {
    Params p = {};
    p.a = a;
    const float s = a.softcap > 0.f ? 2.f * kLog2e * a.scale / a.softcap : kLog2e * a.scale;
    // c above 0, so that c times a masked score is -infinity
    p.c = s < 0.f ? -s : s > 0.f ? s : 0x1p-149f;
    p.flip = s < 0.f ? (T == DT_F32 ? 0x80000000u : 0x80008000u) : 0u;
    p.cap = a.softcap * kLog2e;
    // tokens per transfer: 1024 bytes of rows
    if constexpr (T == DT_F32) {
        if (a.D <= 64) return a.page % 4 ? launch_as<T, 64, 8, 1, 32, 3, false>(p, st) : launch_as<T, 64, 8, 1, 32, 3, true>(p, st);
        if (a.D <= 128) return a.page % 2 ? launch_as<T, 128, 8, 1, 32, 3, false>(p, st) : launch_as<T, 128, 8, 1, 32, 3, true>(p, st);
        if (a.D <= 192) return launch_as<T, 192, 4, 1, 32, 2, true>(p, st);
        return launch_as<T, 256, 4, 1, 32, 2, true>(p, st);
    } else {
        if (a.D <= 64) return a.page % 8 ? launch_as<T, 64, 8, 1, 64, 3, false>(p, st) : launch_as<T, 64, 8, 1, 64, 3, true>(p, st);
        if (a.D <= 128) return a.page % 4 ? launch_as<T, 128, 8, 1, 64, 3, false>(p, st) : launch_as<T, 128, 8, 1, 64, 3, true>(p, st);
        if (a.D <= 192) return a.page % 2 ? launch_as<T, 192, 4, 1, 64, 2, false>(p, st) : launch_as<T, 192, 4, 1, 64, 2, true>(p, st);
        return a.page % 2 ? launch_as<T, 256, 4, 1, 64, 2, false>(p, st) : launch_as<T, 256, 4, 1, 64, 2, true>(p, st);
    }
}

extern template LuxStatus launch_t<DT_F32>(const ChunkArgs&, hipStream_t);
extern template LuxStatus launch_t<DT_F16>(const ChunkArgs&, hipStream_t);
extern template LuxStatus launch_t<DT_BF16>(const ChunkArgs&, hipStream_t);

}  // namespace chunk
}  // namespace lxq
