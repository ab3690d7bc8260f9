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
// launch joins (in the same one the last block of a tile would join alone what all
// waves of the card join here).  Ranges follow each other head by head, and an XCD
// takes a run of ranges, so that its L2 holds the keys that its blocks share.
//
// What bounds it, and what it measured (32 heads on 8 of 128 channels, bf16):
//   16384 tokens of one request: 2.48 ms, 890 TFLOP/s (a large product of the library
//     reaches 1110 to 1270).  The MFMAs are busy 57 % of the cycles in which a CU has
//     work, the rest of which is the softmax, and 44 % of the kernel's, at 1.8 GHz: a
//     fifth of the CUs' time is idle, as ranges are cut by stages alone and the first
//     ranges of a head hold dozens of short tiles, each with a start and an end of
//     two to three stages' time (they end 10 % behind the mean).  The loop of whole,
//     unmasked stages (kPlain, kRuns) brought 2.74 to 2.50: rows of the table looked up
//     for 64 stages at a time (222 scalar instructions per stage and wave became 36),
//     LDS reads kept three or four products ahead by fences.  Two groups of waves in
//     opposite phases, scores of the next stage before the weights of this one, 64 rows
//     per wave and 32-token stages were tried and were no faster.
//   4 chunks of up to 512 tokens among 64 requests of up to 8192: 259 us, 4.2 TB/s of
//     the cache; reading it, with 4.7 TB/s for a large copy, is what remains.
//   64 new tokens on 4096 (f16): 25.5 us, of which the transfers and products of a
//     block's four stages are 5; the start (lengths, table, queries), the meeting of
//     the four groups and the second launch are chains of trips to memory.
#pragma once
#include <type_traits>

#include "chunk_places.h"
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

// a tile that starts in a range and ends behind it: its parts, tokens and heads
struct Cut {
    int32_t parts, first, m, hq;
};

struct Params {
    ChunkArgs a;
    int GT, QT, HQ;   // heads of a tile; tiles of a group; heads of keys times those
    int TB;           // tokens of a tile
    int slots, each;  // places of tiles (some may be empty); places per thread
    DivBy by_tb, by_gt;
    int P, log;       // ranges: 2^log
    float c;          // scores by log2 e are s * c (or, capped, cap tanh(y) with 2 y log2 e = s * c)
    float cap;        // softcap log2 e
    uint32_t flip;    // sign bits of q: c is not negative
    float* part_o;    // [2 P, rows, DP]
    float* part_ml;   // [2 P, rows, 2]
    Cut* cuts;        // [P]
};

// the weight of x, which never falls to 0 before an infinite x; before a finite one it
// does: as small as it is, 2^-126 of a large x may be more than the result
__device__ __forceinline__ float weight_of(float w, float x) { return fabsf(x) == INFINITY ? fmaxf(w, 0x1p-126f) : w; }

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

// a tile, where it is, and a unit in it
struct Found {
    Tile t;
    int r, tile, at;
};
template <int ST>
__device__ __forceinline__ Tile tile_of(const Params& p, int r, int tile) {
    const ChunkArgs& a = p.a;
    const int cap = a.pool > 0 ? a.columns * a.page : 0;
    const int s0 = clamp(a.starts[r], 0, a.T), s1 = clamp(a.starts[r + 1], s0, a.T);
    return tile_at(s0, s1, clamp(a.seq[r], 0, a.columns * a.page), clamp(a.lens[r], 0, cap), tile, p.TB, a.window, ST);
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
// global -> LDS: lane l copies 16 bytes to LDS m0 + 16 l (a transfer reads m0 one
// wait state after it was written at the earliest)
__device__ __forceinline__ void dma16(uint32_t m0v, const void* sbase, uint32_t voff) {
    const uint64_t b = reinterpret_cast<uint64_t>(sbase);
    const uint64_t s = (uint64_t)(uint32_t)uniform((int)(b >> 32)) << 32 | (uint32_t)uniform((int)b);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(uniform((int)m0v)), "v"(voff), "s"(s) : "memory", "m0");
}
__device__ __forceinline__ void dma16a(uint32_t m0v, const void* addr) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(uniform((int)m0v)), "v"(addr) : "memory", "m0");
}

__device__ __forceinline__ float other_half(float v) {
    const uint32_t x = __float_as_uint(v);
    const auto q = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return __uint_as_float((threadIdx.x & 32) ? q[0] : q[1]);
}
// sums with the lane 16 beside this one
__device__ __forceinline__ float both_rows(float v) {
    const uint32_t x = __float_as_uint(v);
    const auto q = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return __uint_as_float(q[0]) + __uint_as_float(q[1]);
}
__device__ __forceinline__ float half_max(float v) {
    const uint32_t x = __float_as_uint(v);
    const auto q = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return fmaxf(__uint_as_float(q[0]), __uint_as_float(q[1]));
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

// How a wave finds its tokens' rows of the cache.  kLanes: each lane its own, with a
// load of the table per transfer.  kRuns: pages hold whole runs of the tokens that a
// wave finds with one entry of the table, so that a run has one scalar address,
// looked up for 64 stages at a time.  kPlain: as kRuns, and head_dim is DP, a power
// of two, and scores are not capped, so that the steps of most stages hold nothing
// but the products and the softmax.
enum { kLanes, kRuns, kPlain };

// T: type of q, cache and out; DP: head_dim rounded up to 64, 96, 128, 192 or 256; RG
// row groups times KG groups of tokens = waves; BT: tokens of a group's part of a
// stage; NS: stages in LDS
template <int T, int DP, int RG, int KG, int BT, int NS, int FORM>
struct Chunk {
    static constexpr int ES = T == DT_F32 ? 4 : 2, E = 16 / ES;  // bytes; elements per 16 bytes
    static constexpr bool EASY = FORM == kPlain;
    static constexpr int RS = (DP == 192 ? 256 : DP == 96 ? 128 : DP) * ES;  // LDS row of a token
    static constexpr int CPR = RS / 16, TI = 64 / CPR;           // its 16-byte chunks; tokens per transfer
    static constexpr int NW = RG * KG, NT = 64 * NW, ST = BT * KG, NI = ST / TI / NW;
    static_assert(NI * TI * NW == ST && TI <= 16, "every wave moves whole runs");
    // tokens that a wave finds with one entry of the table, and how often per stage
    static constexpr int LT = TI * NI < 8 ? TI * NI : 8, NL = TI * NI / LT;
    static constexpr int ROWS = RG * 32;
    static constexpr int kMat = ST * RS, kRings = 2 * NS * kMat;  // LDS: NS slots of keys, then of values
    static constexpr int NK = DP / (2 * E), ND = DP / 32, NB = BT / 32;
    static constexpr int KM = CPR < 16 ? 7 : 15;
    static constexpr int LS = DP + 4;  // row of the groups' meeting, in floats
    static constexpr int kMeet = KG > 1 ? NW * 32 * (LS + 2) * 4 + ROWS * (KG + 2) * 4 : 0;
    static constexpr int kLds = kRings > kMeet ? kRings : kMeet;
    // the weights are 2^kLift exp2(s - m): f16 ends at 2^-24, and many weights
    // below 2^-25 beside a large one may together be most of the result
    static constexpr float kLift = T == DT_F16 ? 14.f : 0.f, kDown = T == DT_F16 ? 0x1p-14f : 1.f;
    // In 16 bits a weight enters the second product as one value of the type, rounded
    // to the nearest: off by as much as the result's own rounding is.  As the sum of
    // two, with a second product, chunks among decoding requests take 300 us where
    // they take 256, and 64 tokens on 4096 27.0 where they take 25.3.  But a tile of at
    // most 16 rows, a request that decodes beside prompts, is as exact as by itself
    // in the decoding step, without a second product: its rows stand in both halves
    // of the 32 columns, and the second half's weights are what the first half's leave
    // out (twin(), leave(); 64 such requests of up to 8192 tokens 195 us where they took 193).
    // m may stay behind the maximum by this much (log2): O is rescaled less often,
    // and weights stay below 2^16 in f16
    static constexpr float kBehind = T == DT_F16 ? 1.f : 8.f;

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
    int found[NL], row_at[NL];  // see find()

    __device__ __forceinline__ explicit Chunk(char* mem) : lds(mem) {
        lane = threadIdx.x & 63;
        w = uniform(threadIdx.x >> 6);
        rg = w % RG;
        kg = w / RG;
        const int ri = lane / CPR, c = lane % CPR;
        koff = (uint32_t)((c ^ k_turn(ri)) * 16);
        voff = (uint32_t)((c ^ v_turn(ri)) * 16);
    }

    // The cache rows where the wave's parts of stages s0 + lane begin, tokens behind
    // the tile's last one taken as its run: 64 stages with one trip to the table
    __device__ __forceinline__ void find(const ChunkArgs& a, const Tile& t, int r, int hk, uint32_t first_tok, int s0) {
#pragma unroll
        for (int i = 0; i < NL; i++) {
            const int tr = or_last_run(t, first_tok + (uint32_t)(s0 + lane) * ST + (uint32_t)(w * NI * TI + i * LT), LT);
            const int col = div_by(tr, a.div);
            int pg = a.table[(int64_t)r * a.columns + col];
            pg = (uint32_t)pg < (uint32_t)a.pool ? pg : 0;
            found[i] = (pg * a.Hk + hk) * a.page + (tr - col * a.page);
        }
    }
    // what the compiler knows to be in flight ends here, not at its first use in a loop
    __device__ __forceinline__ static void settle() { __builtin_amdgcn_s_waitcnt((0x7 << 4) | (0xF << 8)); }
    __device__ __forceinline__ uint32_t lds_at() const { return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds + (uint32_t)(w * NI * 1024); }
    // A stage's rows of keys (V: of values) into the slot at `slot` of their ring:
    // tokens from tb on, those past the tile's last one from its row
    template <bool V>
    __device__ __forceinline__ void fill(const ChunkArgs& a, const Tile& t, int r, int hk, uint32_t tb, uint32_t slot) {
        const uint32_t dst = lds_at() + (V ? NS * kMat : 0) + slot;
        const uint32_t row_bytes = (uint32_t)(a.D * ES);
        const char* cache = static_cast<const char*>(V ? a.vc : a.kc);
        const int ri = lane / CPR;
#pragma unroll
        for (int j = 0; j < NI; j++) {
            const int run = w * NI + j, in = j * TI % LT;  // the run's first token, from where the entry was found
            const uint32_t c = V ? voff ^ (uint32_t)(v_turn(run * TI) * 16) : koff ^ (uint32_t)(k_turn(run * TI) * 16);
            if constexpr (FORM != kLanes) {
                const int i = j * TI / LT;
                const char* from = cache + (uint64_t)(uint32_t)row_at[i] * row_bytes;
                uint32_t at = c + (uint32_t)(ri + in) * row_bytes;
                if (!is_whole(t, tb, ST)) {
                    const int last = t.end - 1 - or_last_run(t, tb + (uint32_t)(w * NI * TI + i * LT), LT);
                    at = c + (uint32_t)(ri + in < last ? ri + in : last) * row_bytes;
                }
                if (EASY || c < row_bytes) dma16(dst + j * 1024, from, at);
            } else {
                const int tok = or_last(t, tb + (uint32_t)(run * TI + ri));
                const int col = div_by(tok, a.div);
                int pg = a.table[(int64_t)r * a.columns + col];
                pg = (uint32_t)pg < (uint32_t)a.pool ? pg : 0;
                const uint64_t row = (uint64_t)(uint32_t)((pg * a.Hk + hk) * a.page + (tok - col * a.page));
                if (c < row_bytes) dma16a(dst + j * 1024, cache + row * row_bytes + c);
            }
        }
    }
    // the same of a stage that is all there
    template <bool V>
    __device__ __forceinline__ void fill_whole(const ChunkArgs& a, uint32_t slot) const {
        const uint32_t dst = lds_at() + (V ? NS * kMat : 0) + slot;
        const uint32_t row_bytes = (uint32_t)((EASY ? DP : a.D) * ES);
#pragma unroll
        for (int j = 0; j < NI; j++) {
            const uint32_t c = V ? voff ^ (uint32_t)(v_turn((w * NI + j) * TI) * 16) : koff ^ (uint32_t)(k_turn((w * NI + j) * TI) * 16);
            const int i = j * TI / LT;
            const char* from = static_cast<const char*>(V ? a.vc : a.kc) + (uint64_t)(uint32_t)row_at[i] * row_bytes;
            const uint32_t at = c + (uint32_t)(lane / CPR + j * TI % LT) * row_bytes;
            if (EASY || c < row_bytes) dma16(dst + j * 1024, from, at);
        }
    }
    // the rows of stage s
    __device__ __forceinline__ void next_rows(const ChunkArgs& a, const Tile& t, int r, int hk, uint32_t first_tok, int s) {
        if constexpr (FORM != kLanes) {
            if ((s & 63) == 0 && s > 0) {
                find(a, t, r, hk, first_tok, s);
                settle();
            }
#pragma unroll
            for (int i = 0; i < NL; i++) row_at[i] = __builtin_amdgcn_readlane(found[i], s & 63);
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

    __device__ __forceinline__ void load_q(const Params& p, const Tile& t, int hk, int qt) {
        const ChunkArgs& a = p.a;
        int head;
        const int i = token_of(p, t, rg * 32 + (lane & (twin(p, t) ? 15 : 31)), qt, head);
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
        seen_by(t, i, a.window, from, to);
        lo = from;
        len = to > from ? to - from : 0;
    }

    // which of the 32 NB tokens from tb on have a page
    __device__ __forceinline__ uint64_t pages_there(const ChunkArgs& a, const Tile& t, int r, uint32_t tb) const {
        const uint32_t tok = tb + (uint32_t)lane;
        const bool in = lane < BT && tok < (uint32_t)t.end;
        const int pg = in ? a.table[(int64_t)r * a.columns + div_by((int)tok, a.div)] : -1;
        return __ballot((uint32_t)pg < (uint32_t)a.pool);
    }

    struct Scores {
        f16v s[NB];
    };
    struct Weights {
        u4 w[T == DT_F32 ? 1 : 2 * NB];
    };

    // Operands of the products that are on their way from LDS: those of AK steps of
    // the first product (a step: 16 bytes of each key row) and AV of the second
    // (a step: 16 tokens, 32 channels; f32: 2 tokens).  The steps are fenced: left to
    // itself the compiler reads each operand right before its product and waits
    static constexpr int AK = T == DT_F32 && DP >= 128 ? 1 : DP == 256 ? 2 : 3, AV = 4;
    static constexpr int NVS = T == DT_F32 ? 16 * NB * ND : 2 * NB * ND;  // steps of the second product
    struct Ahead {
        u4 k[AK][NB];
        u4 v[AV];
    };
    // offsets into the rings of the lane's part of a step
    __device__ __forceinline__ uint32_t key_at(uint32_t slot) const {
        return slot + (uint32_t)((kg * BT + (lane & 31)) * RS) + (uint32_t)(((lane >> 5) ^ k_turn(lane & 31)) * 16);
    }
    __device__ __forceinline__ uint32_t value_at(uint32_t slot) const {
        const int h = lane >> 5, row = NS * ST + kg * BT + 4 * h;
        if constexpr (T == DT_F32) {
            return slot + (uint32_t)(row * RS) + (uint32_t)((((lane & 31) >> 2) ^ v_turn(4 * h)) * 16 + (lane & 3) * 4);
        } else {
            const int i4 = (lane & 15) >> 2;
            return slot + (uint32_t)((row + i4) * RS) + (uint32_t)(((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ v_turn(4 * h + i4)) * 16 + (lane & 1) * 8);
        }
    }
    __device__ __forceinline__ void read_k(u4* x, uint32_t at, int k) const {
#pragma unroll
        for (int b = 0; b < NB; b++)
            x[b] = *reinterpret_cast<const __attribute__((address_space(3))) u4*>((lds_ptr)lds + (at ^ (uint32_t)(k * 32)) + b * 32 * RS);
    }
    __device__ __forceinline__ u4 read_v(uint32_t at, int s) const {
        const int d = s % ND;
        if constexpr (T == DT_F32) {
            const int i = s / ND;  // token pair of all blocks
            return u4{*reinterpret_cast<const __attribute__((address_space(3))) uint32_t*>(
                          (lds_ptr)lds + (at ^ (uint32_t)(d * 128)) + (32 * (i / 16) + (i & 3) + 8 * (i % 16 >> 2)) * RS), 0, 0, 0};
        } else {
            typedef __attribute__((address_space(3))) s4* tr_ptr;
            const lds_ptr from = (lds_ptr)lds + (at ^ (uint32_t)(d * 64)) + 16 * (s / ND) * RS;
            const u2 x = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)from));
            const u2 y = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)(from + 8 * RS)));
            return u4{x[0], x[1], y[0], y[1]};
        }
    }
    __device__ __forceinline__ static void clear(Scores& x) {
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int i = 0; i < 16; i++) x.s[b][i] = 0.f;
    }
    // the first steps' keys, to be read before other work
    __device__ __forceinline__ void begin(Ahead& f, uint32_t at) const {
#pragma unroll
        for (int k = 0; k < AK; k++) read_k(f.k[k], at, k);
        __builtin_amdgcn_sched_barrier(0);
    }
    __device__ __forceinline__ void score(Scores& x, Ahead& f, uint32_t at, int k) const {
#pragma unroll
        for (int b = 0; b < NB; b++) x.s[b] = mfma<T>(f.k[k % AK][b], q[k], x.s[b]);
        if (k + AK < NK) read_k(f.k[k % AK], at, k + AK);
    }
    __device__ __forceinline__ void scores(Scores& x, Ahead& f, uint32_t at, int dim) const {
        clear(x);
#pragma unroll
        for (int k = 0; k < NK; k++) {
            if (!EASY && k > 0 && 2 * k * E >= dim) break;  // nothing but padding from here on
            score(x, f, at, k);
            __builtin_amdgcn_sched_barrier(0);
        }
    }

    // the cap, and -infinity for tokens that the row does not see: those of a group's
    // part of a stage, from position tb on
    __device__ __forceinline__ void mask(const ChunkArgs& a, Scores& x, const Tile& t, int r, uint32_t tb, bool holes) const {
        const int h = lane >> 5;
        const uint32_t from = (uint32_t)lo - tb - (uint32_t)(4 * h);  // against the token's number without the lane's 4 h
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
                x.s[b][i] = (uint32_t)(32 * b + (i & 3) + 8 * (i >> 2)) - from < (uint32_t)len ? x.s[b][i] : -INFINITY;
                if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);
            }
        if (holes) {
            const uint64_t there = pages_there(a, t, r, tb) >> (4 * h);
            const uint32_t bits[2] = {(uint32_t)there, (uint32_t)(there >> 32)};
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    x.s[b][i] = (bits[b] >> ((i & 3) + 8 * (i >> 2))) & 1 ? x.s[b][i] : -INFINITY;
                    if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);
                }
        }
    }
    __device__ __forceinline__ static void limit(const Params& p, Scores& x) {
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int i = 0; i < 16; i++) x.s[b][i] = p.cap * tanh_of(x.s[b][i] * p.c);
    }

    // the running maximum, and o and l by it
    __device__ __forceinline__ void follow(const Scores& x, float c) {
        float mx = kLowest;
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int i = 0; i < 16; i++) mx = fmaxf(mx, x.s[b][i]);
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
    }

    // the weights of x (exp2 of the distance to m, lifted), packed in w where the type
    // has 16 bits
    __device__ __forceinline__ void weigh(Scores& x, float c, Weights& w) {
        // below every product of a maximum: a masked score's weight is 0 then, and
        // so is that of a row with no score yet
        const float from = fmaxf(m * c, -0x1p126f) - kLift;
#pragma unroll
        for (int e = 0; e < NB * 16; e += 2) {
            const int b = e / 16, i = e % 16;
            x.s[b][i] = __builtin_amdgcn_exp2f(fmaf(x.s[b][i], c, -from));
            x.s[b][i + 1] = __builtin_amdgcn_exp2f(fmaf(x.s[b][i + 1], c, -from));
            l += x.s[b][i] + x.s[b][i + 1];
            if constexpr (T != DT_F32) w.w[e / 8][e % 8 / 2] = pack2<T>(x.s[b][i], x.s[b][i + 1]);
        }
    }
    // a tile whose rows stand in the columns twice
    __device__ __forceinline__ static bool twin(const Params& p, const Tile& t) { return T != DT_F32 && t.m * p.GT <= 16; }
    // its packed weights: in the second half of the columns what the type's values leave
    // of x, which is off by 2^-16 (f16: 2^-22) of x at most
    __device__ __forceinline__ void leave(const Scores& x, Weights& w) const {
        if constexpr (T != DT_F32) {
#pragma unroll
            for (int e = 0; e < NB * 16; e += 2) {
                const uint32_t h = (uint32_t)afresh((int)w.w[e / 8][e % 8 / 2]);
                const float hx = T == DT_F16 ? f16_to_f32(h & 0xffffu) : __uint_as_float(h << 16);
                const float hy = T == DT_F16 ? f16_to_f32(h >> 16) : __uint_as_float(h & 0xffff0000u);
                const uint32_t left = pack2<T>(x.s[e / 16][e % 16] - hx, x.s[e / 16][e % 16 + 1] - hy);
                w.w[e / 8][e % 8 / 2] = lane & 16 ? left : h;
                if (e % 4 == 2) __builtin_amdgcn_sched_barrier(0);
            }
        }
    }

    // o += V^T . weights, of the values at `at`
    __device__ __forceinline__ void begin_values(Ahead& f, uint32_t at) const {
#pragma unroll
        for (int s = 0; s < AV; s++) f.v[s] = read_v(at, s);
        __builtin_amdgcn_sched_barrier(0);
    }
    __device__ __forceinline__ void gather(const Scores& x, const Weights& w, Ahead& f, uint32_t at) {
#pragma unroll
        for (int s = 0; s < NVS; s++) {
            const int d = s % ND, i = s / ND;
            if constexpr (T == DT_F32)
                o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(f.v[s % AV][0]), x.s[i / 16][i % 16], o[d], 0, 0, 0);
            else o[d] = mfma<T>(f.v[s % AV], w.w[i], o[d]);
            if (s + AV < NVS) f.v[s % AV] = read_v(at, s + AV);
            __builtin_amdgcn_sched_barrier(0);
        }
    }

    // the maximum by log2 e that goes with l and o
    __device__ __forceinline__ static float top_of(const Params& p, float mm) { return fmaxf(mm * (p.a.softcap > 0.f ? 1.f : p.c), -0x1p126f); }

    // four channels of a row of the tile: into out, or a partial result
    __device__ __forceinline__ static void store4(const Params& p, const Tile& t, int hk, int qt, int to, int row, int d, f4 acc, float top, float sum) {
        if (to >= 0) {
            const int64_t at = (int64_t)to * ROWS + row;
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
    // its own tokens alone.
    __device__ __forceinline__ static void alone(const Params& p, int first, int pos, int n, int r, int hk, int head, int i, int from, int to,
                                              float* part_o, float* part_ml) {
        const ChunkArgs& a = p.a;
        constexpr int NV = (DP + 63) / 64;
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
            const float f = __builtin_amdgcn_exp2f((was - m) * c);
            const float w = __builtin_amdgcn_exp2f(fmaf(s, c, -fmaxf(m * c, -0x1p126f)));
            l = fmaf(l, f, w);
#pragma unroll
            for (int j = 0; j < NV; j++) acc[j] = fmaf(weight_of(w, v[j]), v[j], acc[j] * weight_of(f, acc[j]));
        }
        const float up = 1.f / kDown, top = fmaxf(m * c, -0x1p126f);
        const int tok = first + i, hd = hk * a.G + head;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int d = lane + 64 * j;
            if (part_o) {
                if (d < DP) part_o[d] = acc[j] * up;
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
        for (int i = threadIdx.x * 16; i < kRings; i += NT * 16) *reinterpret_cast<u4*>(lds + i) = u4{0, 0, 0, 0};
    }

    // stages u0 .. u1 - 1 of a tile; to: the slot of a partial result, or -1
    __device__ __forceinline__ void piece(const Tile& t, int r, int hk, int qt, int u0, int u1, int to, uint32_t* bad) {
        const Params& p = argument();
        const ChunkArgs& a = p.a;
        const uint32_t first_tok = stage_at(t, u0, ST), last_tok = stages_end(t, u1, ST);
        const bool any = last_tok > first_tok;
        // the table's entries, for the places of the stages and for pages that are none,
        // and the queries in one trip
        bool none = false;
        if (any) {
            const int c0 = div_by((int)first_tok, a.div), c1 = div_by((int)last_tok - 1, a.div);
            for (int c = c0 + (int)threadIdx.x; c <= c1; c += NT)
                none |= (uint32_t)a.table[(int64_t)r * a.columns + c] >= (uint32_t)a.pool;
            if constexpr (FORM != kLanes) find(a, t, r, hk, first_tok, 0);
        }
        load_q(p, t, hk, qt);
        if (threadIdx.x < RG) bad[threadIdx.x] = 0;
        settle();
        // step j takes stage j, which has arrived then, and fills stage j + L where stage
        // j - 1 was
        constexpr int L = NS - 1;
        const int nu = any ? u1 - u0 : 0;
        auto fill_both = [&](int s, uint32_t slot) {
            next_rows(a, t, r, hk, first_tok, s);
            fill<false>(a, t, r, hk, first_tok + (uint32_t)s * ST, slot);
            fill<true>(a, t, r, hk, first_tok + (uint32_t)s * ST, slot);
        };
#pragma unroll
        for (int s = 0; s < L; s++)
            if (s < nu) fill_both(s, s * kMat);
        const bool holes = __syncthreads_or(none);
        // the wave's rows: the first one's tokens and the last one's
        int head, lo0, hi0, lo1, hi1;
        seen_by(t, token_of(p, t, rg * 32, qt, head), a.window, lo0, hi0);
        seen_by(t, token_of(p, t, rg * 32 + 31, qt, head), a.window, lo1, hi1);
        const bool rows = rg * 32 < t.m * p.GT, halves = twin(p, t);
        m = kLowest;
        l = 0.f;
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[d][i] = 0.f;
        if (any) {
            const float c = !EASY && a.softcap > 0.f ? 1.f : p.c;
            Scores x;
            Weights wt;
            uint32_t here = 0, behind = L * kMat;  // slots of stages j and j - 1
            auto turn = [&] {
                behind = here;
                here = here == (NS - 1) * kMat ? 0 : here + kMat;
            };
            constexpr int kOut = 2 * (L - 1) * NI;  // transfers behind the stage's
            auto step = [&](int j) {
                if (FORM != kLanes && j + L <= nu) wait_vm<kOut>();
                else wait_vm<0>();
                barrier();
                if (j + L < nu) fill_both(j + L, behind);
                const uint32_t tb = first_tok + (uint32_t)j * ST + (uint32_t)(kg * BT);
                if (rows && is_seen(tb, BT, lo0, hi1)) {
                    Ahead f;
                    const uint32_t kat = key_at(here), vat = value_at(here);
                    begin(f, kat);
                    scores(x, f, kat, a.D);
                    if (!EASY && a.softcap > 0.f) limit(p, x);
                    if (holes || !is_inside(tb, BT, lo1, hi0)) mask(a, x, t, r, tb, holes);
                    follow(x, c);
                    begin_values(f, vat);
                    weigh(x, c, wt);
                    if (halves) leave(x, wt);
                    gather(x, wt, f, vat);
                }
                turn();
            };
            // steps in which the wave's rows see all of a stage and whole stages are filled; in
            // the wide tiles they are kept free of what one in many needs
            int ja = 0, jb = 0;
            if (FORM != kLanes && rows && !holes && !(KG == 1 && halves)) {
                steps_inside(first_tok + (uint32_t)(kg * BT), BT, ST, lo1, hi0, ja, jb);
                jb = jb < nu - 1 - L ? jb : nu - 1 - L;
            }
            for (int j = 0; j < nu; j++) {
                for (; FORM != kLanes && j >= ja && j < jb; j++) {
                    Ahead f;
                    wait_vm<kOut>();
                    barrier();
                    const uint32_t kat = key_at(here), vat = value_at(here);
                    begin(f, kat);
                    next_rows(a, t, r, hk, first_tok, j + L);
                    fill_whole<false>(a, behind);
                    fill_whole<true>(a, behind);
                    scores(x, f, kat, a.D);
                    if (!EASY && a.softcap > 0.f) limit(p, x);
                    follow(x, c);
                    begin_values(f, vat);
                    weigh(x, c, wt);
                    if (KG > 1 && halves) leave(x, wt);
                    gather(x, wt, f, vat);
                    turn();
                }
                step(j);
            }
        }
        l += other_half(l);
        if (halves) {
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int i = 0; i < 16; i++) o[d][i] = both_rows(o[d][i]);
        }
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
            // a row's groups' weights, its maximum and sum
            float* weight = ml + NW * 32 * 2;  // [ROWS][KG + 2]
            for (int row = threadIdx.x; row < ROWS; row += NT) {
                float top = -0x1p126f, sum = 0.f;
#pragma unroll
                for (int g = 0; g < KG; g++) top = fmaxf(top, ml[(g * ROWS + row) * 2]);
                float* mine_w = weight + row * (KG + 2);
#pragma unroll
                for (int g = 0; g < KG; g++) {
                    mine_w[g] = __builtin_amdgcn_exp2f(ml[(g * ROWS + row) * 2] - top);
                    sum += ml[(g * ROWS + row) * 2 + 1] * mine_w[g];
                }
                mine_w[KG] = top;
                mine_w[KG + 1] = sum;
            }
            __syncthreads();
            constexpr int per = DP / 4, kTurns = ROWS * per / NT;
            static_assert(kTurns * NT == ROWS * per, "whole turns");
#pragma unroll
            for (int k = 0; k < kTurns; k++) {
                const int x = (int)threadIdx.x + k * NT, row = x / per, d = (x - row * per) * 4;
                const float* its = weight + row * (KG + 2);
                f4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int g = 0; g < KG; g++) acc += *reinterpret_cast<const f4*>(sums + (g * ROWS + row) * LS + d) * its[g];
                if (has_row(e, t, row, qt) && !((bad[row >> 5] >> (row & 31)) & 1)) store4(e, t, hk, qt, to, row, d, acc, its[KG], its[KG + 1]);
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
                const int64_t at = (int64_t)to * ROWS + row;
                alone(e, t.first, t.pos, t.n, r, hk, hd, i, (int)first_tok, (int)last_tok, to >= 0 ? e.part_o + at * DP : nullptr, e.part_ml + at * 2);
            }
        }
    }
};

extern __shared__ __attribute__((aligned(16))) char chunk_lds[];

template <int T, int DP, int RG, int KG, int BT, int NS, int FORM>
__global__ __launch_bounds__(64 * RG * KG, RG * KG / 4) void chunk_kernel(Params p) {
    using A = Chunk<T, DP, RG, KG, BT, NS, FORM>;
    constexpr int NW = A::NW, ST = A::ST;
    __shared__ int part[NW];
    __shared__ Found own;
    __shared__ uint32_t bad[RG];
    const ChunkArgs& a = p.a;
    const int tid = threadIdx.x, lane = tid & 63;
    A x(chunk_lds);
    if (a.D < A::RS / A::ES) x.clear();  // chunks that no transfer fills
    // stages of the thread's places, and of all of them for one head
    const int s0 = tid * p.each, s1 = s0 + p.each < p.slots ? s0 + p.each : p.slots;
    int mine = 0;
    Tile t = {0, 0, 0, 0, 0, 0, 0};
    int r = 0, tile = 0;
    // goes through the thread's places until f() is true of one
    auto walk = [&](auto f) {
        if (s0 >= s1) return;
        r = request_of_place(p, s0);
        int from = place_of(p, r);
        for (int s = s0; s < s1; s++) {
            if (r + 1 < a.R) {
                const int next = place_of(p, r + 1);
                if (next <= s) {
                    r++;
                    from = next;
                }
            }
            tile = s - from;
            t = tile_of<ST>(p, r, tile);
            if (t.m > 0 && f()) return;
        }
    };
    walk([&] {
        mine += t.units;
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
    const Ranges ranges((uint64_t)(uint32_t)(all > 0 ? all : 1) * (uint32_t)p.HQ, p.log);
    // an XCD takes every eighth block: a run of ranges
    const int per = 1 << ranges.log >> 3, b = (int)blockIdx.x;
    const int me = per == 0 ? b : (b >> 3) < per ? (b & 7) * per + (b >> 3) : b;
    Cut out = {0, 0, 0, 0};
    if (all > 0 && me < 1 << ranges.log) {
        const uint64_t lo = ranges.first(me), hi = ranges.first(me + 1);
        int hq = (int)((double)lo / (double)(uint32_t)all);
        if ((uint64_t)hq * (uint32_t)all > lo) hq--;
        if ((uint64_t)(hq + 1) * (uint32_t)all <= lo) hq++;
        const int at = (int)(lo - (uint64_t)hq * (uint32_t)all);
        if (at >= through - mine && at < through) {
            int before = through - mine;
            if (p.each > 1)  // else the thread's one place is still at hand
                walk([&] {
                    if (at < before + t.units) return true;
                    before += t.units;
                    return false;
                });
            own = Found{t, r, tile, at - before};
        }
        __syncthreads();
        auto share = [](const Tile& x) {
            return Tile{uniform(x.first), uniform(x.m), uniform(x.pos), uniform(x.n), uniform(x.base), uniform(x.end), uniform(x.units)};
        };
        t = share(own.t);
        r = uniform(own.r);
        tile = uniform(own.tile);
        uint64_t start = lo - (uint32_t)uniform(own.at);  // of the tile
        int u = ranges.cut(uniform(own.at), t.units);
        while (true) {
            const int u1 = hi >= start + t.units ? t.units : ranges.cut((int)(hi - start), t.units);
            const int hk = p.QT == 1 ? hq : hq / p.QT, qt = hq - hk * p.QT;
            if (u < u1 && t.m > 0 && hq < p.HQ) {
                const bool whole = u == 0 && u1 == t.units;
                if (!whole && u == 0) {
                    const int last = ranges.of(start + t.units - 1);
                    out = Cut{last - (ranges.cut((int)(ranges.first(last) - start), t.units) == t.units) - me + 1, t.first, t.m, hq};
                }
                x.piece(t, r, hk, qt, u, u1, whole ? -1 : 2 * me + (u == 0), bad);
            }
            if (hi <= start + t.units) break;
            // the next tile: of the request, of the next one with new tokens, of the next head
            start += t.units;
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
            t = share(tile_of<ST>(p, r, tile));
            __syncthreads();  // the piece's last readers of LDS
        }
    }
    if (tid == 0) p.cuts[me] = out;
}

// The parts of the tiles that were cut: a wave takes a row, a lane DP / 64 of its
// channels, rounded up (those past DP are another row's and are not stored).  The rows of all cut tiles are dealt out to all waves.
template <int T, int DP, int RG, int KG, int BT, int NS, int FORM>
__global__ __launch_bounds__(512) void join_kernel(Params p) {
    using A = Chunk<T, DP, RG, KG, BT, NS, FORM>;
    constexpr int NV = (DP + 63) / 64;
    const ChunkArgs& a = p.a;
    __shared__ Cut cuts[kChunkRanges];
    __shared__ int through[kChunkRanges], part[8];
    const int tid = threadIdx.x, lane = tid & 63, w = uniform(tid >> 6);
    static_assert(kChunkRanges <= 512, "a thread per range");
    int rows = 0;
    if (tid < p.P) {
        const Cut c = p.cuts[tid];
        cuts[tid] = c;
        rows = c.parts > 0 ? c.m * p.GT : 0;
    }
    int sum_rows = wave_scan(rows);
    if (lane == 63) part[w] = sum_rows;
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        if (i < w) sum_rows += part[i];
        all += part[i];
    }
    if (tid < p.P) through[tid] = sum_rows;
    __syncthreads();
    for (int g = (int)blockIdx.x * 8 + w; g < all; g += (int)gridDim.x * 8) {
        int w0 = 0, end = p.P - 1;  // the first range with more rows through it than g
        while (w0 < end) {
            const int mid = (w0 + end) >> 1;
            if (through[mid] > g) end = mid;
            else w0 = mid + 1;
        }
        w0 = uniform(w0);
        const Cut cut = Cut{uniform(cuts[w0].parts), uniform(cuts[w0].first), uniform(cuts[w0].m), uniform(cuts[w0].hq)};
        const int row = g - uniform(through[w0]) + cut.m * p.GT, hk = cut.hq / p.QT, qt = cut.hq - hk * p.QT;
        const int i = div_by(row, p.by_gt), head = qt * p.GT + row - i * p.GT;
        if (head >= a.G) continue;
        float top = -0x1p126f, sum = 0.f, acc[NV];
#pragma unroll
        for (int j = 0; j < NV; j++) acc[j] = 0.f;
        for (int s0 = 0; s0 < cut.parts; s0 += 64) {
            const int n = cut.parts - s0 < 64 ? cut.parts - s0 : 64;
            constexpr int kB = 8;
            float v[kB][NV];  // n is the wave's: as many loads as parts
            auto load = [&](int s) {
#pragma unroll
                for (int b = 0; b < kB; b++) {
                    if (s + b >= n) break;
                    const float* src = p.part_o + ((int64_t)slot(w0, s0 + s + b) * A::ROWS + row) * DP + lane;
#pragma unroll
                    for (int j = 0; j < NV; j++) v[b][j] = src[64 * j];
                }
            };
            const u2 ml = lane < n ? *reinterpret_cast<const u2*>(p.part_ml + ((int64_t)slot(w0, s0 + lane) * A::ROWS + row) * 2) : u2{0, 0};
            load(0);
            const float tm = lane < n ? __uint_as_float(ml[0]) : -0x1p126f;
            float mx = tm;
#pragma unroll
            for (int k = 1; k < 64; k *= 2) mx = fmaxf(mx, __shfl_xor(mx, k));
            const float to = fmaxf(top, mx), f0 = __builtin_amdgcn_exp2f(top - to);
            top = to;
            const float wgt = lane < n ? __builtin_amdgcn_exp2f(tm - to) : 0.f;
            sum = sum * f0 + wave_sum(lane < n ? wgt * __uint_as_float(ml[1]) : 0.f);
#pragma unroll
            for (int j = 0; j < NV; j++) acc[j] *= weight_of(f0, acc[j]);
            for (int s = 0; s < n; s += kB) {
                if (s > 0) load(s);
#pragma unroll
                for (int b = 0; b < kB; b++) {
                    if (s + b >= n) break;
                    const float f = lane_f(wgt, s + b);
#pragma unroll
                    for (int j = 0; j < NV; j++) acc[j] = fmaf(weight_of(f, v[b][j]), v[b][j], acc[j]);
                }
            }
        }
        const int tok = cut.first + i, hd = hk * a.G + head;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int d = lane + 64 * j;
            if (d < a.D) store_f(a.out, (size_t)((int64_t)tok * a.out_row + (int64_t)hd * a.D + d), T, sum == 0.f ? 0.f : acc[j] / sum);
        }
        if (lane == 0 && a.lse) a.lse[(int64_t)tok * a.H + hd] = sum == 0.f ? -INFINITY : (top + log2f(sum * A::kDown)) * kLn2;
    }
}

template <int T, int DP, int RG, int KG, int BT, int NS, int FORM>
LuxStatus launch_as(Params& p, hipStream_t st) {
    using A = Chunk<T, DP, RG, KG, BT, NS, FORM>;
    const ChunkArgs& a = p.a;
    constexpr int rows = A::ROWS;
    p.GT = a.G < rows ? a.G : rows;
    p.QT = (a.G + p.GT - 1) / p.GT;
    p.HQ = a.Hk * p.QT;
    p.TB = rows / p.GT;
    p.by_tb = DivBy(p.TB);
    p.by_gt = DivBy(p.GT);
    p.slots = a.T / p.TB + a.R;
    p.each = (p.slots + A::NT - 1) / A::NT;
    auto main = chunk_kernel<T, DP, RG, KG, BT, NS, FORM>;
    auto join = join_kernel<T, DP, RG, KG, BT, NS, FORM>;
    static const bool attr = hipFuncSetAttribute((const void*)main, hipFuncAttributeMaxDynamicSharedMemorySize, A::kLds) == hipSuccess;
    if (!attr) return LuxStatus::Internal;
    // a block per CU, and as many as a power of two has
    p.log = 0;
    while ((2 << p.log) <= (a.cus < kChunkRanges ? a.cus : kChunkRanges)) p.log++;
    p.P = 1 << p.log;
    const size_t one = (size_t)rows * (DP + 2) * 2 * 4 + sizeof(Cut);
    if (!a.ws || (size_t)p.P * one > kChunkPartBytes) return LuxStatus::NotSupported;
    p.part_o = reinterpret_cast<float*>(a.ws);
    p.part_ml = p.part_o + (size_t)2 * p.P * rows * DP;
    p.cuts = reinterpret_cast<Cut*>(p.part_ml + (size_t)2 * p.P * rows * 2);
    hipLaunchKernelGGL(main, dim3(p.P), dim3(A::NT), A::kLds, st, p);
    hipLaunchKernelGGL(join, dim3(4 * p.P), dim3(512), 0, st, p);
    return hipGetLastError() == hipSuccess ? LuxStatus::Ok : LuxStatus::Internal;
}

template <int T, int DP, int RG, int KG, int BT, int NS>
LuxStatus launch_page(Params& p, hipStream_t st) {
    using A = Chunk<T, DP, RG, KG, BT, NS, kRuns>;
    if (p.a.page % A::LT != 0) return launch_as<T, DP, RG, KG, BT, NS, kLanes>(p, st);
    if constexpr (A::RS == DP * A::ES)
        if (p.a.D == DP && p.a.softcap == 0.f) return launch_as<T, DP, RG, KG, BT, NS, kPlain>(p, st);
    return launch_as<T, DP, RG, KG, BT, NS, kRuns>(p, st);
}

template <int T>
LuxStatus launch_t(const ChunkArgs& a, hipStream_t st) {
    Params p = {};
    p.a = a;
    const float s = a.softcap > 0.f ? 2.f * kLog2e * a.scale / a.softcap : kLog2e * a.scale;
    // c above 0, so that c times a masked score is -infinity, and finite, so that c times a score of 0 is 0
    p.c = fminf(s < 0.f ? -s : s > 0.f ? s : 0x1p-149f, -kLowest);
    p.flip = s < 0.f ? (T == DT_F32 ? 0x80000000u : 0x80008000u) : 0u;
    p.cap = a.softcap * kLog2e;
    // Tiles of 64 rows (f32 of 128 channels: 128), whose stages are shared out among
    // four (two) groups of waves, where there are few rows: a wave of a wide tile waits
    // longer for its few stages than the narrow tiles' further reads of K and V cost.
    // 32 heads on 8, bf16, one request's new tokens on 4096 held: 64 tokens 25.8 us
    // against 32.5, 256 tokens 54.6 against 56.9, but 512 tokens 86.8 against 80.0 and
    // 4096 tokens 628 against 509.
    const bool few = (int64_t)a.T * a.H < 48 * (int64_t)a.cus;
    // Tiles of 128 rows and two groups, where the requests' rows fill less than three
    // quarters of a wide tile on average, whose waves have only padding then: 4 chunks
    // of up to 512 among 64 requests 260 us, against 313 with wide tiles and 288 with
    // narrow ones; 16384 tokens of one request 3.1 ms against 2.5.
    const bool padded = (int64_t)a.T * a.G < 192 * (int64_t)a.R;
    // 192 channels: eight waves and stages of 32 tokens (8192 tokens on 2048, bf16: 945 to
    // 980 TFLOP/s; four waves and stages of 64 tokens 636, as one wave per SIMD leaves the
    // matrix cores idle in its softmax).  256 channels do not leave the registers for
    // a second wave: 805 to 860, MFMAs busy 40 % of a working CU's cycles.  Both widths'
    // few and padded calls take tiles of 64 rows, two groups of waves.
    if constexpr (T == DT_F32) {
        if (a.D <= 64) return few || padded ? launch_page<T, 64, 2, 4, 32, 2>(p, st) : launch_page<T, 64, 8, 1, 32, 3>(p, st);
        if (a.D <= 96) return few || padded ? launch_page<T, 96, 4, 2, 32, 2>(p, st) : launch_page<T, 96, 8, 1, 32, 3>(p, st);
        if (a.D <= 128) return few || padded ? launch_page<T, 128, 4, 2, 32, 2>(p, st) : launch_page<T, 128, 8, 1, 32, 3>(p, st);
        return a.D <= 192 ? launch_page<T, 192, 4, 1, 32, 2>(p, st) : launch_page<T, 256, 4, 1, 32, 2>(p, st);
    } else if (a.D <= 64) {
        if (few) return launch_page<T, 64, 2, 4, 32, 2>(p, st);
        return padded ? launch_page<T, 64, 4, 2, 64, 2>(p, st) : launch_page<T, 64, 8, 1, 64, 3>(p, st);
    } else if (a.D <= 96) {
        if (few) return launch_page<T, 96, 2, 4, 32, 2>(p, st);
        return padded ? launch_page<T, 96, 4, 2, 64, 2>(p, st) : launch_page<T, 96, 8, 1, 64, 3>(p, st);
    } else if (a.D <= 128) {
        if (few) return launch_page<T, 128, 2, 4, 32, 2>(p, st);
        return padded ? launch_page<T, 128, 4, 2, 64, 2>(p, st) : launch_page<T, 128, 8, 1, 64, 3>(p, st);
    } else if (a.D <= 192) {
        return few || padded ? launch_page<T, 192, 2, 2, 32, 2>(p, st) : launch_page<T, 192, 8, 1, 32, 2>(p, st);
    } else {
        return few || padded ? launch_page<T, 256, 2, 2, 32, 2>(p, st) : launch_page<T, 256, 4, 1, 64, 2>(p, st);
    }
}

extern template LuxStatus launch_t<DT_F32>(const ChunkArgs&, hipStream_t);
extern template LuxStatus launch_t<DT_F16>(const ChunkArgs&, hipStream_t);
extern template LuxStatus launch_t<DT_BF16>(const ChunkArgs&, hipStream_t);

}  // namespace chunk
}  // namespace lxq
