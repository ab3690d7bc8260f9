// chunk_places.h -- where the chunk attention's tiles, stages and ranges lie: whole
// numbers only, which the host compiles too (tests/test_chunk_places.py).
//
// Positions and lengths are below 2^31, but the places that are looked at go on to
// the end of a stage, or of a wave's part of one, up to 256 tokens behind: places
// are uint32_t and compared without a sign.
#pragma once
#include <stdint.h>

#ifdef __HIPCC__
#include <hip/hip_runtime.h>
#define LXQ_BOTH __host__ __device__ __forceinline__
#else
#define LXQ_BOTH inline
#endif

namespace lxq {
namespace chunk {

constexpr int kLeastPiece = 2;

LXQ_BOTH int clamp(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }

// rows and tokens of a tile
struct Tile {
    int first, m;    // first new token (row of q), tokens
    int pos, n;      // position of the first one; tokens held
    int base, end;   // cached tokens that the tile sees lie in [base, end)
    int units;       // stages; a tile that sees nothing has one, which writes its zeros
};
// The tile-th tile of tb tokens of a request whose rows are [s0, s1), whose first new
// token is at `pos` and which holds n tokens; stages of `st` tokens.  pos + s1 - s0 is
// below 2^31.  tile below 0: places of rows before the first request's.
LXQ_BOTH Tile tile_at(int s0, int s1, int pos, int n, int tile, int tb, int window, int st) {
    Tile t;
    const int i0 = tile * tb;
    t.first = s0 + i0;
    t.m = tile < 0 ? 0 : clamp(s1 - s0 - i0, 0, tb);
    t.pos = t.m > 0 ? pos + i0 : 0;
    t.n = n;
    t.end = t.pos + t.m < t.n ? t.pos + t.m : t.n;
    t.base = window > 0 && t.pos + 1 > window ? (t.pos + 1 - window) & ~15 : 0;
    t.units = t.end > t.base ? (int)(((uint32_t)(t.end - t.base) + (uint32_t)st - 1) / (uint32_t)st) : 1;
    return t;
}
// the tokens that the tile's i-th row sees: [from, to)
LXQ_BOTH void seen_by(const Tile& t, int i, int window, int& from, int& to) {
    const int pos = t.pos + i;
    from = window > 0 && pos + 1 > window ? pos + 1 - window : 0;
    to = pos + 1 < t.n ? pos + 1 : t.n;
}

// the first token of stage u, and the end of the stages before u
LXQ_BOTH uint32_t stage_at(const Tile& t, int u, int st) { return (uint32_t)t.base + (uint32_t)u * (uint32_t)st; }
LXQ_BOTH uint32_t stages_end(const Tile& t, int u, int st) {
    const uint32_t at = stage_at(t, u, st);
    return at < (uint32_t)t.end ? at : (uint32_t)t.end;
}
// n tokens from `at` on: all in the tile's; some of [from, to); all of them in it
LXQ_BOTH bool is_whole(const Tile& t, uint32_t at, int n) { return at + (uint32_t)n <= (uint32_t)t.end; }
LXQ_BOTH bool is_seen(uint32_t at, int n, int from, int to) { return at < (uint32_t)to && at + (uint32_t)n > (uint32_t)from; }
LXQ_BOTH bool is_inside(uint32_t at, int n, int from, int to) { return at >= (uint32_t)from && at + (uint32_t)n <= (uint32_t)to; }
// place `at`, or the tile's last one; the first of its run of `run` tokens
LXQ_BOTH int or_last(const Tile& t, uint32_t at) { return at < (uint32_t)t.end ? (int)at : t.end - 1; }
LXQ_BOTH int or_last_run(const Tile& t, uint32_t at, int run) { return at < (uint32_t)t.end ? (int)at : (t.end - 1) & ~(run - 1); }
// The steps [a, b) of a wave whose part of step 0 is the `bt` tokens from t0 on, of step j
// those j st behind, in which all of its tokens are in [from, to)
LXQ_BOTH void steps_inside(uint32_t t0, int bt, int st, int from, int to, int& a, int& b) {
    a = (uint32_t)from > t0 ? (int)(((uint32_t)from - t0 + (uint32_t)st - 1) / (uint32_t)st) : 0;
    b = (uint32_t)to >= t0 + (uint32_t)bt ? (int)(((uint32_t)to - (uint32_t)bt - t0) / (uint32_t)st) + 1 : 0;
}

// The units of all tiles in 2^log equal ranges, none of them empty.  A piece of a tile costs as
// much beyond its units as a few of them: a cut less than `least` units from a
// tile's end is moved there.  Ranges are at least four times as long, so that
// at most one cut moves to each end.
struct Ranges {
    uint64_t units;
    int log, least;
    LXQ_BOTH Ranges(uint64_t n, int l) : units(n), log(l) {
        while (n >> log == 0) log--;
        const uint64_t quarter = n >> (log + 2);
        least = quarter < kLeastPiece ? (int)quarter : kLeastPiece;
    }
    LXQ_BOTH uint64_t first(int w) const { return (units * (uint32_t)w) >> log; }
    // the range of unit u; of one behind all (starts that decrease lay tiles there) the last
    LXQ_BOTH int of(uint64_t u) const {
        if (u >= units) return (1 << log) - 1;
        int w = (int)((double)(u + 1) * (double)(1 << log) / (double)units);  // or one beside it
        while (first(w) > u) w--;
        while (first(w + 1) <= u) w++;
        return w;
    }
    // where a cut `at` units into a tile of n goes
    LXQ_BOTH int cut(int at, int n) const { return at < least ? 0 : n - at < least ? n : at; }
};

}  // namespace chunk
}  // namespace lxq
