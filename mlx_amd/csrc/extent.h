// extent.h -- host arithmetic of the serving operators' argument checks: the
// bytes that strided rows cover, and whether a buffer holds them.  Sizes that
// 64 bits cannot hold count as SIZE_MAX, which no buffer holds.
#pragma once
#include <stddef.h>
#include <stdint.h>

namespace lxh {

// strides and offsets up to 2^40 elements
inline bool stride_ok(int64_t s, int64_t row) { return s == 0 || (s >= row && s <= (1ll << 40)); }
inline bool offset_ok(int64_t o) { return o >= 0 && o <= (1ll << 40); }

// bytes from an array's start to the end of the last of `rows` rows; 2^31 rows
// 2^40 elements apart pass 64 bits
inline size_t extent(int64_t rows, int64_t stride, int64_t row, size_t esz) {
    if (rows <= 0 || row <= 0) return 0;
    int64_t last, end;
    size_t bytes;
    if (__builtin_mul_overflow(rows - 1, stride, &last) || __builtin_add_overflow(last, row, &end) ||
        __builtin_mul_overflow((size_t)end, esz, &bytes))
        return SIZE_MAX;
    return bytes;
}

// `bytes` of a buffer of `size`, from `skip` on
inline bool holds(size_t size, size_t skip, size_t bytes) { return skip <= size && bytes <= size - skip; }

}  // namespace lxh
