// Where the paged cache keeps a position, and how its pages are found: plain
// integer functions, shared by the kernels (paged.hip) and by host code.
#pragma once

#include <stdint.h>

#ifdef __HIPCC__
#define PKV_HD __host__ __device__ __forceinline__
#else
#define PKV_HD inline
#endif

namespace pkv {

// A cache element is an int8 code or a float16 value (2 bytes).  A block is
// the positions a wave of the attention takes at a time: NT tiles of 16, so
// that one position's 16 * NT / 4 elements of a lane fill 16 bytes.
PKV_HD int block_positions(int elem) { return elem == 1 ? 64 : 32; }

// Values are kept transposed a block, [block][dimension][slot]: position p =
// 16 t + 4 q + i of its block (t < NT, q < 4, i < 4) in slot (q NT + t) 4 + i,
// so the 4 NT positions that matrix-core lanes of quarter q multiply are 16
// consecutive bytes.
PKV_HD int value_slot(int elem, int p) {
    const int nt = elem == 1 ? 4 : 2;
    const int t = p >> 4, q = (p >> 2) & 3, i = p & 3;
    return (q * nt + t) * 4 + i;
}

// The page of position `pos` of a table row of `width` pages, or -1 where
// the position or the page is none of the cache's (`pages` of `page`
// positions).
PKV_HD int page_of(const int32_t *row, int64_t width, int page, int64_t pages, int64_t pos) {
    if (pos < 0 || pos >= width * page) return -1;
    const int32_t at = row[pos / page];
    return at >= 0 && at < pages ? at : -1;
}

// A sequence's length as the kernels take it: inside the table's row.
PKV_HD int64_t clamp_len(int64_t len, int64_t width, int page) {
    const int64_t most = width * page;
    return len < 0 ? 0 : (len > most ? most : len);
}

}  // namespace pkv
