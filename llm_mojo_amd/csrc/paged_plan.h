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

// How a call's rows are split over workgroups.  A workgroup takes up to 8 of
// the query heads of a cached head (`tiles` of them cover the group).  Up to kPlanRows rows,
// the blocks of all rows are dealt into splits of one size, the least that
// leaves at most 2^shift splits' worth of whole ones (and kMinBlocks, a
// block a wave): a long row gets many, a short one one, and there are never
// more than `slots`.  More rows fill the card by themselves and are not split (shift -1).
constexpr int kWaves = 4;        // of a workgroup, each taking every kWaves-th block
constexpr int kMinBlocks = 4;    // blocks of the smallest split
constexpr int kPlanRows = 256;   // rows whose lengths a wave holds at once
constexpr int kWorkgroups = 1024;  // aimed at, over all heads

struct Plan {
    int tiles, shift;
    int64_t slots;
};

PKV_HD Plan plan_of(int64_t rows, int n_head, int n_kv) {
    Plan p;
    p.tiles = (n_head / n_kv + 7) / 8;
    p.shift = -1;
    p.slots = rows;
    if (rows > kPlanRows) return p;
    p.shift = 0;
    while (((int64_t)n_kv * p.tiles << (p.shift + 1)) <= kWorkgroups) p.shift++;
    p.slots = rows + ((int64_t)1 << p.shift);
    return p;
}

// Blocks a split, given those of all rows; and splits of a row of nb blocks (at least one, for the row's output).
PKV_HD int64_t split_blocks(int64_t total, int shift) {
    const int64_t n = (total >> shift) + 1;
    return n < kMinBlocks ? kMinBlocks : (n > 0x7fffffff ? 0x7fffffff : n);
}
PKV_HD uint32_t row_splits(uint32_t nb, uint32_t blocks) { return nb <= blocks ? 1 : (nb - 1) / blocks + 1; }

// Byte offsets of a call's workspace: per row the first split and their
// number, per (split, head) the reference and sum of its exponentials, and its sums of values.
struct Work {
    int64_t ml, sums, bytes;
};
PKV_HD Work work_of(const Plan &p, int64_t rows, int n_head, int hd) {
    Work w;
    const int64_t slots = p.shift < 0 ? 0 : p.slots;
    w.ml = (rows * 8 + 255) & ~(int64_t)255;
    w.sums = w.ml + ((slots * n_head * 8 + 255) & ~(int64_t)255);
    w.bytes = w.sums + slots * n_head * hd * 4;
    return w;
}

}  // namespace pkv
