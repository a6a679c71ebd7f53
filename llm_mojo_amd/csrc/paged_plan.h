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

// A block is the positions a wave of the attention takes at a time: two
// tiles of 16.
constexpr int kBlock = 32;

// Values are kept transposed a block, [block][dimension][slot]: position p =
// 16 t + 4 q + i of its block (t < 2, q < 4, i < 4) in slot 8 q + 4 t + i, so
// the eight positions that matrix-core lanes of quarter q multiply lie
// together.
PKV_HD int value_slot(int p) { return ((p >> 2) & 3) * 8 + (p >> 4) * 4 + (p & 3); }

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
// the query heads of a cached head (`tiles` of them cover the group).  Up to
// kPlanRows rows, the blocks of all rows in one line are cut into columns of
// one size, and a workgroup takes what a column has of a row (a segment): a
// long row gets many, a short one one.  More rows fill the card by
// themselves: a workgroup a row (columns 0).
constexpr int kWaves = 4;         // of a workgroup, each taking every kWaves-th block
constexpr int kMinBlocks = 16;    // of a column
constexpr int kPlanRows = 256;    // rows whose lengths a wave holds at once
constexpr int kWorkgroups = 2048;
constexpr int64_t kMaxBlocks = (int64_t)1 << 31;  // of all rows' tables, where they are cut into columns

struct Plan {
    int tiles, columns;
};

PKV_HD Plan plan_of(int64_t rows, int n_head, int n_kv) {
    Plan p;
    p.tiles = (n_head / n_kv + 7) / 8;
    p.columns = 0;
    if (rows > kPlanRows) return p;
    const int64_t all = (int64_t)n_kv * p.tiles;
    p.columns = all >= kWorkgroups ? 1 : (int)(kWorkgroups / all);
    return p;
}

// Blocks of a column, given those of all rows: at most `columns` columns, a multiple of the waves.
PKV_HD uint32_t column_blocks(uint32_t total, int columns) {
    const uint32_t n = total / (uint32_t)columns + 1;
    return n < (uint32_t)kMinBlocks ? (uint32_t)kMinBlocks : (n + kWaves - 1) / kWaves * kWaves;
}

// Row r, whose blocks are [begin, end) of the line, has its segments of columns begin / per ... in slots
// r + column: the pairs of (row, column) go up in one or both along the line, so no two share a slot, and
// the row of a slot is the number of rows k with k + 1 + end of k / per at most the slot.
PKV_HD int64_t slots_of(const Plan &p, int64_t rows) { return p.columns ? p.columns + rows : 0; }

// Byte offsets of a call's workspace: per row its first and last column, per
// (slot, head) the reference and sum of its exponentials, and its sums of values.
struct Work {
    int64_t ml, sums, bytes;
};
PKV_HD Work work_of(const Plan &p, int64_t rows, int n_head, int hd) {
    Work w;
    const int64_t slots = slots_of(p, rows);
    w.ml = (rows * 8 + 255) & ~(int64_t)255;
    w.sums = w.ml + ((slots * n_head * 8 + 255) & ~(int64_t)255);
    w.bytes = w.sums + slots * n_head * hd * 4;
    return w;
}

}  // namespace pkv
