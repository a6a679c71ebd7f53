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
// kPlanRows rows, a row of more than `per` blocks (per_of, from the sum over
// all rows) is cut into segments of one size, each a workgroup; the segments
// of all rows, one after another, are the slots of the grid and of the
// workspace.  More rows fill the card by themselves: a workgroup a row
// (columns 0), as do tables of `uncut` blocks at most, whose rows end before a
// second launch would have joined their parts.
//
// kWorkgroups: 2.7 times those that run at once.  4 rows of float16, 342 MB:
// 1536 64.9 us, 2048 62.2, 2560 62.1; 64 rows of int8, 1082 MB: 199, 201, 202.
// kPlanRows: 300 rows of up to 16384 positions and one head, each its own
// workgroup 255 us, cut 139; 600 rows 203 and 151.
constexpr int kWaves = 4;         // of a workgroup, each taking every kWaves-th block
constexpr int kPlanRows = 1024;   // rows whose lengths a wave holds at once
constexpr int kWorkgroups = 2048;
constexpr int64_t kMaxBlocks = (int64_t)1 << 31;  // of all rows' tables, where they may be cut

// A segment's least blocks, by how many of the CUs rows and heads alone give a
// workgroup, and twice as many in a table that is not cut.  In a graph, us:
// 1 row x 8 heads of 900 float16 positions cut into 8 blocks 11.8, uncut 17.7, of
// 500 12.2 and 11.6; 16 x 8 of 1000 int8 uncut 14.8, cut 16.4, of 2000 in 16
// blocks 20.3, in 8 25; 32 x 8 of 1000 uncut 16.1, in 16 21, and in a table for
// 4096 whole 19.4, in 8 25.8.
constexpr int kCUs = 256;

struct Plan {
    int tiles, columns;
    uint32_t least, uncut;  // blocks of a row, and of a table, that is not cut
};

PKV_HD Plan plan_of(int64_t rows, int n_head, int n_kv) {
    Plan p;
    p.tiles = (n_head / n_kv + 7) / 8;
    const int64_t all = (int64_t)n_kv * p.tiles;
    p.columns = rows > kPlanRows ? 0 : (all >= kWorkgroups ? 1 : (int)(kWorkgroups / all));
    p.least = rows * all >= kCUs ? 32 : (rows * all >= kCUs / 2 ? 16 : 8);
    p.uncut = 2 * p.least;
    return p;
}

// Blocks of a segment at most, given those of all rows.
PKV_HD uint32_t per_of(uint32_t total, int columns, uint32_t least) {
    const uint32_t n = total / (uint32_t)columns + 1;
    return n < least ? least : (n + kWaves - 1) / kWaves * kWaves;
}
// Segments of a row, and their blocks (the last one's may be fewer): a multiple of the waves, so a row may
// need fewer of them than it has slots.
PKV_HD uint32_t segments_of(uint32_t blocks, uint32_t per) { return (blocks + per - 1) / per; }
PKV_HD uint32_t segment_blocks(uint32_t blocks, uint32_t segments) {
    return ((blocks + segments - 1) / segments + kWaves - 1) / kWaves * kWaves;
}

// Slots at most: a segment a row, and one a column, since per is above total / columns.
PKV_HD int64_t slots_of(const Plan &p, int64_t rows) { return p.columns ? p.columns + rows : 0; }

// Byte offsets of a call's workspace: per row its first slot and its segments, per
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
