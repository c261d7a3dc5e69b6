// The plan of shared-prefix decode attention: what its planner writes and the
// attention and combine kernels read.
#pragma once

#include <stdint.h>

namespace vtx_prefix {

// Query rows of a workgroup, at most (rows of 256 columns: two waves share 32).
constexpr int tile_rows(int head_dim) { return head_dim == 256 ? 64 : 128; }

constexpr int kMinShared = 128;  // tokens from which a run's pages are read once for all
constexpr int kMinChunk = 128;   // tokens of a chunk, at least
constexpr int kXcds = 8;
constexpr int64_t kMaxSegments = 1 << 22;

constexpr int kHeadInts = 16;  // before everything else

// One workgroup's work: `rows` query rows of the requests from the segment's
// on (row0 + r: request (row0 + r) / G after it, head (row0 + r) % G) against
// `pages` entries of the table from `start` on.
struct alignas(32) Item {
  int32_t segment;
  int32_t row0, rows;
  int32_t start, pages;
  int32_t out;   // first partial row, -1: the rows' only result
  int32_t last;  // the last of the entries is the segment's last
  int32_t reserved;
};

// Per segment: first partial row of its run's chunks, their count, rows from one
// to the next, first partial row of its own chunks (G rows each), their count.
constexpr int kCombineInts = 8;
constexpr int kScratchInts = 9;  // per segment, and 2 more per head (planner only)

// Sizes and places (in int32) of a plan.  Each kv head has a list of items of its
// own, item k of head h at items + 8 (h * most_items + k), and rows of its own.
struct Layout {
  int64_t leaders, shared, combine, counts, items;
  int64_t common, scratch;  // planner only
  int64_t size;
  int64_t slots, most_items, most_rows;  // of a head
};
Layout layout_of(int64_t batch, int64_t heads, int group_size, int head_dim, int cus);

}  // namespace vtx_prefix
