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
constexpr int64_t kMaxSegments = 1 << 24;

// Header, int32 each.
constexpr int kHeadItems = 0;
constexpr int kHeadInts = 16;

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
constexpr int kScratchInts = 9;  // per segment, and 2 more (planner only)

// Places in the plan, in int32.
struct Layout {
  int64_t leaders, shared, combine, items;
  int64_t common, scratch;  // planner only
  int64_t size;
};

int aimed_items(int head_dim, int cus);
int64_t most_items(int64_t segments, int group_size, int head_dim, int64_t slots);
int64_t most_rows(int64_t segments, int group_size, int head_dim, int64_t slots);
Layout layout_of(int64_t segments, int64_t items);

}  // namespace vtx_prefix
