// The plan of shared-prefix decode attention: what its planner writes and the
// attention and combine kernels read.
#pragma once

#include <stdint.h>

namespace vtx_prefix {

constexpr int kTileRows = 128;      // query rows per item
constexpr int kMinShared = 128;     // tokens from which a run's pages are read once for all
constexpr int kMinChunk = 128;      // tokens of a chunk, at least
constexpr int64_t kMaxSegments = 1 << 24;

// Header, int32 each.
constexpr int kHeadRunItems = 0;  // items of runs, listed first
constexpr int kHeadOwnItems = 1;  // items of single requests
constexpr int kHeadRows = 2;      // partial rows in all
constexpr int kHeadInts = 16;

// One workgroup's work: `rows` query rows of the requests from the segment's
// on (row r: request r / G after it, its head r % G) against pages
// [page0, page1) of the segment.
struct alignas(32) Item {
  int32_t segment;
  int32_t row0, rows;
  int32_t page0, page1;
  int32_t out;   // first partial row, -1: the rows' only result
  int32_t last;  // page1 is the segment's last page
  int32_t reserved;
};

// Per segment: first partial row of its run's chunks, their count, rows from one
// to the next, first partial row of its own chunks (G rows each), their count.
constexpr int kCombineInts = 8;
constexpr int kSegmentInts = 2;  // (planner only) a run's requests and shared pages, at its first element

// Places in the plan, in int32.
struct Layout {
  int64_t leaders, shared, combine, items;
  int64_t common, scratch, segments, offsets, rows;  // planner only
  int64_t size;
};

int aimed_items(int head_dim, int cus);
int64_t most_items(int64_t segments, int group_size, int64_t slots);
int64_t most_rows(int64_t segments, int group_size, int64_t slots);
Layout layout_of(int64_t segments, int64_t items);

}  // namespace vtx_prefix
