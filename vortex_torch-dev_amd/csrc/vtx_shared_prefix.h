// The plan of shared-prefix decode attention: what its planner writes and the
// attention and combine kernels read.
#pragma once

#include <stdint.h>

namespace vtx_prefix {

// Query rows of a workgroup, at most (rows of 256 columns: two waves share 32).
constexpr int tile_rows(int head_dim) { return head_dim == 256 ? 64 : 128; }

// Tokens from which a run's pages are read once for all: fewer cost more in
// partial results (a layer of 32 runs of eight requests of 8 x 2 heads, read by each
// and once: behind up to 64 tokens 17.0 / 21.2 us, up to 200 35.0 / 24.3, of which
// those past 128 alone once 29.4).  How many requests share them is not looked at.
constexpr int kMinShared = 128;
// Tokens of a chunk: one item per compute unit from kMinChunk on, and past
// kFewChunk one per workgroup slot (us a layer with 256 / 512 / 1024 for it: 64
// requests of 8 x 4 heads behind 8k 33.2 / 27.7 / 29.4, 256 of 8 x 2 behind 8k 46.0 /
// 44.3 / 39.7, 32 of 8 x 2 behind 16k 34.2 / 30.5 / 31.4, 48 of 8 x 1 behind 32k, D 64,
// 28.8 / 25.1 / 29.5, 64 of 8 x 4 behind 32k 64.9 / 61.8 / 60.6).
constexpr int kMinChunk = 128, kFewChunk = 512;
// Own tokens up to which four requests share a workgroup, a wave each, where a
// head has more requests than half its workgroup slots (four waves to so few
// tokens of one request are all latency: 256 requests of up to 128 own tokens
// behind 4k, D 64, 24.7 us a layer, apart 20.6; 256 of 8 heads each with up to 16
// behind 16k 163 and 155; but 4 behind 1k 10.2 and 10.8).
constexpr int short_tokens(int head_dim) { return head_dim == 256 ? 0 : 128; }
static_assert(short_tokens(64) <= kMinChunk, "one chunk each");
constexpr int kXcds = 8;
constexpr int64_t kMaxSegments = 1 << 22;

constexpr int kHeadInts = 16;  // before everything else

// One workgroup's work: `rows` query rows of the requests from the segment's
// on (row0 + r: request (row0 + r) / G after it, head (row0 + r) % G) against
// `pages` entries of the table from `start` on.  Where last is kApart: `pages`
// requests from the segment's on, one per wave, each against its own entries.
constexpr int kApart = 2;
struct alignas(32) Item {
  int32_t segment;
  int32_t row0, rows;
  int32_t start, pages;
  int32_t out;   // first partial row, -1: the rows' only result
  int32_t last;  // the last of the entries is the segment's last
  int32_t reserved;
};

// Per segment: first partial row of its run's chunks, their count, rows from one
// to the next, first partial row of its own chunks (G rows each), their count,
// where its own entries start in the table, and how many there are.
constexpr int kCombineInts = 8;
constexpr int kScratchInts = 10;  // per segment, and 2 more per head (planner only)

// Sizes and places (in int32) of a plan.  Each kv head has a list of items of its
// own, item k of head h at items + 8 (h * most_items + k), and rows of its own.
struct Layout {
  int64_t leaders, shared, combine, counts, items;
  int64_t common, scratch;  // planner only
  int64_t size;
  int64_t slots, cus, most_items, most_rows;  // a head's share, and its lists
};
Layout layout_of(int64_t batch, int64_t heads, int group_size, int head_dim, int cus);

}  // namespace vtx_prefix
