// Planner of shared-prefix decode attention for gfx950: which requests of a
// block table share leading pages, and how the attention's work is divided.
//
// Segment s = b * H + h (request b, kv head h) of a table holds pages
// kv_indices[kv_indptr[s] .. kv_indptr[s+1]).  Per kv head, consecutive
// requests with pages form a run while their group ids are equal (without
// ids: while their first entries are).  A run of several requests shares its
// longest common prefix of entries, less than every request's page count, so
// that each keeps at least its last page (the only one that may be partial).
// The table decides: what ids promise is checked against the entries.
//
// Two launches: one workgroup per segment finds the length of the prefix it
// has in common with the request before (the minimum of these over a run is
// the run's); one workgroup then scans the segments, head by head, into runs,
// and writes the work items of the attention: (rows of a run or a request) x
// (pages of a chunk), at most kTileRows rows each, chunks sized so that all
// items together are a few per workgroup slot of the device.
#include "vtx_shared_prefix.h"

#include "vtx_device.h"
#include "vtx_host.h"

namespace {

using namespace vtx_prefix;

struct PlanArgs {
  const int32_t* indptr;
  const int32_t* indices;
  int64_t indices_len;
  const int32_t* ids;
  int32_t B, H, G, P;
  int32_t slots;      // items aimed at
  int32_t max_items;  // room for
  int32_t min_tokens; // of a chunk
  Layout at;
  int32_t* plan;
};

// Pages of segment s (0: none, or a range outside the table), from `start`.
__device__ __forceinline__ int pages_of(const PlanArgs& a, int s, int& start) {
  start = a.indptr[s];
  const long long end = a.indptr[s + 1];
  return start >= 0 && end > start && end <= a.indices_len ? (int)(end - start) : 0;
}

// common[s]: entries that segment (b, h) has in common with (b - 1, h), or -1
// where no run goes through the two.
constexpr int kCompareThreads = 256;
constexpr int kAhead = 4;  // entries per thread and pass
__global__ __launch_bounds__(kCompareThreads) void prefix_compare_kernel(PlanArgs a) {
  __shared__ int s_first;
  const int s = blockIdx.x, b = s / a.H;
  int* out = a.plan + a.at.common + s;
  int start, before;
  const int n = pages_of(a, s, start);
  const int m = b > 0 ? pages_of(a, s - a.H, before) : 0;
  bool linked = n > 0 && m > 0;
  if (linked)
    linked = a.ids ? a.ids[b] == a.ids[b - 1] : a.indices[start] == a.indices[before];
  if (!linked) {  // uniform
    if (threadIdx.x == 0) *out = -1;
    return;
  }
  const int len = min(n, m);
  if (threadIdx.x == 0) s_first = len;
  __syncthreads();
  for (int at = 0; at < len; at += kCompareThreads * kAhead) {
    int x[kAhead], y[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = min(at + k * kCompareThreads + (int)threadIdx.x, len - 1);
      x[k] = a.indices[start + (long long)i];
      y[k] = a.indices[before + (long long)i];
    }
    int first = len;
#pragma unroll
    for (int k = kAhead - 1; k >= 0; --k)
      if (x[k] != y[k]) first = min(at + k * kCompareThreads + (int)threadIdx.x, len - 1);
    if (first < len) atomicMin(&s_first, first);
    __syncthreads();
    const bool found = s_first < len;
    __syncthreads();
    if (found) break;  // uniform
  }
  if (threadIdx.x == 0) *out = s_first;
}

constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / vtx::kWave;

// Exclusive scan over the workgroup of four sums at a time; `all`: the totals.
struct Four {
  int v[4];
};
__device__ __forceinline__ Four block_scan(Four x, int (*lds)[4], Four& all) {
  const int wave = threadIdx.x / vtx::kWave, lane = vtx::lane_id();
  Four inc = x;
#pragma unroll
  for (int i = 0; i < 4; ++i) inc.v[i] = (int)vtx::wave_prefix_sum((uint32_t)x.v[i]);
  if (lane == vtx::kWave - 1)
    for (int i = 0; i < 4; ++i) lds[wave][i] = inc.v[i];
  __syncthreads();
  Four r;
  for (int i = 0; i < 4; ++i) {
    int before = 0, total = 0;
    for (int w = 0; w < kPlanWaves; ++w) {
      before += w < wave ? lds[w][i] : 0;
      total += lds[w][i];
    }
    r.v[i] = before + inc.v[i] - x.v[i];
    all.v[i] = total;
  }
  __syncthreads();
  return r;
}

// A stretch of segments in head-major order as the scan sees it: the run that
// its last element lies in.
struct Run {
  int start;   // first element of that run, -1: before the stretch
  int shared;  // minimum over the run's elements seen so far
};
__device__ __forceinline__ Run join(const Run& a, const Run& b) {
  return b.start >= 0 ? b : Run{a.start, min(a.shared, b.shared)};
}

// Units of up to `per` pages of n: their count, each of ceil(n / count) pages.
__device__ __forceinline__ int chunks(int n, int per, int& pages) {
  const int c = n > 0 ? (n + per - 1) / per : 0;
  pages = c > 0 ? (n + c - 1) / c : 0;
  return c > 0 ? (n + pages - 1) / pages : 0;
}

__global__ __launch_bounds__(kPlanThreads) void prefix_plan_kernel(PlanArgs a) {
  __shared__ int s_scan[kPlanWaves][4];
  __shared__ int s_run[kPlanWaves][2];
  __shared__ unsigned long long s_total;
  const int S = a.B * a.H, tid = threadIdx.x, wave = tid / vtx::kWave, lane = vtx::lane_id();
  const int each = (S + kPlanThreads - 1) / kPlanThreads;
  const int i0 = min(S, tid * each), i1 = min(S, i0 + each);
  int32_t* plan = a.plan;
  const int32_t* common = plan + a.at.common;
  int32_t* first = plan + a.at.scratch;  // of an element's run
  int32_t* info = plan + a.at.segments;
  auto seg = [&](int i) { return (i % a.B) * a.H + i / a.B; };  // element i = h * B + b

  // 1. Runs.  Every element's run so far; a run's last element then has the
  // run's minimum, and publishes (elements, pages) where its first one reads.
  Run mine{-1, 0x7fffffff};
  for (int i = i0; i < i1; ++i) {
    const int s = seg(i);
    int start;
    const int limit = pages_of(a, s, start) - 1;
    const int c = i % a.B == 0 ? -1 : common[s];
    mine = join(mine, c < 0 ? Run{i, limit} : Run{-1, min(c, limit)});
  }
  Run inc = mine;
#pragma unroll
  for (int d = 1; d < vtx::kWave; d <<= 1) {
    const Run o{__shfl_up(inc.start, d), __shfl_up(inc.shared, d)};
    if (lane >= d) inc = join(o, inc);
  }
  if (lane == vtx::kWave - 1) {
    s_run[wave][0] = inc.start;
    s_run[wave][1] = inc.shared;
  }
  if (tid == 0) s_total = 0;
  __syncthreads();
  Run at{-1, 0x7fffffff};
  for (int w = 0; w < wave; ++w) at = join(at, Run{s_run[w][0], s_run[w][1]});
  {
    const Run o{__shfl_up(inc.start, 1), __shfl_up(inc.shared, 1)};
    if (lane > 0) at = join(at, o);
  }
  for (int i = i0; i < i1; ++i) {
    const int s = seg(i);
    int start;
    const int limit = pages_of(a, s, start) - 1;
    const int c = i % a.B == 0 ? -1 : common[s];
    at = join(at, c < 0 ? Run{i, limit} : Run{-1, min(c, limit)});
    first[i] = at.start;
    const bool last = i + 1 == S || (i + 1) % a.B == 0 || common[seg(i + 1)] < 0;
    if (last) {
      const int n = i + 1 - at.start, h8 = kSegmentInts * at.start;
      info[h8 + 0] = n;
      info[h8 + 1] = n > 1 ? max(0, at.shared) : 0;
    }
  }
  __syncthreads();

  // 2. What is shared; the work in tokens x row tiles, and from it the chunks.
  unsigned long long work = 0;
  for (int i = i0; i < i1; ++i) {
    const int s = seg(i), f = first[i], n = info[kSegmentInts * f], e = info[kSegmentInts * f + 1];
    int start;
    const int pages = pages_of(a, s, start);
    plan[a.at.leaders + s] = f % a.B;
    plan[a.at.shared + s] = e;
    const int used = (long long)e * a.P >= kMinShared ? e : 0;
    const int tiles = (int)(((long long)n * a.G + kTileRows - 1) / kTileRows);
    if (f == i) work += (unsigned long long)tiles * used * a.P;
    work += (unsigned long long)(pages - used) * a.P;
  }
  atomicAdd(&s_total, work);
  __syncthreads();
  const unsigned long long even = (s_total + a.slots - 1) / a.slots;
  const int tokens = (int)min(max(even, (unsigned long long)a.min_tokens), 0x3fffffffull);
  const int per = (int)((tokens + (long long)a.P - 1) / a.P);

  // 3. Items and partial rows of every element: its run's (first element only)
  // and its own.
  Four count{{0, 0, 0, 0}};  // run items, own items, partial rows of runs, of requests
  auto measure = [&](int i, int& tiles, int& rc, int& rp, int& oc, int& op, int& used, int& n) {
    const int s = seg(i), f = first[i];
    n = info[kSegmentInts * f];
    const int e = info[kSegmentInts * f + 1];
    int start;
    const int pages = pages_of(a, s, start);
    used = (long long)e * a.P >= kMinShared ? e : 0;
    tiles = (int)(((long long)n * a.G + kTileRows - 1) / kTileRows);
    rc = chunks(used, per, rp);
    oc = chunks(pages - used, per, op);
  };
  for (int i = i0; i < i1; ++i) {
    int tiles, rc, rp, oc, op, used, n;
    measure(i, tiles, rc, rp, oc, op, used, n);
    if (first[i] == i) {
      count.v[0] += tiles * rc;
      count.v[2] += n * a.G * rc;
    }
    count.v[1] += oc;
    count.v[3] += rc + oc > 1 ? oc * a.G : 0;  // (a single partial result is the result)
  }
  Four all;
  Four off = block_scan(count, s_scan, all);
  int32_t* item_at = plan + a.at.offsets;  // run items before element i, own items before element i
  for (int i = i0; i < i1; ++i) {
    int tiles, rc, rp, oc, op, used, n;
    measure(i, tiles, rc, rp, oc, op, used, n);
    item_at[i] = off.v[0];
    item_at[S + 1 + i] = off.v[1];
    int32_t* run_row = plan + a.at.rows + i;  // partial rows of the run, at its first element; of the request
    if (first[i] == i) {
      run_row[0] = off.v[2];
      off.v[0] += tiles * rc;
      off.v[2] += n * a.G * rc;
    }
    run_row[S] = all.v[2] + off.v[3];
    off.v[1] += oc;
    off.v[3] += rc + oc > 1 ? oc * a.G : 0;
  }
  const bool fits = all.v[0] + all.v[1] <= a.max_items;  // (always: slots and max_items belong together)
  if (tid == 0) {
    item_at[S] = all.v[0];
    item_at[2 * S + 1] = all.v[1];
    plan[kHeadRunItems] = fits ? all.v[0] : 0;
    plan[kHeadOwnItems] = fits ? all.v[1] : 0;
    plan[kHeadRows] = all.v[2] + all.v[3];
  }
  __syncthreads();

  // 4. The items, every thread some of both kinds; the element by bisection.
  if (fits) {
    const int total = all.v[0] + all.v[1];
    for (int k = tid; k < total; k += kPlanThreads) {
      const bool run = k < all.v[0];
      const int32_t* list = run ? item_at : item_at + S + 1;
      const int j = run ? k : k - all.v[0];
      int lo = 0, hi = S;  // list[lo] <= j < list[hi]
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (list[mid] <= j) lo = mid;
        else hi = mid;
      }
      const int i = lo, in = j - list[i];
      int tiles, rc, rp, oc, op, used, n;
      measure(i, tiles, rc, rp, oc, op, used, n);
      int start;
      const int pages = pages_of(a, seg(i), start);
      Item it;
      it.segment = seg(i);
      if (run) {  // the tiles of a chunk side by side: they read the same pages
        const int c = in / tiles, t = in - c * tiles, rows = n * a.G;
        it.row0 = t * kTileRows;
        it.rows = min(rows - it.row0, kTileRows);
        it.page0 = c * rp;
        it.page1 = min(used, it.page0 + rp);
        it.out = plan[a.at.rows + i] + c * rows + it.row0;
      } else {
        it.row0 = 0;
        it.rows = a.G;
        it.page0 = used + in * op;
        it.page1 = min(pages, it.page0 + op);
        it.out = rc + oc > 1 ? plan[a.at.rows + S + i] + in * a.G : -1;
      }
      it.reserved = 0;
      it.last = it.page1 == pages ? 1 : 0;
      reinterpret_cast<Item*>(plan + a.at.items)[k] = it;
    }
  }
  __syncthreads();

  // 5. Where the combine launch finds a segment's partial rows.
  for (int i = i0; i < i1; ++i) {
    int tiles, rc, rp, oc, op, used, n;
    measure(i, tiles, rc, rp, oc, op, used, n);
    const int f = first[i];
    int32_t* to = plan + a.at.combine + (long long)kCombineInts * seg(i);
    to[0] = plan[a.at.rows + f] + (i - f) * a.G;
    to[1] = rc;
    to[2] = n * a.G;
    to[3] = plan[a.at.rows + S + i];
    to[4] = oc;
  }
}

}  // namespace

namespace vtx_prefix {

// Workgroups of the attention that the device holds at a time, and the items
// that a plan aims at.
int aimed_items(int head_dim, int cus) { return cus * (head_dim == 64 ? 6 : (head_dim == 128 ? 4 : 2)); }

int64_t most_items(int64_t segments, int group_size, int64_t slots) {
  // Runs: tiles x ceil(pages / per) <= tiles x pages / per + tiles, at most one
  // run per two segments; requests: pages / per + 1 each.  The sums of x / per
  // are at most `slots` together.
  return slots + segments + segments / 2 + segments * group_size / kTileRows + 1;
}

int64_t most_rows(int64_t segments, int group_size, int64_t slots) {
  // n * G rows per chunk of a run (at most kTileRows per tile), G per chunk of a request.
  return slots * kTileRows + 2 * segments * group_size;
}

Layout layout_of(int64_t segments, int64_t items) {
  Layout l;
  int64_t at = kHeadInts;
  auto take = [&](int64_t n) {
    const int64_t r = at;
    at += (n + 7) / 8 * 8;  // (32-byte items)
    return r;
  };
  l.leaders = take(segments);
  l.shared = take(segments);
  l.combine = take(kCombineInts * segments);
  l.items = take((int64_t)(sizeof(Item) / sizeof(int32_t)) * items);
  l.common = take(segments);
  l.scratch = take(segments);
  l.segments = take(kSegmentInts * segments);
  l.offsets = take(2 * (segments + 1));
  l.rows = take(2 * segments);
  l.size = at;
  return l;
}

}  // namespace vtx_prefix

extern "C" int64_t vtx_shared_prefix_plan_len(int32_t batch_size, int32_t num_kv_heads, int32_t group_size,
                                              int32_t head_dim) {
  const int cus = vtx::device_cu_count();
  if (batch_size < 0 || num_kv_heads < 1 || cus <= 0 || !vtx_paged_decode_attention_supported(head_dim, group_size))
    return 0;
  const int64_t S = (int64_t)batch_size * num_kv_heads;
  if (S > kMaxSegments) return 0;
  return layout_of(S, most_items(S, group_size, aimed_items(head_dim, cus))).size;
}

extern "C" int vtx_plan_shared_prefix(const int32_t* kv_indptr, const int32_t* kv_indices, int64_t kv_indices_len,
                                      const int32_t* group_ids, int32_t batch_size, int32_t num_kv_heads,
                                      int32_t group_size, int32_t head_dim, int32_t page_size, int32_t* plan,
                                      int64_t plan_len, void* stream) {
  vtx::clear_error();
  if (batch_size < 0 || num_kv_heads < 1 || page_size < 1 || kv_indices_len < 0)
    return vtx::fail(VTX_E_INVALID, "plan_shared_prefix: bad sizes");
  if (!vtx_paged_decode_attention_supported(head_dim, group_size))
    return vtx::fail(VTX_E_INVALID, "plan_shared_prefix: head_dim %d with %d query heads per kv head not supported",
                     head_dim, group_size);
  const int64_t S = (int64_t)batch_size * num_kv_heads;
  if (S > kMaxSegments) return vtx::fail(VTX_E_INVALID, "plan_shared_prefix: too many segments");
  if (S == 0) return VTX_OK;
  if (!kv_indptr || !plan || (kv_indices_len > 0 && !kv_indices))
    return vtx::fail(VTX_E_INVALID, "plan_shared_prefix: null pointer");
  const int cus = vtx::device_cu_count();
  if (cus <= 0) return vtx::fail(VTX_E_DEVICE, "plan_shared_prefix: device query failed");
  PlanArgs a;
  a.slots = aimed_items(head_dim, cus);
  a.max_items = (int32_t)most_items(S, group_size, a.slots);
  a.at = layout_of(S, a.max_items);
  if (plan_len < a.at.size || reinterpret_cast<uintptr_t>(plan) % 32)
    return vtx::fail(VTX_E_INVALID, "plan_shared_prefix: plan of %lld int32 (32-byte aligned) needed, got %lld",
                     (long long)a.at.size, (long long)plan_len);
  a.indptr = kv_indptr;
  a.indices = kv_indices;
  a.indices_len = kv_indices_len;
  a.ids = group_ids;
  a.B = batch_size;
  a.H = num_kv_heads;
  a.G = group_size;
  a.P = page_size;
  a.min_tokens = kMinChunk;
  a.plan = plan;
  hipStream_t s = vtx::as_stream(stream);
  prefix_compare_kernel<<<(int)S, kCompareThreads, 0, s>>>(a);
  prefix_plan_kernel<<<1, kPlanThreads, 0, s>>>(a);
  return vtx::check_launch("plan_shared_prefix");
}
