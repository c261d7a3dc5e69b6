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
// Sharing has one level, the minimum over the run: where all requests begin
// with a page and groups of them go on alike behind it, only ids tell the groups
// apart (32 groups of eight behind 4k tokens, 8 x 2 heads, all behind one common
// page: 315 us a layer without ids, 98 with).
//
// Two launches, or one for few requests.  One wave per segment finds the length
// of the prefix that it has in common with the request before (the minimum of
// these over a run is the run's).  One workgroup per kv head then scans its
// requests into runs and writes the head's work items: (rows of a run or a
// request) x (entries of a chunk), tile_rows rows at most, chunks sized so that a
// head has its share of the device's workgroup slots.  (One workgroup for all
// heads is bound by its instructions: plans of 265 requests of 8 heads 29.8 us,
// this way 10.7; of 69 16.6 and 9.1.)  Latency bounds both: the loads of the
// comparison, then a chain of steps in one workgroup.  More requests than fit
// in LDS keep their numbers in the plan's memory (4096 of 8 heads 106 us).
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
  int32_t tile_shift;  // log2 of an item's rows, at most
  int32_t apart;       // short_tokens
  Layout at;
  int32_t* plan;
};

// Pages of segment s (0: none, or a range outside the table), from `start`.
__device__ __forceinline__ int pages_of(const PlanArgs& a, int s, int& start) {
  start = a.indptr[s];
  const long long end = a.indptr[s + 1];
  return start >= 0 && end > start && end <= a.indices_len ? (int)(end - start) : 0;
}

// Entries that segment s = (b, h) has in common with (b - 1, h), or -1 where no
// run goes through the two.  One wave.
constexpr int kAhead = 8;  // entries per lane and pass
__device__ __forceinline__ int common_entries(const PlanArgs& a, int s) {
  const int lane = vtx::lane_id(), b = s / a.H;
  int start, before;
  const int n = pages_of(a, s, start);
  const int m = b > 0 ? pages_of(a, s - a.H, before) : 0;
  const bool named = a.ids && b > 0;
  const bool same = named ? a.ids[b] == a.ids[b - 1] : true;
  if (n == 0 || m == 0 || !same) return -1;  // uniform
  const int len = min(n, m);
  int common = len;
  for (int at = 0; at < len; at += vtx::kWave * kAhead) {
    int x[kAhead], y[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = min(at + k * vtx::kWave + lane, len - 1);
      x[k] = a.indices[start + (long long)i];
      y[k] = a.indices[before + (long long)i];
    }
    uint64_t differ[kAhead], any = 0;
#pragma unroll
    for (int k = 0; k < kAhead; ++k) any |= differ[k] = __ballot(x[k] != y[k]);
    if (any) {
#pragma unroll
      for (int k = kAhead - 1; k >= 0; --k)
        if (differ[k]) common = at + k * vtx::kWave + __builtin_ctzll(differ[k]);
      common = min(common, len - 1);  // (lanes past the end compare the last entry)
      break;
    }
  }
  return !named && common == 0 ? -1 : common;  // (other first entries: another run)
}

constexpr int kCompareWaves = 4;
__global__ __launch_bounds__(kCompareWaves* vtx::kWave) void prefix_compare_kernel(PlanArgs a) {
  const int s = blockIdx.x * kCompareWaves + vtx::uniform(threadIdx.x / vtx::kWave);
  if (s >= a.B * a.H) return;
  const int common = common_entries(a, s);
  if (vtx::lane_id() == 0) a.plan[a.at.common + s] = common;
}

constexpr int kPlanThreads = 256;
constexpr int kPlanWaves = kPlanThreads / vtx::kWave;

// Exclusive scan over the workgroup of four sums at a time; `all`: the totals.
struct Four {
  int v[4];
};
__device__ __forceinline__ Four block_scan(const Four& x, int (*lds)[4], Four& all) {
  const int wave = threadIdx.x / vtx::kWave, lane = vtx::lane_id();
  Four r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int inc = (int)vtx::wave_prefix_sum((uint32_t)x.v[i]);
    if (lane == vtx::kWave - 1) lds[wave][i] = inc;
    r.v[i] = inc - x.v[i];
    all.v[i] = 0;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kPlanWaves; ++w)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int y = lds[w][i];
      r.v[i] += w < wave ? y : 0;
      all.v[i] += y;
    }
  return r;
}

// A stretch of a head's requests as the scan sees it: the run that its last
// request lies in.
struct Run {
  int start;   // first request of that run, -1: before the stretch
  int shared;  // minimum over the run's requests seen so far
};
__device__ __forceinline__ Run join(const Run& a, const Run& b) {
  return b.start >= 0 ? b : Run{a.start, min(a.shared, b.shared)};
}

// Chunks of up to `per` pages of n: their count, each of ceil(n / count) pages.
__device__ __forceinline__ uint32_t chunks(uint32_t n, uint32_t per, uint32_t& pages) {
  pages = 0;
  if (n == 0) return 0;
  const uint32_t c = (n + per - 1) / per;
  pages = c == 1 ? n : (n + c - 1) / c;
  return c == 1 ? 1 : (n + pages - 1) / pages;
}

constexpr int kLdsRequests = 2048;
// Requests up to which, in a table whose buffer has room for no more than one pass
// of entries a segment (the host does not know how many it holds), the second launch
// compares them itself (4 requests 8.3 us in two launches, 6.6 in one; 16 8.4 and
// 8.8, and a launch less of the host's time; 32 8.5 and 11.5).
constexpr int kFewRequests = 16;

// Per request of the head (a run's numbers at its first one), in LDS or in the plan.
struct Tables {
  int32_t *start, *pages, *first, *size, *shared, *run_items, *own_items, *run_rows, *own_rows, *apart;
};
__device__ __forceinline__ Tables tables_at(int32_t* p, int n) {
  return Tables{p,         p + n,     p + 2 * n,     p + 3 * n,     p + 4 * n, p + 5 * n,
                p + 6 * n + 1, p + 7 * n + 2, p + 8 * n + 2, p + 9 * n + 2};
}

// How a request's work is cut: its run's (counted at the first one) and its own.
struct Cut {
  uint32_t tiles, run_chunks, run_pages;
  uint32_t own_chunks, own_pages;
  int used, size;  // shared pages that are read once; the run's requests
  bool apart;      // with its three neighbours in one item
};

// kCompare: finds the common entries itself, kPlanWaves requests at a time.
template <bool kLds, bool kCompare>
__global__ __launch_bounds__(kPlanThreads) void prefix_plan_kernel(PlanArgs a) {
  __shared__ int32_t s_tables[kLds ? kScratchInts * kLdsRequests + 2 : 1];
  __shared__ int s_scan[kPlanWaves][4];
  __shared__ int s_run[kPlanWaves][2];
  __shared__ unsigned long long s_total[kPlanWaves];
  const int B = a.B, h = blockIdx.x, tid = threadIdx.x, wave = tid / vtx::kWave, lane = vtx::lane_id();
  const int each = (B + kPlanThreads - 1) / kPlanThreads;
  const int i0 = min(B, tid * each), i1 = min(B, i0 + each);
  int32_t* plan = a.plan;
  const Tables t = tables_at(kLds ? s_tables : plan + a.at.scratch + (int64_t)h * (kScratchInts * (int64_t)B + 2), B);

  // 1. What each request holds, and in `first` for now what it has in common
  // with the one before.
  for (int i = tid; i < B; i += kPlanThreads) {
    const int s = i * a.H + h;
    int start;
    t.pages[i] = pages_of(a, s, start);
    t.start[i] = start;
    if constexpr (!kCompare) t.first[i] = plan[a.at.common + s];
  }
  if constexpr (kCompare)
    for (int i = vtx::uniform(wave); i < B; i += kPlanWaves) {
      const int common = common_entries(a, i * a.H + h);
      if (lane == 0) t.first[i] = common;
    }
  __syncthreads();

  // 2. Runs, by a scan; a run's last request then has the run's minimum and
  // leaves (requests, shared pages) at its first.
  auto step = [&](int i) {
    const int limit = t.pages[i] - 1, c = t.first[i];
    return c < 0 ? Run{i, limit} : Run{-1, min(c, limit)};
  };
  Run mine{-1, 0x7fffffff};
  for (int i = i0; i < i1; ++i) mine = join(mine, step(i));
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
  const bool next_starts = i1 >= B || t.first[i1] < 0;  // (read before its thread writes over it)
  __syncthreads();
  Run at{-1, 0x7fffffff};
#pragma unroll
  for (int w = 0; w < kPlanWaves; ++w)
    if (w < wave) at = join(at, Run{s_run[w][0], s_run[w][1]});
  {
    const Run o{__shfl_up(inc.start, 1), __shfl_up(inc.shared, 1)};
    if (lane > 0) at = join(at, o);
  }
  for (int i = i0; i < i1; ++i) {
    at = join(at, step(i));
    t.first[i] = at.start;
    if (i + 1 < i1 ? t.first[i + 1] < 0 : next_starts) {
      const int n = i + 1 - at.start;
      t.size[at.start] = n;
      t.shared[at.start] = n > 1 ? max(0, at.shared) : 0;
    }
  }
  __syncthreads();

  // 3. What is shared; the work in tokens x row tiles, and from it the chunks.
  auto tiles_of = [&](int n) { return (uint32_t)(n * a.G + (1 << a.tile_shift) - 1) >> a.tile_shift; };
  auto used_of = [&](int e) { return (long long)e * a.P >= kMinShared ? e : 0; };
  unsigned long long work = 0;  // in pages
  for (int i0 = 0; i0 < B; i0 += kPlanThreads) {  // (all lanes: requests 4 j .. 4 j + 3 lie in one wave)
    const int i = i0 + tid;
    int own = 0;
    if (i < B) {
      const int s = i * a.H + h, f = t.first[i], e = t.shared[f], used = used_of(e);
      plan[a.at.leaders + s] = f;
      plan[a.at.shared + s] = e;
      if (f == i) work += (unsigned long long)tiles_of(t.size[f]) * used;
      own = t.pages[i] - used;
      work += (unsigned long long)own;
    }
    const uint64_t few = __ballot((long long)own * a.P <= a.apart), some = __ballot(own > 0);
    const int four = lane & ~3;
    if (i < B) t.apart[i] = (few >> four & 15) == 15 && __builtin_popcountll(some >> four & 15) > 1;
  }
#pragma unroll
  for (int d = 1; d < vtx::kWave; d <<= 1) work += __shfl_xor(work, d);
  if (lane == 0) s_total[wave] = work;
  __syncthreads();
  work = 0;
#pragma unroll
  for (int w = 0; w < kPlanWaves; ++w) work += s_total[w];
  // (rounded up: most_items counts on no fewer pages a chunk than work / slots)
  auto share = [&](int64_t parts) {
    const double x = (double)work / (double)parts * (1 + 1e-9) + 1;
    return (uint32_t)(x < 1e9 ? x : 1e9);
  };
  const uint32_t least = (uint32_t)(kMinChunk + a.P - 1) / (uint32_t)a.P;
  const uint32_t few = (uint32_t)(kFewChunk + a.P - 1) / (uint32_t)a.P;
  const uint32_t per = max(max(share(a.at.slots), least), min(share(a.at.cus), few));

  // 4. Items and partial rows of every request, and their places by a scan.
  auto cut = [&](int i) {
    Cut c;
    const int f = t.first[i];
    c.size = t.size[f];
    c.used = used_of(t.shared[f]);
    c.tiles = tiles_of(c.size);
    c.run_chunks = chunks(c.used, per, c.run_pages);
    c.own_chunks = chunks(t.pages[i] - c.used, per, c.own_pages);
    c.apart = t.apart[i];
    return c;
  };
  auto count_of = [&](int i, const Cut& c) {
    const bool head = t.first[i] == i, joined = c.run_chunks + c.own_chunks > 1;
    return Four{{head ? (int)(c.tiles * c.run_chunks) : 0, c.apart ? i % 4 == 0 : (int)c.own_chunks,
                 head ? c.size * a.G * (int)c.run_chunks : 0,
                 joined ? (int)c.own_chunks * a.G : 0}};  // (a single partial result is the result)
  };
  Four count{{0, 0, 0, 0}};
  for (int i = i0; i < i1; ++i) {
    const Four x = count_of(i, cut(i));
#pragma unroll
    for (int k = 0; k < 4; ++k) count.v[k] += x.v[k];
  }
  Four all;
  Four off = block_scan(count, s_scan, all);
  const int row0 = (int)(h * a.at.most_rows);
  off.v[2] += row0;
  off.v[3] += row0 + all.v[2];
  for (int i = i0; i < i1; ++i) {
    t.run_items[i] = off.v[0];
    t.own_items[i] = off.v[1];
    t.run_rows[i] = off.v[2];
    t.own_rows[i] = off.v[3];
    if (i + 1 < i1) {
      const Four x = count_of(i, cut(i));
#pragma unroll
      for (int k = 0; k < 4; ++k) off.v[k] += x.v[k];
    }
  }
  const int total = all.v[0] + all.v[1];
  const bool fits = total <= a.at.most_items;  // (always: slots and most_items belong together)
  if (tid == 0) {
    t.run_items[B] = all.v[0];
    t.own_items[B] = all.v[1];
    plan[a.at.counts + h] = fits ? total : 0;
  }
  __syncthreads();

  // 5. Where the combine launch finds a segment's partial rows.
  for (int i = tid; i < B; i += kPlanThreads) {
    const Cut c = cut(i);
    const int f = t.first[i];
    int4* to = reinterpret_cast<int4*>(plan + a.at.combine + (long long)kCombineInts * (i * a.H + h));
    to[0] = int4{t.run_rows[f] + (i - f) * a.G, (int)c.run_chunks, c.size * a.G, t.own_rows[i]};
    to[1] = int4{(int)c.own_chunks, t.start[i] + c.used, t.pages[i] - c.used, 0};
  }

  // 6. The items, every thread some of both kinds; the request by bisection.
  // Item k of head h is workgroup k * H + h of the attention, on XCD (k * H + h)
  // % 8: the head's items go round `rounds` XCDs, and each of these takes a
  // stretch of the runs' items, the row tiles of a chunk side by side in it, so
  // that a chunk's pages come into one L2 once.
  const int rounds = kXcds / ((a.H & -a.H) < kXcds ? (a.H & -a.H) : kXcds);
  const int stretch = all.v[0] / rounds, more = all.v[0] % rounds;
  Item* items = reinterpret_cast<Item*>(plan + a.at.items) + h * a.at.most_items;
  for (int k = tid; fits && k < total; k += kPlanThreads) {
    const bool run = k < all.v[0];
    const int x = k & (rounds - 1);
    const int32_t* list = run ? t.run_items : t.own_items;
    const int j = run ? x * stretch + min(x, more) + k / rounds : k - all.v[0];
    int lo = 0, hi = B;  // list[lo] <= j < list[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (list[mid] <= j) lo = mid;
      else hi = mid;
    }
    const int i = lo, in = j - list[i];
    const Cut c = cut(i);
    Item it;
    it.segment = i * a.H + h;
    int page0;
    if (run) {
      const int chunk = (uint32_t)in / c.tiles, tile = in - chunk * c.tiles, rows = c.size * a.G;
      it.row0 = tile << a.tile_shift;
      it.rows = min(rows - it.row0, 1 << a.tile_shift);
      page0 = chunk * c.run_pages;
      it.pages = min(c.used - page0, (int)c.run_pages);
      it.out = t.run_rows[i] + chunk * rows + it.row0;
    } else {
      it.row0 = 0;
      it.rows = a.G;
      page0 = c.used + in * c.own_pages;
      it.pages = min(t.pages[i] - page0, (int)c.own_pages);
      it.out = c.run_chunks + c.own_chunks > 1 ? t.own_rows[i] + in * a.G : -1;
    }
    it.start = t.start[i] + page0;
    it.last = page0 + it.pages == t.pages[i] ? 1 : 0;
    if (!run && c.apart) {
      it.pages = min(B - i, 4);
      it.last = kApart;
    }
    it.reserved = 0;
    items[k] = it;
  }
}

}  // namespace

namespace vtx_prefix {

Layout layout_of(int64_t batch, int64_t heads, int group_size, int head_dim, int cus) {
  Layout l;
  const int64_t segments = batch * heads, tile = tile_rows(head_dim);
  // All heads' items together: the workgroups that the device holds at a time.
  // (Twice as many, each half as long: 256 requests of 8 heads each behind 16k
  // tokens 165 us a layer for 158, 64 of 4 behind 32k 76 for 63: more partial
  // results.)
  const int64_t slots = cus * (head_dim == 64 ? 3 : 2);
  l.slots = (slots + heads - 1) / heads;
  l.cus = (cus + heads - 1) / heads;
  // Runs: tiles x ceil(pages / per) <= tiles x pages / per + tiles, at most one run
  // per two requests; requests: pages / per + 1 each.  The sums of x / per are at
  // most `slots` together.
  l.most_items = l.slots + batch + batch / 2 + batch * group_size / tile + 2;
  // n * G rows per chunk of a run (at most `tile` per tile), G per chunk of a request.
  l.most_rows = l.slots * tile + 2 * batch * group_size;
  int64_t at = kHeadInts;
  auto take = [&](int64_t n) {
    const int64_t r = at;
    at += (n + 7) / 8 * 8;  // (32-byte items)
    return r;
  };
  l.leaders = take(segments);
  l.shared = take(segments);
  l.combine = take(kCombineInts * segments);
  l.counts = take(heads);
  l.items = take((int64_t)(sizeof(Item) / sizeof(int32_t)) * l.most_items * heads);
  l.common = take(segments);
  l.scratch = take(batch > kLdsRequests ? kScratchInts * segments + 2 * heads : 0);
  l.size = at;
  return l;
}

}  // namespace vtx_prefix

extern "C" int64_t vtx_shared_prefix_plan_len(int32_t batch_size, int32_t num_kv_heads, int32_t group_size,
                                              int32_t head_dim) {
  const int cus = vtx::device_cu_count();
  if (batch_size < 0 || num_kv_heads < 1 || cus <= 0 || !vtx_paged_decode_attention_supported(head_dim, group_size))
    return 0;
  if ((int64_t)batch_size * num_kv_heads > kMaxSegments) return 0;
  return layout_of(batch_size, num_kv_heads, group_size, head_dim, cus).size;
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
  a.at = layout_of(batch_size, num_kv_heads, group_size, head_dim, cus);
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
  a.tile_shift = vtx::log2_exact(tile_rows(head_dim));
  a.apart = 2 * batch_size > a.at.slots ? short_tokens(head_dim) : 0;
  a.plan = plan;
  hipStream_t s = vtx::as_stream(stream);
  if (batch_size <= kFewRequests && kv_indices_len <= (int64_t)vtx::kWave * kAhead * S) {
    prefix_plan_kernel<true, true><<<num_kv_heads, kPlanThreads, 0, s>>>(a);
  } else {
    prefix_compare_kernel<<<(int)((S + kCompareWaves - 1) / kCompareWaves), kCompareWaves * vtx::kWave, 0, s>>>(a);
    if (batch_size <= kLdsRequests) prefix_plan_kernel<true, false><<<num_kv_heads, kPlanThreads, 0, s>>>(a);
    else prefix_plan_kernel<false, false><<<num_kv_heads, kPlanThreads, 0, s>>>(a);
  }
  return vtx::check_launch("plan_shared_prefix");
}
