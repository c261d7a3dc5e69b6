// Page-finish reductions of keys (or values) held in 8 bits, for gfx950:
// page_reduce.hip's dim 1 over a pool of codes and factors (vtx_quant.h).  For
// every loc entry whose token closes a page and every kv head h, the P tokens of
// tile (loc / P) * H + h give one row of C statistics per output, rounded to
// bf16.  Codes times a power of two are bf16 values, and the rows are taken in
// page_reduce.hip's order, so the outputs are bit for bit those of the same
// reduction over a bf16 pool that holds the values (e4m3 values under 2^-130 have
// bits that bf16 has not; they are added as they are) - but where rows are no numbers:
// Max and Min, which there pass a NaN by, are NaN, since a row with an infinity is held
// as NaN here, and a bound that left it out would not bound the page.
//
// Bound by HBM for a burst of pages (16,384 pages of 8 heads, Max + Min, 71 us, 4.8
// TB/s), by the launch and two dependent loads (loc, codes) for a decode step (64
// requests 3.5 us).  As there, a workgroup scans 256 loc entries and keeps the
// pages they close, and several share a block's tiles.  Few tiles: a wave takes one
// at a time, lane = (row group, 8 columns), the codes of 16 to 64 rows of a tile
// loaded before the first is used.  Many (of up to 16 rows): lane = (tile, 8
// columns), 64 / LPR tiles of a wave at a time, which a lane reduces alone, all its
// rows in flight and nothing between the lanes.
#include <algorithm>

#include "vtx_device.h"
#include "vtx_host.h"
#include "vtx_page_reduce.h"
#include "vtx_quant.h"

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / vtx::kWave;
constexpr int kMaxShare = 16;  // workgroups that share one block of entries; of few blocks twice as many
constexpr int kMostAtOnce = 2 * kMaxShare * kWaves * 8;  // tiles of them at a time, 8 of a wave
using vtx::Acc;

struct PageArgs {
  vtx::PageReduceArgs r;  // (r.x is not used)
  const unsigned char* codes;
  const unsigned char* scales;  // this pool's bytes, two apart
  int64_t last_page;
};

// vtx::collect_pages without the entries past the pool, however far they lie.
__device__ __forceinline__ int collect(const PageArgs& a, long long* first_row, int* wave_count) {
  const int lane = vtx::lane_id(), wave = threadIdx.x / vtx::kWave;
  const long long e = (long long)blockIdx.x * kThreads + threadIdx.x;
  long long page = -1;
  if (e < a.r.nnz) {
    const long long pos = a.r.loc[e];
    if (pos >= 0) {
      page = a.r.page_shift >= 0 ? pos >> a.r.page_shift : pos / a.r.page;
      if (page > a.last_page || pos - page * a.r.page != a.r.page - 1) page = -1;
    }
  }
  const uint64_t m = __ballot(page >= 0);
  if (lane == 0) wave_count[wave] = __popcll(m);
  __syncthreads();
  int before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    before += w < wave ? wave_count[w] : 0;
    total += wave_count[w];
  }
  if (page >= 0) first_row[before + vtx::lanes_below(m)] = page * a.r.heads;
  __syncthreads();
  return total;
}

// 8 codes, read once (ld16_stream says why).
__device__ __forceinline__ uint2 load8(const unsigned char* p) {
  typedef uint32_t v2u __attribute__((ext_vector_type(2)));
  const v2u t = __builtin_nontemporal_load(reinterpret_cast<const v2u*>(p));
  return uint2{t.x, t.y};
}

template <int kCodes, int NEED>
__device__ __forceinline__ void add8(Acc (&acc)[8], const uint2& w, uint32_t byte, bool in) {
  const float s = vtx::factor(byte);
  float f[4];
  vtx::decode4<kCodes>(w.x, f);
#pragma unroll
  for (int e = 0; e < 4; ++e) vtx::acc_add_if<NEED | vtx::kKeepNan>(acc[e], f[e] * s, in);
  vtx::decode4<kCodes>(w.y, f);
#pragma unroll
  for (int e = 0; e < 4; ++e) vtx::acc_add_if<NEED | vtx::kKeepNan>(acc[4 + e], f[e] * s, in);
}

// Row groups kG0 .. kG0 + kN - 1 (group g: rows g, g + G, ..., in order) of a lane's
// columns, folded pairwise as page_reduce.hip folds them: ((0 + 1) + (2 + 3)) + ..
template <int kCodes, int G, int kG0, int kN, int NEED>
__device__ __forceinline__ void fold_groups(const uint2 (&w)[16], const uint32_t (&b)[16], int R, Acc (&s)[8]) {
  if constexpr (kN == 1) {
#pragma unroll
    for (int e = 0; e < 8; ++e) vtx::acc_init<NEED>(s[e]);
#pragma unroll
    for (int r = kG0; r < 16; r += G) add8<kCodes, NEED>(s, w[r], b[r], r < R);
  } else {
    Acc lower[8];
    fold_groups<kCodes, G, kG0, kN / 2, NEED>(w, b, R, lower);
    fold_groups<kCodes, G, kG0 + kN / 2, kN / 2, NEED>(w, b, R, s);
#pragma unroll
    for (int e = 0; e < 8; ++e) vtx::acc_fold<NEED | vtx::kKeepNan>(lower[e], s[e]);
  }
}

// C = 8 LPR, LPR | 64: page_reduce.hip's row groups (g: rows g, g + 64 / LPR, ..)
// and their fold.  kBatch: rows of a group in flight; 0: a lane per column.
template <int kCodes, int LPR, int NEED, int kBatch>
__global__ __launch_bounds__(kThreads) void reduce_quant_kernel(PageArgs a) {
  constexpr int kGroups = vtx::kWave / LPR;
  __shared__ long long first_row[kThreads];
  __shared__ int wave_count[kWaves];
  const int pages = collect(a, first_row, wave_count);
  const int lane = vtx::lane_id(), grp = lane / LPR, cv = lane % LPR;
  const int wave = threadIdx.x / vtx::kWave;
  const int R = a.r.rows_per_tile, C = a.r.cols, tiles = pages * a.r.heads;
  constexpr int kAtOnce = kBatch == 0 ? kGroups : 1;
  for (int t0 = (blockIdx.y * kWaves + wave) * kAtOnce; t0 < tiles; t0 += gridDim.y * kWaves * kAtOnce) {
    const int t = kBatch == 0 ? t0 + grp : t0;
    if (t >= tiles) continue;
    const long long row = first_row[t / a.r.heads] + (t % a.r.heads);
    if (!vtx::tile_in_range(a.r, row)) continue;
    const unsigned char* base = a.codes + row * (long long)R * C + cv * 8;
    const unsigned char* sc = a.scales + row * (long long)R * 2;
    Acc acc[8];
    if constexpr (kBatch == 0) {
      uint2 w[16];
      uint32_t b[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int at = r < R ? r : R - 1;
        w[r] = load8(base + at * C);
        b[r] = sc[2 * at];
      }
      fold_groups<kCodes, kGroups, 0, kGroups, NEED>(w, b, R, acc);
      vtx::tile_store_vec(a.r, row, cv, acc);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) vtx::acc_init<NEED>(acc[e]);
      for (int r0 = grp; r0 < R; r0 += kBatch * kGroups) {
        uint2 w[kBatch];
        uint32_t b[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const int r = r0 + u * kGroups, at = r < R ? r : R - 1;
          w[u] = load8(base + (long long)at * C);
          b[u] = sc[2 * (long long)at];
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) add8<kCodes, NEED>(acc, w[u], b[u], r0 + u * kGroups < R);
      }
#pragma unroll
      for (int d = LPR; d < vtx::kWave; d <<= 1)
#pragma unroll
        for (int e = 0; e < 8; ++e) vtx::acc_merge_xor<NEED | vtx::kKeepNan>(acc[e], d);
      if (grp == 0) vtx::tile_store_vec(a.r, row, cv, acc);
    }
  }
}

// Any width: a lane per column, its rows in order.
template <int kCodes>
__global__ __launch_bounds__(kThreads) void reduce_quant_any_kernel(PageArgs a) {
  __shared__ long long first_row[kThreads];
  __shared__ int wave_count[kWaves];
  const int pages = collect(a, first_row, wave_count);
  const int wave = threadIdx.x / vtx::kWave;
  const int R = a.r.rows_per_tile, C = a.r.cols, tiles = pages * a.r.heads;
  for (int t = blockIdx.y * kWaves + wave; t < tiles; t += gridDim.y * kWaves) {
    const long long row = first_row[t / a.r.heads] + (t % a.r.heads);
    if (!vtx::tile_in_range(a.r, row)) continue;
    for (int c = vtx::lane_id(); c < C; c += vtx::kWave) {
      Acc acc;
      vtx::acc_init(acc);
      for (int r = 0; r < R; ++r) {
        float f[4];
        vtx::decode4<kCodes>(a.codes[(row * R + r) * C + c], f);
        vtx::acc_add<vtx::kNeedAll | vtx::kKeepNan>(acc, f[0] * vtx::factor(a.scales[(row * R + r) * 2]));
      }
#pragma unroll
      for (int o = 0; o < vtx::kPageReduceMaxOut; ++o)
        if (o < a.r.n_out) {
          const uint32_t bits = vtx::acc_value(acc, a.r.out_type[o], R);
          if (a.r.out_dtype[o] == VTX_DTYPE_BF16) reinterpret_cast<uint16_t*>(a.r.out[o])[row * C + c] = (uint16_t)bits;
          else reinterpret_cast<uint32_t*>(a.r.out[o])[row * C + c] = bits << 16;
        }
    }
  }
}

template <int kCodes, int LPR, int NEED>
void launch_need(const PageArgs& a, int at_once, dim3 grid, hipStream_t s) {
  constexpr int kGroups = vtx::kWave / LPR, kBatch = kGroups >= 8 ? 2 : 16 / kGroups > 8 ? 8 : 16 / kGroups;
  if constexpr (vtx::lane_tiles_fit(LPR, NEED)) {
    if (at_once > 1) {
      reduce_quant_kernel<kCodes, LPR, NEED, 0><<<grid, kThreads, 0, s>>>(a);
      return;
    }
  }
  // (taller tiles: more rows in flight, as far as registers allow)
  if (a.r.rows_per_tile > 16) reduce_quant_kernel<kCodes, LPR, NEED, 2 * kBatch><<<grid, kThreads, 0, s>>>(a);
  else reduce_quant_kernel<kCodes, LPR, NEED, kBatch><<<grid, kThreads, 0, s>>>(a);
}

constexpr int kEnvelope = vtx::kNeedMax | vtx::kNeedMin;
// Single reductions and Max + Min get their own code; other mixes accumulate every
// statistic.
constexpr int instance_need(int need) {
  return need == vtx::kNeedSum || need == vtx::kNeedMax || need == vtx::kNeedMin || need == kEnvelope ? need
                                                                                                     : vtx::kNeedAll;
}

template <int kCodes, int LPR>
void launch_vec(const PageArgs& a, int need, int at_once, dim3 grid, hipStream_t s) {
  switch (instance_need(need)) {
    case vtx::kNeedSum: launch_need<kCodes, LPR, vtx::kNeedSum>(a, at_once, grid, s); break;
    case vtx::kNeedMax: launch_need<kCodes, LPR, vtx::kNeedMax>(a, at_once, grid, s); break;
    case vtx::kNeedMin: launch_need<kCodes, LPR, vtx::kNeedMin>(a, at_once, grid, s); break;
    case kEnvelope: launch_need<kCodes, LPR, kEnvelope>(a, at_once, grid, s); break;
    default: launch_need<kCodes, LPR, vtx::kNeedAll>(a, at_once, grid, s); break;
  }
}

template <int kCodes>
void launch_codes(const PageArgs& a, int need, bool vec, int at_once, dim3 grid, hipStream_t s) {
  const int lpr = a.r.cols / 8;
  if (vec && lpr == 8) launch_vec<kCodes, 8>(a, need, at_once, grid, s);
  else if (vec && lpr == 16) launch_vec<kCodes, 16>(a, need, at_once, grid, s);
  else if (vec && lpr == 32) launch_vec<kCodes, 32>(a, need, at_once, grid, s);
  else if (vec && lpr == 64) launch_vec<kCodes, 64>(a, need, at_once, grid, s);
  else reduce_quant_any_kernel<kCodes><<<grid, kThreads, 0, s>>>(a);
}

}  // namespace

extern "C" int vtx_page_reduce_quant(const void* x, const void* scales, int64_t x_rows, int32_t page_size, int32_t cols,
                                     int32_t codes, int32_t n_out, void* const* outs, const int32_t* out_dtypes,
                                     const int32_t* reduce_types, int64_t out_rows, const int64_t* loc, int64_t nnz,
                                     int32_t num_kv_heads, void* stream) {
  vtx::clear_error();
  if (n_out < 1 || n_out > vtx::kPageReduceMaxOut || !outs || !out_dtypes || !reduce_types)
    return vtx::fail(VTX_E_INVALID, "page_reduce_quant: need 1..%d outputs", vtx::kPageReduceMaxOut);
  if (x_rows < 0 || out_rows < 0 || page_size < 1 || cols < 1 || num_kv_heads < 1 || nnz < 0)
    return vtx::fail(VTX_E_INVALID, "page_reduce_quant: bad sizes");
  if (codes != VTX_CODES_E4M3 && codes != VTX_CODES_INT8)
    return vtx::fail(VTX_E_INVALID, "page_reduce_quant: unknown codes %d", codes);
  // (a block's tiles, and a round of its workgroups past them, are counted in an int)
  if (num_kv_heads > (0x7fffffff - kMostAtOnce) / kThreads)
    return vtx::fail(VTX_E_INVALID, "page_reduce_quant: too many heads");
  PageArgs a;
  bool aligned = reinterpret_cast<uintptr_t>(x) % 8 == 0;
  int need = 0;
  for (int o = 0; o < vtx::kPageReduceMaxOut; ++o) {
    const bool used = o < n_out;
    a.r.out[o] = used ? outs[o] : nullptr;
    a.r.out_dtype[o] = used ? out_dtypes[o] : VTX_DTYPE_BF16;
    a.r.out_type[o] = used ? reduce_types[o] : VTX_REDUCE_MEAN;
    if (!used) continue;
    if (reduce_types[o] < VTX_REDUCE_MEAN || reduce_types[o] > VTX_REDUCE_L2NORM)
      return vtx::fail(VTX_E_INVALID, "page_reduce_quant: unknown reduce type %d", reduce_types[o]);
    if (out_dtypes[o] != VTX_DTYPE_BF16 && out_dtypes[o] != VTX_DTYPE_F32)
      return vtx::fail(VTX_E_INVALID, "page_reduce_quant: unknown output dtype %d", out_dtypes[o]);
    aligned = aligned && vtx::aligned16(outs[o]);
    need |= vtx::need_of(reduce_types[o]);
  }
  if (nnz == 0) return VTX_OK;
  if (!x || !scales || !loc) return vtx::fail(VTX_E_INVALID, "page_reduce_quant: null pointer");
  for (int o = 0; o < n_out; ++o)
    if (!outs[o]) return vtx::fail(VTX_E_INVALID, "page_reduce_quant: null output %d", o);
  const long long blocks = (nnz + kThreads - 1) / kThreads;
  if (blocks > 0x7fffffffLL) return vtx::fail(VTX_E_INVALID, "page_reduce_quant: loc too long");
  a.r.x = nullptr;
  a.r.x_rows = x_rows;
  a.r.rows_per_tile = page_size;
  a.r.cols = cols;
  a.r.n_out = n_out;
  a.r.out_rows = out_rows;
  a.r.loc = loc;
  a.r.nnz = nnz;
  a.r.heads = num_kv_heads;
  a.r.page = page_size;
  a.r.page_shift = vtx::log2_exact(page_size);
  a.codes = static_cast<const unsigned char*>(x);
  a.scales = static_cast<const unsigned char*>(scales);
  a.last_page = x_rows / num_kv_heads - 1;
  const bool vec = cols % 8 == 0 && aligned;
  // One round of the workgroups' waves takes a block's tiles of whole pages where
  // sixteen can, and sixteen share a block while the grid is under 512
  // (page_reduce.hip has the reasons); of up to 16 blocks, decode steps, 32, so that
  // no wave takes two tiles one after the other (8 heads, sixteen / 32: 256 entries
  // 7.6 / 5.1 us, Max + Min 9.1 / 5.8, 4096 9.6 / 7.0).
  const long long tiles = (page_size < kThreads ? kThreads / page_size : 1) * (long long)num_kv_heads;
  // Several tiles of a wave at a time pay where there are more than waves to take
  // them, earlier with two statistics, whose fold across lanes is longer; 256 columns
  // have two a wave, which gain nothing.  One at a time / several, Mean, 128 columns:
  // 8192 tiles 8.8 / 9.8 us, 16,384 14.0 / 12.7, 131,072 79.5 / 74.2; Max + Min: 4096
  // tiles 7.7 / 6.1, 131,072 108 / 72, 1024 of one head 4.4 / 5.8; 256 columns, Mean,
  // 131,072 122 / 130.  Two statistics of 1024 entries and more, of 8 heads, which may
  // be a burst's or a decode step's: a burst 4.2 / 5.6, of 2048 5.1 / 5.9, steps 6.7 /
  // 5.2 and 6.8 / 5.3, so several, which are never far off.
  const int lpr = cols / 8, stats = __builtin_popcount(instance_need(need));
  const bool lanes = vec && page_size <= 16 && (lpr == 8 || lpr == 16) &&
                     vtx::lane_tiles_fit(lpr, instance_need(need)) &&
                     (blocks * tiles >= (stats > 1 ? 4096 : 16384) || (stats > 1 && blocks >= 4 && tiles >= 64));
  const int at_once = lanes ? vtx::kWave / lpr : 1;
  const long long round = (tiles + kWaves * at_once - 1) / (kWaves * at_once);
  const long long share = std::min<long long>(std::max(round, (512 + blocks - 1) / blocks),
                                              blocks <= 16 ? 2 * kMaxShare : kMaxShare);
  const dim3 grid((unsigned)blocks, (unsigned)share);
  hipStream_t s = vtx::as_stream(stream);
  if (codes == VTX_CODES_E4M3) launch_codes<VTX_CODES_E4M3>(a, need, vec, at_once, grid, s);
  else launch_codes<VTX_CODES_INT8>(a, need, vec, at_once, grid, s);
  return vtx::check_launch("page_reduce_quant");
}
