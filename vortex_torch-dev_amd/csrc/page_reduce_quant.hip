// Page-finish reductions of keys (or values) held in 8 bits, for gfx950:
// page_reduce.hip's dim 1 over a pool of codes and factors (vtx_quant.h).  For
// every loc entry whose token closes a page and every kv head h, the P tokens of
// tile (loc / P) * H + h give one row of C statistics per output, rounded to
// bf16.  Codes times a power of two are bf16 values, and the rows are taken in
// page_reduce.hip's order, so the outputs are bit for bit those of the same
// reduction over a bf16 pool that holds the values.
//
// Bound by HBM for a burst of pages, by the launch and three dependent loads
// (loc, codes, output) for a decode step.  As there, a workgroup scans 256 loc
// entries and keeps the pages they close, and several share a block's tiles.  A
// wave takes tiles one at a time: lane = (row group, 8 columns), all of a
// 16-row tile's codes and factors loaded before the first is used.
#include <algorithm>

#include "vtx_device.h"
#include "vtx_host.h"
#include "vtx_page_reduce.h"
#include "vtx_quant.h"

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / vtx::kWave;
constexpr int kMaxShare = 16;  // workgroups that share one block of entries
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

template <int kCodes, int NEED>
__device__ __forceinline__ void add8(Acc (&acc)[8], const uint2& w, uint32_t byte, bool in) {
  const float s = vtx::factor(byte);
  float f[4];
  vtx::decode4<kCodes>(w.x, f);
#pragma unroll
  for (int e = 0; e < 4; ++e) vtx::acc_add_if<NEED>(acc[e], f[e] * s, in);
  vtx::decode4<kCodes>(w.y, f);
#pragma unroll
  for (int e = 0; e < 4; ++e) vtx::acc_add_if<NEED>(acc[4 + e], f[e] * s, in);
}

// C = 8 LPR, LPR | 64: page_reduce.hip's row groups (g: rows g, g + 64 / LPR, ..)
// and their fold.
template <int kCodes, int LPR, int NEED>
__global__ __launch_bounds__(kThreads) void reduce_quant_kernel(PageArgs a) {
  constexpr int kGroups = vtx::kWave / LPR;
  constexpr int kBatch = 16 / kGroups < 2 ? 2 : (16 / kGroups > 8 ? 8 : 16 / kGroups);
  __shared__ long long first_row[kThreads];
  __shared__ int wave_count[kWaves];
  const int pages = collect(a, first_row, wave_count);
  const int lane = vtx::lane_id(), grp = lane / LPR, cv = lane % LPR;
  const int wave = threadIdx.x / vtx::kWave;
  const int R = a.r.rows_per_tile, tiles = pages * a.r.heads;
  for (int t = blockIdx.y * kWaves + wave; t < tiles; t += gridDim.y * kWaves) {
    const long long row = first_row[t / a.r.heads] + (t % a.r.heads);
    if (!vtx::tile_in_range(a.r, row)) continue;
    const unsigned char* base = a.codes + row * (long long)R * a.r.cols + cv * 8;
    const unsigned char* sc = a.scales + row * (long long)R * 2;
    Acc acc[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) vtx::acc_init<NEED>(acc[e]);
    for (int r0 = grp; r0 < R; r0 += kBatch * kGroups) {
      uint2 w[kBatch];
      uint32_t b[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int r = r0 + u * kGroups, at = r < R ? r : R - 1;
        w[u] = *reinterpret_cast<const uint2*>(base + (long long)at * a.r.cols);
        b[u] = sc[2 * at];
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u) add8<kCodes, NEED>(acc, w[u], b[u], r0 + u * kGroups < R);
    }
#pragma unroll
    for (int d = LPR; d < vtx::kWave; d <<= 1)
#pragma unroll
      for (int e = 0; e < 8; ++e) vtx::acc_merge_xor<NEED>(acc[e], d);
    if (grp == 0) vtx::tile_store_vec(a.r, row, cv, acc);
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
        vtx::acc_add(acc, f[0] * vtx::factor(a.scales[(row * R + r) * 2]));
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

template <int kCodes, int LPR>
void launch_vec(const PageArgs& a, int need, dim3 grid, hipStream_t s) {
  switch (need) {
    case vtx::kNeedSum: reduce_quant_kernel<kCodes, LPR, vtx::kNeedSum><<<grid, kThreads, 0, s>>>(a); break;
    case vtx::kNeedMax: reduce_quant_kernel<kCodes, LPR, vtx::kNeedMax><<<grid, kThreads, 0, s>>>(a); break;
    case vtx::kNeedMin: reduce_quant_kernel<kCodes, LPR, vtx::kNeedMin><<<grid, kThreads, 0, s>>>(a); break;
    case vtx::kNeedMax | vtx::kNeedMin:
      reduce_quant_kernel<kCodes, LPR, vtx::kNeedMax | vtx::kNeedMin><<<grid, kThreads, 0, s>>>(a);
      break;
    default: reduce_quant_kernel<kCodes, LPR, vtx::kNeedAll><<<grid, kThreads, 0, s>>>(a); break;
  }
}

template <int kCodes>
void launch_codes(const PageArgs& a, int need, bool vec, dim3 grid, hipStream_t s) {
  const int lpr = a.r.cols / 8;
  if (vec && lpr == 8) launch_vec<kCodes, 8>(a, need, grid, s);
  else if (vec && lpr == 16) launch_vec<kCodes, 16>(a, need, grid, s);
  else if (vec && lpr == 32) launch_vec<kCodes, 32>(a, need, grid, s);
  else if (vec && lpr == 64) launch_vec<kCodes, 64>(a, need, grid, s);
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
  if (num_kv_heads > 0x7fffffff / kThreads) return vtx::fail(VTX_E_INVALID, "page_reduce_quant: too many heads");
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
  // One round of the workgroups' waves takes a block's tiles of whole pages where
  // sixteen can, and sixteen share a block while the grid is under 512
  // (page_reduce.hip has the reasons).
  const long long tiles = (page_size < kThreads ? kThreads / page_size : 1) * (long long)num_kv_heads;
  const long long share =
      std::min<long long>(std::max((tiles + kWaves - 1) / kWaves, (512 + blocks - 1) / blocks), kMaxShare);
  const dim3 grid((unsigned)blocks, (unsigned)share);
  const bool vec = cols % 8 == 0 && aligned;
  hipStream_t s = vtx::as_stream(stream);
  if (codes == VTX_CODES_E4M3) launch_codes<VTX_CODES_E4M3>(a, need, vec, grid, s);
  else launch_codes<VTX_CODES_INT8>(a, need, vec, grid, s);
  return vtx::check_launch("page_reduce_quant");
}
