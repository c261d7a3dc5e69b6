// Rotates new queries and keys to their positions and writes the new keys and
// values into the paged K / V pools for gfx950 (set_kv.hip with the position
// rotation on the way).
//
// For token i < nnz with table row (cos, sin) = cos_sin[positions[i]] and a
// query or key row x of rotary width R <= D, pair j < R / 2:
//   a' = a cos_j - b sin_j,  b' = b cos_j + a sin_j
// with (a, b) = (x[j], x[j + R/2]), or (x[2j], x[2j + 1]) interleaved; columns
// from R on stay.  fp32 arithmetic, one rounding to the rows' type.  Queries go
// to q_out, keys to pool row (loc / P) * (P * H) + h * P + loc % P of the K
// pool, values unchanged to the same row of the V pool.  A token whose pool row
// lies outside the pool stores nothing there (its queries are still rotated);
// one whose position lies outside the table is skipped altogether.
//
// Bound by memory (6 operations per pair): every row is read and written once
// (65,536 tokens of 16 + 2 x 8 heads of 128 bf16 columns: 204 us, 5.4 TB/s; one
// token 2.7 us).  A unit of work is two 16-byte vectors of one row, both halves
// of its pairs, so a pair's two columns meet in one thread and q_out may be q
// itself; rows of other widths or alignments take element-wide units, which are
// bound by their accesses (32,768 tokens of 16 + 2 x 8 heads of 80 columns, 40 of
// them rotated, 240 us, 1.4 TB/s; all 80 rotated, in vectors, 90 us, 3.8 TB/s).
#include "vtx_device.h"
#include "vtx_host.h"

namespace {

constexpr int kThreads = 256;

struct RopeArgs {
  const unsigned char* q;
  unsigned char* qo;
  const unsigned char* nk;
  const unsigned char* nv;
  unsigned char* kc;
  unsigned char* vc;
  const int64_t* loc;
  const int64_t* pos;
  const float* table;
  int64_t cache_rows, table_rows;
  int64_t last_page;  // the pool's last page, -1: none
  int64_t q_tok, q_head, qo_tok, qo_head, k_tok, k_head, v_tok, v_head;  // strides in elements
  uint32_t units, per_row, per_token;  // work units in all, of a row, of a token
  int32_t q_heads, heads, D, R, page;
};

// N consecutive elements of a row, as fp32.
template <typename T, int N>
struct Vec {
  T e[N];
};
template <typename T, int N>
__device__ __forceinline__ Vec<T, N> load(const T* p) {
  if constexpr (N * sizeof(T) == 16) {
    return __builtin_bit_cast(Vec<T, N>, vtx::ld16_stream(p));
  } else {
    static_assert(N == 1, "16 bytes or one element");
    return Vec<T, N>{{*p}};
  }
}
template <typename T, int N>
__device__ __forceinline__ void store(T* p, const Vec<T, N>& v) {
  if constexpr (N * sizeof(T) == 16) {
    vtx::st16(p, __builtin_bit_cast(vtx::U4, v));
  } else {
    *p = v.e[0];
  }
}

// One unit: columns c0 .. + N and c1 .. + N of row x, rotated (or copied) to row
// y.  Neighbouring threads take neighbouring vectors of one half and then of the
// other (8191 tokens of 32 + 2 x 4 fp16 heads, neighbouring pairs: two adjacent
// vectors a thread 44.0 us, this way 31.5; 65,536 of 16 + 2 x 8 222 and 204).
template <typename T, int N, bool kPairs>
__device__ __forceinline__ void unit(const RopeArgs& a, const T* x, T* y, const float* cs, int u, bool rotate) {
  const int half = a.R / 2, turned = !kPairs && rotate ? half / N : 0;  // units of both halves of pairs
  const bool rot = u < turned;
  int c0, c1;
  if (rot) {
    c0 = u * N;
    c1 = c0 + half;
  } else if (kPairs && N == 1) {
    c0 = 2 * u;
    c1 = c0 + 1;
  } else {  // the vectors of the other columns, first half and second half
    const int base = turned > 0 ? a.R : 0;
    c0 = base + (u - turned) * N;
    c1 = c0 + ((a.D - base) / N + 1) / 2 * N;
  }
  const bool two = c1 < a.D;
  Vec<T, N> va = load<T, N>(x + c0), vb = va;
  if (two) vb = load<T, N>(x + c1);
  // (interleaved with R a multiple of N only: the second vector may be past R)
  if constexpr (kPairs) {
    if (rotate && c0 < a.R) {
      if constexpr (N == 1) {
        const float p = (float)va.e[0], r = (float)vb.e[0], c = cs[c0 / 2], s = cs[half + c0 / 2];
        va.e[0] = (T)fmaf(p, c, -r * s);
        vb.e[0] = (T)fmaf(r, c, p * s);
      } else {
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          Vec<T, N>& v = w ? vb : va;
          const int c = w ? c1 : c0;
          if (c < a.R) {
#pragma unroll
            for (int j = 0; j < N / 2; ++j) {
              const float p = (float)v.e[2 * j], r = (float)v.e[2 * j + 1];
              const float co = cs[c / 2 + j], si = cs[half + c / 2 + j];
              v.e[2 * j] = (T)fmaf(p, co, -r * si);
              v.e[2 * j + 1] = (T)fmaf(r, co, p * si);
            }
          }
        }
      }
    }
  } else if (rot) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float p = (float)va.e[j], r = (float)vb.e[j], co = cs[c0 + j], si = cs[half + c0 + j];
      va.e[j] = (T)fmaf(p, co, -r * si);
      vb.e[j] = (T)fmaf(r, co, p * si);
    }
  }
  store<T, N>(y + c0, va);
  if (two) store<T, N>(y + c1, vb);
}

template <typename T, int N, bool kPairs>
__global__ __launch_bounds__(kThreads) void set_kv_rope_kernel(RopeArgs a) {
  const uint32_t it = blockIdx.x * (uint32_t)kThreads + threadIdx.x;
  if (it >= a.units) return;
  const uint32_t i = it / a.per_token, in_token = it - i * a.per_token;
  const int slot = (int)(in_token / a.per_row), u = (int)(in_token - slot * a.per_row);
  const long long at = a.pos[i];
  if (at < 0 || at >= a.table_rows) return;
  const float* cs = a.table + at * a.R;
  if (slot < a.q_heads) {
    const T* x = reinterpret_cast<const T*>(a.q) + i * a.q_tok + slot * a.q_head;
    T* y = reinterpret_cast<T*>(a.qo) + i * a.qo_tok + slot * a.qo_head;
    unit<T, N, kPairs>(a, x, y, cs, u, true);
    return;
  }
  const long long loc = a.loc[i];
  if (loc < 0) return;
  const long long page = loc / a.page;
  if (page > a.last_page) return;  // (first of all: a far page's row leaves 64 bits and may come back inside)
  const bool key = slot < a.q_heads + a.heads;
  const int h = slot - a.q_heads - (key ? 0 : a.heads);
  const long long row = page * ((long long)a.page * a.heads) + (long long)h * a.page + (loc - page * a.page);
  if (row >= a.cache_rows) return;
  const T* x = key ? reinterpret_cast<const T*>(a.nk) + i * a.k_tok + h * a.k_head
                   : reinterpret_cast<const T*>(a.nv) + i * a.v_tok + h * a.v_head;
  T* y = reinterpret_cast<T*>(key ? a.kc : a.vc) + row * a.D;
  unit<T, N, kPairs>(a, x, y, cs, u, key);
}

template <typename T, int N>
void launch(const RopeArgs& a, bool pairs, hipStream_t s) {
  const uint32_t grid = (a.units + kThreads - 1) / kThreads;
  if (pairs) set_kv_rope_kernel<T, N, true><<<grid, kThreads, 0, s>>>(a);
  else set_kv_rope_kernel<T, N, false><<<grid, kThreads, 0, s>>>(a);
}

template <typename T>
int launch_type(RopeArgs a, int64_t nnz, bool pairs, bool wide, hipStream_t s) {
  constexpr int N = 16 / (int)sizeof(T);
  a.per_row = (uint32_t)((a.D + 2 * (wide ? N : 1) - 1) / (2 * (wide ? N : 1)));
  a.per_token = a.per_row * (uint32_t)(a.q_heads + 2 * a.heads);
  // (units are counted in 32 bits: more tokens than that take several launches)
  const int64_t most = 0x7fffffffLL / a.per_token;
  for (int64_t i = 0; i < nnz; i += most) {
    RopeArgs b = a;
    b.units = (uint32_t)((nnz - i < most ? nnz - i : most) * a.per_token);
    b.q += i * a.q_tok * (int64_t)sizeof(T);
    b.qo += i * a.qo_tok * (int64_t)sizeof(T);
    b.nk += i * a.k_tok * (int64_t)sizeof(T);
    b.nv += i * a.v_tok * (int64_t)sizeof(T);
    b.loc += i;
    b.pos += i;
    if (wide) launch<T, N>(b, pairs, s);
    else launch<T, 1>(b, pairs, s);
    const int rc = vtx::check_launch("set_kv_buffer_rope");
    if (rc != VTX_OK) return rc;
  }
  return VTX_OK;
}

}  // namespace

extern "C" int vtx_set_kv_buffer_rope(void* k_cache, void* v_cache, int64_t cache_rows, const void* q, void* q_out,
                                      const void* new_k, const void* new_v, const int64_t* strides,
                                      const int64_t* loc, const int64_t* positions, const float* cos_sin,
                                      int64_t table_rows, int64_t nnz, int32_t q_heads, int32_t num_kv_heads,
                                      int32_t head_dim, int32_t rotary_dim, int32_t dtype, int32_t page_size,
                                      int32_t interleaved, void* stream) {
  vtx::clear_error();
  if (nnz < 0 || q_heads < 0 || num_kv_heads < 1 || head_dim < 1 || page_size < 1 || cache_rows < 0 || table_rows < 0)
    return vtx::fail(VTX_E_INVALID, "set_kv_buffer_rope: bad sizes");
  if (rotary_dim < 2 || rotary_dim % 2 || rotary_dim > head_dim)
    return vtx::fail(VTX_E_INVALID, "set_kv_buffer_rope: rotary_dim %d must be even and 2..head_dim", rotary_dim);
  if (dtype != VTX_DTYPE_BF16 && dtype != VTX_DTYPE_F32 && dtype != VTX_DTYPE_F16)
    return vtx::fail(VTX_E_INVALID, "set_kv_buffer_rope: unknown element type %d", dtype);
  if (((int64_t)q_heads + 2LL * num_kv_heads) * ((head_dim + 1) / 2) > 0x7fffffffLL)
    return vtx::fail(VTX_E_INVALID, "set_kv_buffer_rope: token too wide");
  if (nnz == 0) return VTX_OK;
  if (!k_cache || !v_cache || !new_k || !new_v || !loc || !positions || !cos_sin || !strides ||
      (q_heads > 0 && (!q || !q_out)))
    return vtx::fail(VTX_E_INVALID, "set_kv_buffer_rope: null pointer");
  RopeArgs a;
  a.q = static_cast<const unsigned char*>(q);
  a.qo = static_cast<unsigned char*>(q_out);
  a.nk = static_cast<const unsigned char*>(new_k);
  a.nv = static_cast<const unsigned char*>(new_v);
  a.kc = static_cast<unsigned char*>(k_cache);
  a.vc = static_cast<unsigned char*>(v_cache);
  a.loc = loc;
  a.pos = positions;
  a.table = cos_sin;
  a.cache_rows = cache_rows;
  a.table_rows = table_rows;
  a.last_page = cache_rows > 0 ? (cache_rows - 1) / ((int64_t)page_size * num_kv_heads) : -1;
  a.q_tok = q_heads > 0 ? strides[0] : 0;
  a.q_head = q_heads > 0 ? strides[1] : 0;
  a.qo_tok = q_heads > 0 ? strides[2] : 0;
  a.qo_head = q_heads > 0 ? strides[3] : 0;
  a.k_tok = strides[4];
  a.k_head = strides[5];
  a.v_tok = strides[6];
  a.v_head = strides[7];
  a.units = a.per_row = a.per_token = 0;
  a.q_heads = q_heads;
  a.heads = num_kv_heads;
  a.D = head_dim;
  a.R = rotary_dim;
  a.page = page_size;
  const int n = dtype == VTX_DTYPE_F32 ? 4 : 8;  // elements of 16 bytes
  bool wide = head_dim % n == 0 && (interleaved ? rotary_dim % n == 0 : (rotary_dim / 2) % n == 0) &&
              vtx::aligned16(k_cache) && vtx::aligned16(v_cache) && vtx::aligned16(new_k) && vtx::aligned16(new_v) &&
              (q_heads == 0 || (vtx::aligned16(q) && vtx::aligned16(q_out)));
  wide = wide && ((a.q_tok | a.q_head | a.qo_tok | a.qo_head | a.k_tok | a.k_head | a.v_tok | a.v_head) % n) == 0;
  hipStream_t s = vtx::as_stream(stream);
  switch (dtype) {
    case VTX_DTYPE_F32: return launch_type<float>(a, nnz, interleaved != 0, wide, s);
    case VTX_DTYPE_F16: return launch_type<_Float16>(a, nnz, interleaved != 0, wide, s);
    default: return launch_type<__bf16>(a, nnz, interleaved != 0, wide, s);
  }
}
