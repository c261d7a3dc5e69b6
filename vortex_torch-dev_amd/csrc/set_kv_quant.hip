// Quantises new keys and values into 8-bit paged K / V pools, and reads such
// rows back, for gfx950.  The format: vtx_quant.h.
//
// Token i < nnz, kv head h: its key and value rows x go to pool row
// (loc / P) * (P * H) + h * P + loc % P, each as the codes of x 2^(127 - b), b
// from the row's largest absolute value; the two bytes b to that row of the
// exponents.  A token whose slot lies outside the pool is not stored.  Reading
// back gives code 2^(b - 127), rounded to the rows' type, zeros for such slots.
//
// Bound by memory (three operations per value): 65,536 tokens of 8 heads of 128
// bf16 columns 77 us (5.2 TB/s; a large copy reaches 4.9), 131,072 read back 163 us
// (5.0); by the launch for a step (one token 2.4 us).  A row's lanes take 8 columns
// each, of the key and of the value: the largest value is found among 2 to 64
// lanes by exchanges inside the wave, and both rows' loads are in flight at once.
// Rows of other widths or alignments take one wave each, an element a lane.
#include "vtx_device.h"
#include "vtx_host.h"
#include "vtx_quant.h"

namespace {

constexpr int kThreads = 256;
constexpr int kCols = 8;  // columns of a lane

struct QuantArgs {
  unsigned char* k;
  unsigned char* v;
  unsigned char* scales;
  unsigned char* nk;  // new rows, or the rows read back
  unsigned char* nv;
  const int64_t* loc;
  int64_t k_tok, k_head, v_tok, v_head;  // strides in elements
  int64_t last_page;
  uint32_t items;  // (token, head) pairs
  int32_t heads, D, page, page_shift;
};

// 8 columns of a row: their bits, and as fp32.
template <typename T>
struct Row8;
template <>
struct Row8<float> {
  vtx::U4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = vtx::ld16_stream(p);
    b = vtx::ld16_stream(p + 4);
  }
  __device__ __forceinline__ uint32_t amax() const {
    const uint32_t x = max(max(a.x & 0x7fffffffu, a.y & 0x7fffffffu), max(a.z & 0x7fffffffu, a.w & 0x7fffffffu));
    const uint32_t y = max(max(b.x & 0x7fffffffu, b.y & 0x7fffffffu), max(b.z & 0x7fffffffu, b.w & 0x7fffffffu));
    return max(x, y);
  }
  __device__ __forceinline__ void values(float (&f)[8]) const {
    const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(w[i]);
  }
  static __device__ __forceinline__ void store(float* p, const float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i += 4)
      vtx::st16(p + i, vtx::U4{__float_as_uint(f[i]), __float_as_uint(f[i + 1]), __float_as_uint(f[i + 2]),
                               __float_as_uint(f[i + 3])});
  }
};
// (two-byte types: bits of absolute values order as the values do)
__device__ __forceinline__ uint32_t amax16(const vtx::U4& a) {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  auto half = [](uint32_t w) { return __builtin_bit_cast(u16x2, w & 0x7fff7fffu); };
  const u16x2 m = __builtin_elementwise_max(__builtin_elementwise_max(half(a.x), half(a.y)),
                                            __builtin_elementwise_max(half(a.z), half(a.w)));
  return m.x > m.y ? m.x : m.y;
}
template <>
struct Row8<__bf16> {
  vtx::U4 a;
  __device__ __forceinline__ void load(const __bf16* p) { a = vtx::ld16_stream(p); }
  __device__ __forceinline__ uint32_t amax() const { return amax16(a) << 16; }
  __device__ __forceinline__ void values(float (&f)[8]) const { vtx::unpack8(a, f); }
  static __device__ __forceinline__ void store(__bf16* p, const float (&f)[8]) {
    vtx::st16(p, vtx::U4{vtx::bf16_pair(f[0], f[1]), vtx::bf16_pair(f[2], f[3]), vtx::bf16_pair(f[4], f[5]),
                         vtx::bf16_pair(f[6], f[7])});
  }
};
template <>
struct Row8<_Float16> {
  typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
  vtx::U4 a;
  __device__ __forceinline__ void load(const _Float16* p) { a = vtx::ld16_stream(p); }
  __device__ __forceinline__ uint32_t amax() const {  // (an infinity's and a NaN's bits stay those)
    return __float_as_uint((float)__builtin_bit_cast(_Float16, (uint16_t)amax16(a)));
  }
  __device__ __forceinline__ void values(float (&f)[8]) const {
    const f16x8 h = __builtin_bit_cast(f16x8, a);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (float)h[i];
  }
  static __device__ __forceinline__ void store(_Float16* p, const float (&f)[8]) {
    f16x8 h;
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = (_Float16)f[i];
    vtx::st16(p, __builtin_bit_cast(vtx::U4, h));
  }
};

struct alignas(8) U2 {
  uint32_t x, y;
};

template <int kCodes>
__device__ __forceinline__ U2 encode8(const float (&f)[8], uint32_t b) {
  const float s = vtx::inverse_factor(b);
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = b == 255u ? 0.f : f[i] * s;
  return U2{vtx::encode4<kCodes>(y[0], y[1], y[2], y[3]), vtx::encode4<kCodes>(y[4], y[5], y[6], y[7])};
}

// LPR lanes (a power of two) per (token, head), D = 8 columns of each or fewer.
template <typename T, int kCodes, int LPR>
__global__ __launch_bounds__(kThreads) void set_kv_quant_kernel(QuantArgs a) {
  const uint32_t it = (blockIdx.x * (uint32_t)kThreads + threadIdx.x) / LPR;
  const int c = (int)(threadIdx.x % LPR) * kCols;
  const bool mine = it < a.items && c < a.D;
  const uint32_t i = mine ? it / (uint32_t)a.heads : 0u;
  const int h = mine ? (int)(it - i * (uint32_t)a.heads) : 0;
  const long long row =
      mine ? vtx::pool_row(a.loc[i], h, a.heads, a.page, a.page_shift, a.last_page) : -1;
  Row8<T> k, v;
  uint32_t ka = 0, va = 0;
  if (row >= 0) {
    k.load(reinterpret_cast<const T*>(a.nk) + i * a.k_tok + h * a.k_head + c);
    v.load(reinterpret_cast<const T*>(a.nv) + i * a.v_tok + h * a.v_head + c);
    ka = k.amax();
    va = v.amax();
  }
#pragma unroll
  for (int d = 1; d < LPR; d <<= 1) {
    ka = max(ka, vtx::xshfl(ka, d));
    va = max(va, vtx::xshfl(va, d));
  }
  if (row < 0) return;
  const uint32_t kb = vtx::row_exponent<kCodes>(ka), vb = vtx::row_exponent<kCodes>(va);
  float f[8];
  k.values(f);
  *reinterpret_cast<U2*>(a.k + row * a.D + c) = encode8<kCodes>(f, kb);
  v.values(f);
  *reinterpret_cast<U2*>(a.v + row * a.D + c) = encode8<kCodes>(f, vb);
  if (c == 0) *reinterpret_cast<uint16_t*>(a.scales + row * 2) = (uint16_t)(kb | (vb << 8));
}

// Any width and alignment: one wave per (token, head), key and value one after
// the other, read twice (the second time from a cache).
template <typename T, int kCodes>
__global__ __launch_bounds__(kThreads) void set_kv_quant_any_kernel(QuantArgs a) {
  const uint32_t it = blockIdx.x * (uint32_t)(kThreads / vtx::kWave) + threadIdx.x / vtx::kWave;
  if (it >= a.items) return;  // uniform in a wave
  const int lane = vtx::lane_id();
  const uint32_t i = it / (uint32_t)a.heads;
  const int h = (int)(it - i * (uint32_t)a.heads);
  const long long row = vtx::pool_row(a.loc[i], h, a.heads, a.page, a.page_shift, a.last_page);
  if (row < 0) return;
  for (int part = 0; part < 2; ++part) {
    const T* x = part ? reinterpret_cast<const T*>(a.nv) + i * a.v_tok + h * a.v_head
                      : reinterpret_cast<const T*>(a.nk) + i * a.k_tok + h * a.k_head;
    unsigned char* y = (part ? a.v : a.k) + row * a.D;
    uint32_t m = 0;
    for (int c = lane; c < a.D; c += vtx::kWave) m = max(m, __float_as_uint((float)x[c]) & 0x7fffffffu);
#pragma unroll
    for (int d = 1; d < vtx::kWave; d <<= 1) m = max(m, vtx::xshfl(m, d));
    const uint32_t b = vtx::row_exponent<kCodes>(m);
    const float s = vtx::inverse_factor(b);
    for (int c = lane; c < a.D; c += vtx::kWave)
      y[c] = (unsigned char)vtx::encode4<kCodes>(b == 255u ? 0.f : (float)x[c] * s, 0.f, 0.f, 0.f);
    if (lane == 0) a.scales[row * 2 + part] = (unsigned char)b;
  }
}

template <typename T, int kCodes, int LPR>
__global__ __launch_bounds__(kThreads) void read_kv_quant_kernel(QuantArgs a) {
  const uint32_t it = (blockIdx.x * (uint32_t)kThreads + threadIdx.x) / LPR;
  const int c = (int)(threadIdx.x % LPR) * kCols;
  if (it >= a.items || c >= a.D) return;
  const uint32_t i = it / (uint32_t)a.heads;
  const int h = (int)(it - i * (uint32_t)a.heads);
  const long long row = vtx::pool_row(a.loc[i], h, a.heads, a.page, a.page_shift, a.last_page);
  U2 k{0u, 0u}, v{0u, 0u};
  uint32_t b = 0;
  if (row >= 0) {
    k = *reinterpret_cast<const U2*>(a.k + row * a.D + c);
    v = *reinterpret_cast<const U2*>(a.v + row * a.D + c);
    b = *reinterpret_cast<const uint16_t*>(a.scales + row * 2);
  }
  auto put = [&](const U2& w, uint32_t byte, T* to) {
    const float s = vtx::factor(byte);
    float f[8];
    float (&lo)[4] = *reinterpret_cast<float(*)[4]>(f), (&hi)[4] = *reinterpret_cast<float(*)[4]>(f + 4);
    vtx::decode4<kCodes>(w.x, lo);
    vtx::decode4<kCodes>(w.y, hi);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] *= s;
    Row8<T>::store(to, f);
  };
  put(k, b & 0xffu, reinterpret_cast<T*>(a.nk) + i * a.k_tok + h * a.k_head + c);
  put(v, b >> 8, reinterpret_cast<T*>(a.nv) + i * a.v_tok + h * a.v_head + c);
}

template <typename T, int kCodes>
__global__ __launch_bounds__(kThreads) void read_kv_quant_any_kernel(QuantArgs a) {
  const uint32_t it = blockIdx.x * (uint32_t)(kThreads / vtx::kWave) + threadIdx.x / vtx::kWave;
  if (it >= a.items) return;
  const uint32_t i = it / (uint32_t)a.heads;
  const int h = (int)(it - i * (uint32_t)a.heads);
  const long long row = vtx::pool_row(a.loc[i], h, a.heads, a.page, a.page_shift, a.last_page);
  for (int part = 0; part < 2; ++part) {
    T* y = part ? reinterpret_cast<T*>(a.nv) + i * a.v_tok + h * a.v_head
                : reinterpret_cast<T*>(a.nk) + i * a.k_tok + h * a.k_head;
    const float s = row >= 0 ? vtx::factor(a.scales[row * 2 + part]) : 0.f;
    for (int c = vtx::lane_id(); c < a.D; c += vtx::kWave) {
      float f[4] = {0.f, 0.f, 0.f, 0.f};
      if (row >= 0) vtx::decode4<kCodes>((part ? a.v : a.k)[row * a.D + c], f);
      y[c] = (T)(f[0] * s);
    }
  }
}

template <typename T, int kCodes, bool kRead, int LPR>
void launch_wide(const QuantArgs& a, hipStream_t s) {
  const uint32_t grid = (uint32_t)(((uint64_t)a.items * LPR + kThreads - 1) / kThreads);
  if constexpr (kRead) read_kv_quant_kernel<T, kCodes, LPR><<<grid, kThreads, 0, s>>>(a);
  else set_kv_quant_kernel<T, kCodes, LPR><<<grid, kThreads, 0, s>>>(a);
}

template <typename T, int kCodes, bool kRead>
int launch_type(const QuantArgs& all, int64_t items, bool wide, hipStream_t s) {
  // (items are counted in 32 bits, with their lanes: more tokens take several launches)
  const int64_t most = 0x1000000LL / all.heads > 0 ? 0x1000000LL / all.heads : 1;  // tokens
  const int64_t tokens = items / all.heads;
  for (int64_t i = 0; i < tokens; i += most) {
    QuantArgs a = all;
    a.items = (uint32_t)((tokens - i < most ? tokens - i : most) * all.heads);
    a.nk += i * a.k_tok * (int64_t)sizeof(T);
    a.nv += i * a.v_tok * (int64_t)sizeof(T);
    a.loc += i;
    const int lanes = (a.D + kCols - 1) / kCols;
    if (!wide) {
      const uint32_t grid = (a.items + kThreads / vtx::kWave - 1) / (kThreads / vtx::kWave);
      if constexpr (kRead) read_kv_quant_any_kernel<T, kCodes><<<grid, kThreads, 0, s>>>(a);
      else set_kv_quant_any_kernel<T, kCodes><<<grid, kThreads, 0, s>>>(a);
    } else if (lanes <= 8) {
      launch_wide<T, kCodes, kRead, 8>(a, s);
    } else if (lanes <= 16) {
      launch_wide<T, kCodes, kRead, 16>(a, s);
    } else if (lanes <= 32) {
      launch_wide<T, kCodes, kRead, 32>(a, s);
    } else {
      launch_wide<T, kCodes, kRead, 64>(a, s);
    }
    const int rc = vtx::check_launch(kRead ? "read_kv_buffer_quant" : "set_kv_buffer_quant");
    if (rc != VTX_OK) return rc;
  }
  return VTX_OK;
}

template <bool kRead>
int quant_impl(const char* what, void* k_cache, void* v_cache, void* scales, int64_t cache_rows, void* rows_k,
               void* rows_v, const int64_t* strides, const int64_t* loc, int64_t nnz, int32_t num_kv_heads,
               int32_t head_dim, int32_t dtype, int32_t codes, int32_t page_size, void* stream) {
  vtx::clear_error();
  if (nnz < 0 || num_kv_heads < 1 || head_dim < 1 || page_size < 1 || cache_rows < 0)
    return vtx::fail(VTX_E_INVALID, "%s: bad sizes", what);
  if (num_kv_heads > (1 << 24)) return vtx::fail(VTX_E_INVALID, "%s: too many heads", what);
  if (dtype != VTX_DTYPE_BF16 && dtype != VTX_DTYPE_F32 && dtype != VTX_DTYPE_F16)
    return vtx::fail(VTX_E_INVALID, "%s: unknown element type %d", what, dtype);
  if (codes != VTX_CODES_E4M3 && codes != VTX_CODES_INT8)
    return vtx::fail(VTX_E_INVALID, "%s: unknown codes %d", what, codes);
  if (nnz == 0) return VTX_OK;
  if (!k_cache || !v_cache || !scales || !rows_k || !rows_v || !loc || !strides)
    return vtx::fail(VTX_E_INVALID, "%s: null pointer", what);
  if (reinterpret_cast<uintptr_t>(scales) % 2)
    return vtx::fail(VTX_E_INVALID, "%s: scales must be 2-byte aligned", what);
  QuantArgs a;
  a.k = static_cast<unsigned char*>(k_cache);
  a.v = static_cast<unsigned char*>(v_cache);
  a.scales = static_cast<unsigned char*>(scales);
  a.nk = static_cast<unsigned char*>(rows_k);
  a.nv = static_cast<unsigned char*>(rows_v);
  a.loc = loc;
  a.k_tok = strides[0];
  a.k_head = strides[1];
  a.v_tok = strides[2];
  a.v_head = strides[3];
  a.last_page = cache_rows / ((int64_t)page_size * num_kv_heads) - 1;
  a.items = 0;
  a.heads = num_kv_heads;
  a.D = head_dim;
  a.page = page_size;
  a.page_shift = vtx::log2_exact(page_size);
  const int n = dtype == VTX_DTYPE_F32 ? 4 : 8;  // elements of 16 bytes
  const bool wide = head_dim % kCols == 0 && head_dim <= kCols * vtx::kWave && vtx::aligned16(rows_k) &&
                    vtx::aligned16(rows_v) && ((a.k_tok | a.k_head | a.v_tok | a.v_head) % n) == 0 &&
                    (reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) % 8 == 0;
  const int64_t items = nnz * num_kv_heads;
  hipStream_t s = vtx::as_stream(stream);
  auto go = [&](auto zero) {
    using T = decltype(zero);
    return codes == VTX_CODES_E4M3 ? launch_type<T, VTX_CODES_E4M3, kRead>(a, items, wide, s)
                                   : launch_type<T, VTX_CODES_INT8, kRead>(a, items, wide, s);
  };
  switch (dtype) {
    case VTX_DTYPE_F32: return go(0.f);
    case VTX_DTYPE_F16: return go((_Float16)0.f);
    default: return go((__bf16)0.f);
  }
}

}  // namespace

extern "C" int vtx_set_kv_buffer_quant(void* k_cache, void* v_cache, void* scales, int64_t cache_rows,
                                       const void* new_k, const void* new_v, const int64_t* strides,
                                       const int64_t* loc, int64_t nnz, int32_t num_kv_heads, int32_t head_dim,
                                       int32_t dtype, int32_t codes, int32_t page_size, void* stream) {
  return quant_impl<false>("set_kv_buffer_quant", k_cache, v_cache, scales, cache_rows, const_cast<void*>(new_k),
                           const_cast<void*>(new_v), strides, loc, nnz, num_kv_heads, head_dim, dtype, codes, page_size,
                           stream);
}

extern "C" int vtx_read_kv_buffer_quant(const void* k_cache, const void* v_cache, const void* scales,
                                        int64_t cache_rows, void* k_out, void* v_out, const int64_t* strides,
                                        const int64_t* loc, int64_t nnz, int32_t num_kv_heads, int32_t head_dim,
                                        int32_t dtype, int32_t codes, int32_t page_size, void* stream) {
  return quant_impl<true>("read_kv_buffer_quant", const_cast<void*>(k_cache), const_cast<void*>(v_cache),
                          const_cast<void*>(scales), cache_rows, k_out, v_out, strides, loc, nnz, num_kv_heads,
                          head_dim, dtype, codes, page_size, stream);
}
