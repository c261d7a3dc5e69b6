// The 8-bit paged cache: codes (e4m3 or int8) of the K and V pools, and one
// exponent byte per token, kv head and pool.
//
// A row of head_dim values x is held as codes c and a byte b, x = c 2^(b - 127),
// with the least b by which the row's largest value fits the codes' largest (448
// or 127), and no less than 1.  Why a power of two: x / 2^(b - 127) is exact, so
// a value's code does not depend on how the quotient was taken; e4m3 loses
// nothing (its steps are as fine at every scale), int8 at most one bit of 8; and
// a factor is put together from its byte by one shift.  A row with a value that
// is not finite is held as zeros with b = 255, 2^128 in this arithmetic, an
// infinity: zero times it is not a number, in every kernel that reads the row.
#pragma once

#include "vtx_device.h"

namespace vtx {

// The exponent byte of a row by its largest absolute value (fp32 bits, not
// negative).  The exponent field E of that value less the codes' largest
// exponent, and one more where its mantissa is past that code's (1.75 of 448,
// 127 / 64 of 127): the addition carries into E exactly then.
template <int kCodes>
__device__ __forceinline__ uint32_t row_exponent(uint32_t amax) {
  if (amax >= 0x7f800000u) return 255u;
  const int e = kCodes == VTX_CODES_E4M3 ? (int)((amax + 0x1fffffu) >> 23) - 8 : (int)((amax + 0x1ffffu) >> 23) - 6;
  return (uint32_t)(e < 1 ? 1 : e);
}
// 2^(127 - b), by which a row is multiplied before it is rounded; 0 for b = 255
// (infinities and NaNs are not: the callers hold zeros for such rows).
__device__ __forceinline__ float inverse_factor(uint32_t b) {
  return b == 255u ? 0.f : __uint_as_float((254u - b) << 23);
}
// 2^(b - 127); 0 for b = 0, which no row is written with.
__device__ __forceinline__ float factor(uint32_t b) { return __uint_as_float(b << 23); }

// Four values within the codes' range, rounded to the nearest code (ties to
// even), packed in order.
template <int kCodes>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
  if constexpr (kCodes == VTX_CODES_E4M3) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
    return (uint32_t)w;
  } else {
    // 1.5 2^23 added: the sum's step is 1 and its low byte the value's
    const float m = 12582912.f;
    const uint32_t ab = __builtin_amdgcn_perm(__float_as_uint(b + m), __float_as_uint(a + m), 0x0c0c0400u);
    const uint32_t cd = __builtin_amdgcn_perm(__float_as_uint(d + m), __float_as_uint(c + m), 0x04000c0cu);
    return ab | cd;
  }
}

// The values of four packed codes.
template <int kCodes>
__device__ __forceinline__ void decode4(uint32_t w, float (&f)[4]) {
  if constexpr (kCodes == VTX_CODES_E4M3) {
    f[0] = __builtin_amdgcn_cvt_f32_fp8((int)w, 0);
    f[1] = __builtin_amdgcn_cvt_f32_fp8((int)w, 1);
    f[2] = __builtin_amdgcn_cvt_f32_fp8((int)w, 2);
    f[3] = __builtin_amdgcn_cvt_f32_fp8((int)w, 3);
  } else {
    f[0] = (float)(int8_t)(w & 0xffu);
    f[1] = (float)(int8_t)((w >> 8) & 0xffu);
    f[2] = (float)(int8_t)((w >> 16) & 0xffu);
    f[3] = (float)(int8_t)(w >> 24);
  }
}

// Packed codes as bf16 pairs, which hold every code: bytes 0 and 1, and 2 and 3.
template <int kCodes>
__device__ __forceinline__ void decode_pairs(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (kCodes == VTX_CODES_E4M3) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false);
    const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true);
    lo = __builtin_bit_cast(uint32_t, a);
    hi = __builtin_bit_cast(uint32_t, b);
  } else {
    float f[4];
    decode4<kCodes>(w, f);
    lo = __builtin_amdgcn_perm(__float_as_uint(f[1]), __float_as_uint(f[0]), 0x07060302u);
    hi = __builtin_amdgcn_perm(__float_as_uint(f[3]), __float_as_uint(f[2]), 0x07060302u);
  }
}

// The pool row ((page * H + h) * P + slot) of slot `pos` and head h, or -1 where
// it lies outside the pool of last_page + 1 pages (-1: none).
__device__ __forceinline__ long long pool_row(long long pos, int h, int heads, int page_size, int page_shift,
                                              long long last_page) {
  if (pos < 0) return -1;
  const long long page = page_shift >= 0 ? pos >> page_shift : pos / page_size;
  if (page > last_page) return -1;  // (before it is multiplied: a far page's row leaves 64 bits)
  return (page * heads + h) * page_size + (pos - page * page_size);
}

}  // namespace vtx
