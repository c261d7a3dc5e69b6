// Decode attention over an 8-bit paged cache (vtx_quant.h) for gfx950: one new
// token per request, grouped query heads, any block table.
//
// Segment s = b * H + h attends to its tokens t (the pages of its table range,
// the last of them partly filled); each of its G query heads gets
//   o = sum_t p_t v_t / sum_t p_t,  p_t = 2^(x_t - m),  x_t = log2 e f(scale q.k_t) - slope2 (n - 1 - t)
// over any partition of the tokens into parts with an m each; the parts join by
// weights 2^(m - max m).  f(y) = cap tanh(y / cap), or y.  Keys and values are
// k_t = kc_t 2^ek, v_t = vc_t 2^ev: codes, which bf16 holds exactly, and powers of
// two, which multiply the scores and the weights.
//
// Both products run on the matrix cores (v_mfma_f32_16x16x32_bf16), transposed so
// that a lane holds one query head: S^T = K Q^T leaves lane l with head l % 16 and
// tokens 4 (l / 16) .. + 4 of 16, so the softmax stays in the lane, and two such
// tiles' weights are the B operand of O^T = V^T P^T as they stand, if V^T takes
// its tokens in the same order: a lane loads D / 16 codes of eight tokens and
// transposes them by byte permutations on their way to bf16.  So K and V go from
// memory to registers to the matrix cores: no LDS, no barriers among the waves.
// Weights go in as two bf16 values, their rounding and what it left (2^-17 of a
// weight), and fp16 queries likewise (exactly): the matrix cores have time, the
// launch waits for memory.
//
// 4 waves per workgroup (one where segments are many and tiny), 32 tokens of a wave
// at a time; the next ones' keys are requested behind the scores and their values
// behind the weighted sum, into the registers that these leave, and the next
// segment's first ones before the waves' results are joined.  How a table's pages
// are divided among workgroups: divide_pages, ranges_of; a segment that lies in
// several has its parts joined by a second launch.
//
// Bound by HBM where there are many tokens (32 requests of up to 32k, 8 x 8 heads of
// 128 columns, 213 us, 5.8 TB/s; a large copy, which writes half of it, reaches 4.9 to
// 5.0), by five dependent trips to memory and the second launch where there are few
// (one request of 4096 tokens 12.0 us, of 128, in one launch, 6.1).
#include <algorithm>
#include <cfloat>

#include "vtx_device.h"
#include "vtx_host.h"
#include "vtx_quant.h"

namespace {

constexpr int kAllWaves = 4;     // of a workgroup, but where segments are many and tiny (ranges_of): 1
constexpr int kHeads = 16;       // query heads of a matrix tile
constexpr int kTile = 32;        // tokens of a wave at a time
constexpr int kStage = 1024;     // page rows staged in LDS at a time
constexpr int kBounds = 1024;    // bounds of a table that are brought to LDS whole
constexpr int kMinTokens = 128;  // tokens of a range at least: a tile per wave
constexpr int kTiny = 256;       // tokens of a tiny segment
constexpr float kLog2e = 1.4426950408889634f;

// A divisor that the host knows: three scalar instructions and two corrections
// for the compiler's division by an unknown, which takes a tenth of a microsecond
// where nothing runs beside it.
struct Divisor {
  uint32_t d, m;  // m: 2^32 / d, rounded down (2^32 - 1 for 1)
};
__device__ __forceinline__ uint32_t divide(uint32_t x, Divisor v) {
  uint32_t q = __umulhi(x, v.m), r = x - q * v.d;  // (one or two too small)
  if (r >= v.d) {
    ++q;
    r -= v.d;
  }
  return r >= v.d ? q + 1 : q;
}
inline Divisor divisor(long long d) {
  return Divisor{(uint32_t)d, d == 1 ? 0xffffffffu : (uint32_t)((1LL << 32) / d)};
}

struct QAttnArgs {
  const uint16_t* q;
  uint16_t* o;
  const unsigned char* k;
  const unsigned char* v;
  const unsigned char* scales;
  int64_t rows;  // pool rows (page * H + h)
  const int32_t* indptr;
  const int32_t* indices;
  int64_t indices_len;
  const int32_t* last_len;
  const float* slopes;  // [H * G], or null
  int64_t q_batch, q_kv, q_head;  // strides in elements
  int32_t segments, H, G, P, p_shift;
  bool tiny;               // a wave each
  bool balanced;           // no compute unit has much more than its share of the segments
  Divisor by_segments, by_heads, by_slots, by_cus, by_least, by_pitch;
  int32_t window;  // the last tokens that count; 0: all
  int32_t pitch;   // places of a segment on a spaced line; 0: the line is another
  float c;         // scale log2 e
  float cap;       // cap log2 e, or 0
  float by_cap;    // 1 over that
  int32_t workers, slots;  // workgroups (0: one per segment), and how many of them the card holds
  int32_t least;           // pages of a range
  int32_t join;            // (head, four columns) of a joining workgroup
  float* acc;       // [2 slots, G, D]
  float2* ml;       // [2 slots, G]
  int32_t* places;  // [segments + 1], of a packed line
};

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// How a table's pages are divided, from their total alone.
//
// Few long segments: all pages in a line, one segment's after another's, and a
// range of the line for each workgroup that the card holds, whole tiles of all
// waves; where the pages divide evenly among the segments a whole part of one, if
// that costs the fullest compute unit no more than a quarter (fewer parts to join,
// and a workgroup's waves start over less often).  A workgroup meets the segments
// of its range one after another.
//
// Short segments, or many equal ones (chunk > 0): a workgroup each, and those longer
// than a chunk, twice a workgroup's share and 1024 tokens at least, are cut into
// equal parts, the first with that workgroup, the others with workgroups behind the
// segments'.  Many uneven long ones stay on the line, which evens them out.
// Line / chunks, 128 columns: 512 segments of up to 64 tokens 18.5 / 9.7 us, of up to
// 1024 34.9 / 27.3, of up to 4096 66 / 75; 512 of 512 tokens each 21.2 / 20.0, 1024 of
// 2048 109 / 96, 2048 of 512 62 / 56.  (Where single requests of a few tokens lie among
// long ones the line is the slower one: ranges_of has figures.)
struct Division {
  uint32_t per;    // pages of a range
  uint32_t chunk;  // pages of a part at most; 0: ranges
};
__device__ __forceinline__ Division divide_pages(const QAttnArgs& a, uint32_t total) {
  const uint32_t even = divide(total + (uint32_t)a.slots - 1u, a.by_slots), least = (uint32_t)a.least;
  const uint32_t S = (uint32_t)a.segments, m = divide(total, a.by_segments);
  const uint32_t mean = m + (m * S < total ? 1u : 0u);
  if (a.tiny || mean < least || (mean < 2u * even && (mean <= 8u * least || (a.balanced && m * S == total))))
    return Division{even, max(max(2u * even, 8u * least), mean)};
  Division v{divide(max(even, least) + least - 1u, a.by_least) * least, 0u};
  if (m >= v.per && m * S == total) {
    const uint32_t many = m / v.per, per = (m - 1u) / many + 1u;  // ranges of a segment
    const uint64_t fullest = (uint64_t)(divide(S * many - 1u, a.by_cus) + 1u) * per;
    if (4 * fullest <= 5 * (uint64_t)(divide(total - 1u, a.by_cus) + 1u)) v.per = per;
  }
  return v;
}
// Parts of a segment of so many pages.
__device__ __forceinline__ uint32_t parts_of(int pages, uint32_t chunk) {
  return (uint32_t)pages <= chunk ? 1u : ((uint32_t)pages - 1u) / chunk + 1u;
}
__device__ __forceinline__ uint32_t table_pages(const QAttnArgs& a, int first, int end) {
  const uint32_t all = end > first ? (uint32_t)end - (uint32_t)first : 0u, len = (uint32_t)a.indices_len;
  return all < len ? all : len;
}

// A segment's pages that count.
struct Segment {
  int start;          // of them, in the table
  int pages, tokens;  // tokens from the first of these pages on, the last page's included
  int skip;           // tokens of the first page that the window leaves out
  bool over;          // more tokens than an int counts, with the requests past the end: none of them do
};
__device__ __forceinline__ Segment segment_of(const QAttnArgs& a, int p0, int p1, int last) {
  Segment g{p0, 0, 0, 0, false};
  if (p0 >= 0 && p1 > p0 && (int64_t)p1 <= a.indices_len && a.rows > 0) {
    last = last < 0 ? 0 : (last > a.P ? a.P : last);
    const long long n = (long long)(p1 - p0 - 1) * a.P + last;
    g.over = n >= (1LL << 30);
    if (n > 0 && !g.over) {
      g.pages = p1 - p0;
      g.tokens = (int)n;
      if (a.window > 0 && g.tokens > a.window) {
        const int lo = g.tokens - a.window, pg = a.p_shift >= 0 ? lo >> a.p_shift : lo / a.P;
        g.start += pg;
        g.pages -= pg;
        g.tokens -= pg * a.P;
        g.skip = lo - pg * a.P;
      }
    }
  }
  return g;
}

// Its place on the line: [at, end), both 0 where it has none.
struct Place {
  uint32_t at, end;
};
__device__ __forceinline__ Place place_of(const Segment& g, uint32_t at, uint32_t total) {
  const bool ok = g.pages > 0 && at < total && (uint32_t)g.pages <= total - at;
  return ok ? Place{at, at + (uint32_t)g.pages} : Place{0u, 0u};
}

__device__ __forceinline__ uint32_t parts_at(const QAttnArgs& a, int s, uint32_t chunk) {
  return parts_of(segment_of(a, a.indptr[s], a.indptr[s + 1], a.last_len[s]).pages, chunk);
}
// A thread's sum of parts, held below kMostParts, which is more than there are rows
// for (ranges_of: a few thousand): in a table that decreases segments overlap, their
// parts are any number, and 32 bits of a workgroup's sum are to hold it all the same.
constexpr uint32_t kMostParts = 1u << 22;
__device__ __forceinline__ uint32_t add_parts(uint32_t sum, uint32_t n) { return min(sum + n, kMostParts); }
// The parts of the cut segments before segment s.  Every thread of the workgroup
// calls it; sums: LDS, an entry per wave.
template <int T>
__device__ __forceinline__ uint32_t parts_before(const QAttnArgs& a, int s, uint32_t chunk, float* sums) {
  uint32_t mine = 0;
  for (int j = threadIdx.x; j < s; j += T) {
    const uint32_t n = parts_at(a, j, chunk);
    mine = add_parts(mine, n > 1u ? n : 0u);
  }
  mine = vtx::wave_sum(mine);
  if (vtx::lane_id() == 0) sums[threadIdx.x / vtx::kWave] = __uint_as_float(mine);
  __syncthreads();
  uint32_t all = 0;
#pragma unroll
  for (int i = 0; i < T / vtx::kWave; ++i) all += __float_as_uint(sums[i]);
  return (uint32_t)vtx::uniform((int)all);
}

// How many of the segments end at or before place v0 of the line, which is the
// number of the first that does not: every wave by itself, 64 bounds at a time.
// bound(j): the table's j-th.
template <typename Bound>
__device__ __forceinline__ int segments_before(int S, int first, uint32_t v0, Bound bound) {
  int lo = 0, len = S;
  while (true) {
    const int step = (len + vtx::kWave - 1) / vtx::kWave;  // (0: nothing left)
    const int j = lo + (vtx::lane_id() + 1) * step;
    const bool in = step > 0 && j <= lo + len;
    const int p = bound(in ? j : 0);
    const uint64_t m = __ballot(in && (p <= first || (uint32_t)p - (uint32_t)first <= v0));
    // (as many as the first bound past v0 leaves, also of a table that decreases)
    const int c = m == ~0ull ? vtx::kWave : __builtin_ctzll(~m);
    lo += c * step;
    if (step <= 1) return vtx::uniform(lo);
    len = min(step - 1, S - lo);
  }
}

// What a wave holds of 16 query heads: running maximum (base 2), sum (of this
// lane's tokens) and output.
template <int kD>
struct Heads {
  float m, l;
  f32x4 o[kD / 16];
};

// The heads' fragments: bf16 ones in registers, a copy in every wave; fp16 ones,
// twice as many, in LDS, one copy for all waves (in registers they spilled: 128
// columns, 32 requests of up to 8k tokens 77 us, so 66; bf16 ones in LDS cost 1 us
// of 65).  After the tiles the waves' outputs take their place there.
template <int kD, bool kHalf, int kWaves>
struct Queries {
  static constexpr int kOwn = kHalf ? (kD / 32 + kWaves - 1) / kWaves : kD / 32;  // of a wave
  vtx::U4 raw[kOwn];
};
template <int kD, bool kHalf, int kWaves>
struct Shared {
  static constexpr int kOut = kD + 4;  // floats of a head's outputs: 16 heads' pieces in all banks
  union {
    vtx::U4 q[kHalf ? 2 : 1][kHalf ? kD / 32 : 1][vtx::kWave];  // rounded to bf16, and what that left
    float o[kWaves][kHeads][kOut];
  };
};

// 32 tokens' keys on their way, and their values and factors.
template <int kD>
struct Keys {
  vtx::U4 k[2][kD / 64];
};
template <int kD>
struct Values {
  uint32_t v[2][4][kD / 64];  // 16-token half, token, codes
  uint2 sc[2];                // (K, V) bytes of this lane's four tokens of a half
};

// Loads of 16 tokens of one page by buffer loads: a lane's place among them is a
// constant register, the tokens' address a scalar, and tokens past `bytes` cost
// nothing and read as zeros, so the loop's loads stand behind no branch.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const unsigned char* p, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, (int)bytes, 0x27000);
}
constexpr int kStream = 2;  // read once: the non-temporal hint
template <int N>
__device__ __forceinline__ void load_words(__amdgpu_buffer_rsrc_t r, int at, uint32_t (&to)[N]) {
  if constexpr (N == 1) {
    to[0] = __builtin_amdgcn_raw_buffer_load_b32(r, at, 0, kStream);
  } else if constexpr (N == 2) {
    const auto t = __builtin_amdgcn_raw_buffer_load_b64(r, at, 0, kStream);
    to[0] = t[0];
    to[1] = t[1];
  } else {
    const auto t = __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, kStream);
    to[0] = t[0];
    to[1] = t[1];
    to[2] = t[2];
    to[3] = t[3];
  }
}

template <int kD>
__device__ __forceinline__ void load_v(const unsigned char* p, uint32_t (&to)[kD / 64]) {
  if constexpr (kD == 64) {
    to[0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(p));
  } else if constexpr (kD == 128) {
    typedef uint32_t v2u __attribute__((ext_vector_type(2)));
    const v2u t = __builtin_nontemporal_load(reinterpret_cast<const v2u*>(p));
    to[0] = t.x;
    to[1] = t.y;
  } else {
    const vtx::U4 t = vtx::ld16_stream(p);
    to[0] = t.x;
    to[1] = t.y;
    to[2] = t.z;
    to[3] = t.w;
  }
}

// The growth of a score over the running maximum (base 2) from which on that
// follows: until then weights of up to 2^8 are as exact as those of up to 1, and
// the outputs stay as they are.
constexpr float kGrowth = 8.f;

// Scores of 32 tokens, without their factors.
template <int kD, int kCodes, bool kHalf, int kWaves>
__device__ __forceinline__ void score(const Shared<kD, kHalf, kWaves>& sh, const Queries<kD, kHalf, kWaves>& own,
                                      const Keys<kD>& t, f32x4 (&s)[2]) {
  int lane = vtx::lane_id();
  if constexpr (kHalf) asm volatile("" : "+v"(lane));  // (read for every tile: kept out of the registers)
#pragma unroll
  for (int h = 0; h < 2; ++h) s[h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < kD / 64; ++j) {
    vtx::U4 q[kHalf ? 4 : 2];
#pragma unroll
    for (int e = 0; e < (kHalf ? 4 : 2); ++e) {
      if constexpr (kHalf) q[e] = sh.q[e / 2][2 * j + e % 2][lane];
      else q[e] = own.raw[2 * j + e];
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      vtx::U4 f0, f1;
      vtx::decode_pairs<kCodes>(t.k[h][j].x, f0.x, f0.y);
      vtx::decode_pairs<kCodes>(t.k[h][j].y, f0.z, f0.w);
      vtx::decode_pairs<kCodes>(t.k[h][j].z, f1.x, f1.y);
      vtx::decode_pairs<kCodes>(t.k[h][j].w, f1.z, f1.w);
      auto mul = [&](const vtx::U4& k, const vtx::U4& x) {
        s[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, k), __builtin_bit_cast(bf16x8, x),
                                                       s[h], 0, 0, 0);
      };
      mul(f0, q[0]);
      mul(f1, q[1]);
      if constexpr (kHalf) {
        mul(f0, q[2]);
        mul(f1, q[3]);
      }
    }
  }
}

// cap tanh(y / cap), to 2^-20 of itself whatever the cap, with z = y / cap: under 0.75
// by five terms of Lambert's continued fraction of tanh(z) / z, (1 + u / 9 + u^2 / 945)
// / (1 + 4 u / 9 + u^2 / 63) with u = z^2 (2^-27 off), which is 1 for a cap that nothing
// comes near; from there on by (e - 1) / (e + 1), e = 2^(2 z log2 e), where e - 1 loses
// nothing that counts.  A NaN stays one.  cap - 2 cap / (e + 1) is shorter and off by
// 2^-22 of the cap, however small y is: 48 requests of up to 8k tokens, 256 columns,
// 68.0 us, so 68.8; skipped where no score of a tile needs e, 68.6.
__device__ __forceinline__ float capped(float y, float cap, float by_cap) {
  const float z = y * by_cap, u = z * z;
  const bool small = !(fabsf(z) >= 0.75f);
  const float e = __builtin_amdgcn_exp2f(fminf(fmaxf(z, -12.f), 12.f) * (2.f * kLog2e));
  const float n = small ? fmaf(u, fmaf(u, 1.f / 945.f, 1.f / 9.f), 1.f) : e - 1.f;
  const float d = small ? fmaf(u, fmaf(u, 1.f / 63.f, 4.f / 9.f), 1.f) : e + 1.f;
  return (small ? y : cap) * (n * __builtin_amdgcn_rcpf(d));
}

// Their weights, and the values by these.  bad: tokens of this lane that do not
// count (where masked); far: the distance of its first one; slope: base 2.
template <int kD, int kCodes>
__device__ __forceinline__ void attend(const QAttnArgs& a, Heads<kD>& w, const f32x4 (&s)[2], Values<kD>& t,
                                       bool masked, uint32_t bad, float far, float slope) {
  if (masked) {  // uniform
    // tokens that do not count may be anything, NaN too: their values become zeros
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool out = (bad >> (4 * h + i)) & 1u;
#pragma unroll
        for (int x = 0; x < kD / 64; ++x) t.v[h][i][x] = out ? 0u : t.v[h][i][x];
      }
      t.sc[h].x &= ((bad >> (4 * h)) & 1u ? 0u : 0xffffu) | ((bad >> (4 * h + 1)) & 1u ? 0u : 0xffff0000u);
      t.sc[h].y &= ((bad >> (4 * h + 2)) & 1u ? 0u : 0xffffu) | ((bad >> (4 * h + 3)) & 1u ? 0u : 0xffff0000u);
    }
  }
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t two = (i & 2) ? t.sc[i / 4].y : t.sc[i / 4].x;
    const uint32_t bits = (i & 1) ? (two << 7) & 0x7f800000u : (two << 23) & 0x7f800000u;
    x[i] = s[i / 4][i % 4] * (a.c * __uint_as_float(bits));
  }
  if (a.cap != 0.f) {  // uniform
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = capped(x[i], a.cap, a.by_cap);
  }
  if (a.slopes) {  // uniform
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = fmaf(-slope, far - (float)(16 * (i / 4) + i % 4), x[i]);
  }
  if (masked) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (bad >> i) & 1u ? -INFINITY : x[i];
  }
  float mx = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
  if (__ballot(mx > w.m + kGrowth)) {  // uniform
    mx = fmaxf(mx, vtx::xshfl(mx, 16));
    mx = fmaxf(mx, vtx::xshfl(mx, 32));
    const float nm = fmaxf(w.m, mx);
    const float f = nm == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(w.m - nm);
    w.l *= f;
#pragma unroll
    for (int d = 0; d < kD / 16; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) w.o[d][i] *= f;
    w.m = nm;
  }
  const float base = w.m == -INFINITY ? 0.f : w.m;
  uint32_t hi[4], lo[4];
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const uint32_t two = (i & 2) ? t.sc[i / 4].y : t.sc[i / 4].x;
    const float p0 = __builtin_amdgcn_exp2f(x[i] - base), p1 = __builtin_amdgcn_exp2f(x[i + 1] - base);
    w.l += p0 + p1;
    const float w0 = p0 * __uint_as_float((two << 15) & 0x7f800000u);
    const float w1 = p1 * __uint_as_float((two >> 1) & 0x7f800000u);
    hi[i / 2] = vtx::bf16_pair(w0, w1);
    lo[i / 2] = vtx::bf16_pair(w0 - vtx::bf16_lo(hi[i / 2]), w1 - vtx::bf16_hi(hi[i / 2]));
  }
  const bf16x8 bh = __builtin_bit_cast(bf16x8, vtx::U4{hi[0], hi[1], hi[2], hi[3]});
  const bf16x8 bl = __builtin_bit_cast(bf16x8, vtx::U4{lo[0], lo[1], lo[2], lo[3]});
#pragma unroll
  for (int x4 = 0; x4 < kD / 64; ++x4) {
    uint32_t f[4][4];  // column 4 x4 + .., token pair
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        const uint32_t p = t.v[h][i][x4], r = t.v[h][i + 1][x4];
        const int at = 2 * h + i / 2;
        if constexpr (kCodes == VTX_CODES_E4M3) {
          vtx::decode_pairs<kCodes>(__builtin_amdgcn_perm(r, p, 0x05010400u), f[0][at], f[1][at]);
          vtx::decode_pairs<kCodes>(__builtin_amdgcn_perm(r, p, 0x07030602u), f[2][at], f[3][at]);
        } else {
          float u[4], v[4];
          vtx::decode4<kCodes>(p, u);
          vtx::decode4<kCodes>(r, v);
#pragma unroll
          for (int c = 0; c < 4; ++c)
            f[c][at] = __builtin_amdgcn_perm(__float_as_uint(v[c]), __float_as_uint(u[c]), 0x07060302u);
        }
      }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const bf16x8 v = __builtin_bit_cast(bf16x8, vtx::U4{f[c][0], f[c][1], f[c][2], f[c][3]});
      w.o[4 * x4 + c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, bh, w.o[4 * x4 + c], 0, 0, 0);
      w.o[4 * x4 + c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, bl, w.o[4 * x4 + c], 0, 0, 0);
    }
  }
}

// fp32 -> the queries' type.
template <bool kHalf>
__device__ __forceinline__ uint32_t round2(float a, float b) {
  if constexpr (kHalf) {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, f16x2{(_Float16)a, (_Float16)b});
  } else {
    return vtx::bf16_pair(a, b);
  }
}

// The result of sums O and L: zeros where nothing was seen, NaN where a score was.
__device__ __forceinline__ float inverse_sum(float L) { return L > 0.f ? 1.f / L : (L == 0.f ? 0.f : NAN); }

// Workgroups of a compute unit: as many as the registers let in.
template <int kD>
constexpr int kPerCu = kD == 256 ? 2 : (kD == 128 ? 3 : 4);

// kWaves 1: a workgroup per segment, or per part of one (Division's chunks).
template <int kD, int kCodes, bool kHalf, bool kPages16, int kWaves>
__global__ __launch_bounds__(kWaves* vtx::kWave, kPerCu<kD>) void quant_attention_kernel(QAttnArgs a) {
  constexpr int kThreads = kWaves * vtx::kWave;
  constexpr bool kLine = kWaves > 1;
  constexpr int kStage = kLine ? ::kStage : 128;
  __shared__ int32_t s_ptr[kLine ? kBounds : 1], s_last[kLine ? kBounds : 1], s_rows[kStage];
  __shared__ float s_m[kWaves][kHeads], s_l[kWaves][kHeads];
  __shared__ alignas(16) Shared<kD, kHalf, kWaves> sh;

  const int tid = threadIdx.x, lane = vtx::lane_id();
  const int wave = vtx::uniform(tid / vtx::kWave);
  const int c16 = lane % 16, g4 = lane / 16;
  const int S = a.segments, G = a.G, P = a.P;

  // This workgroup's range of the line, and its first segment.  How the line is laid
  // out: the table's own pages; with a window the pages that count, closely packed,
  // or where the segments are too many for a sum over all of them at equal distances
  // (segments shorter than the window leave gaps).  A table of few segments is
  // brought to LDS whole, so that all its bounds cost one trip.
  int first = 0, seg = (int)blockIdx.x;
  uint32_t total = 0, v0 = 0, v1 = 1;
  uint32_t chunk = 0;  // a segment's parts have at most so many pages (0: ranges of the line)
  int nth = 0;         // which of them is this workgroup's
  int part_row = 0;    // where its result goes
  const bool whole = a.workers == 0, few = kLine && !whole && S < kBounds, packed = few && a.window > 0;  // uniform
  if (!whole) {
    if (packed) {
      constexpr int kEach = kLine ? kBounds / kThreads : 1;
      uint32_t pages[kEach], mine = 0;
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int j = tid * kEach + i;
        pages[i] = j < S ? (uint32_t)segment_of(a, a.indptr[j], a.indptr[j + 1], a.last_len[j]).pages : 0u;
        mine += pages[i];
      }
      uint32_t before = vtx::wave_prefix_sum(mine) - mine;
      if (lane == vtx::kWave - 1) s_m[wave][0] = __uint_as_float(before + mine);
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kWaves; ++i) {
        const uint32_t x = __float_as_uint(s_m[i][0]);
        before += i < wave ? x : 0u;
        total += x;
      }
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int j = tid * kEach + i;
        if (j <= S) {
          s_ptr[j] = (int32_t)before;
          if (blockIdx.x == 0) a.places[j] = (int32_t)before;  // for the join
        }
        before += pages[i];
      }
      total = (uint32_t)vtx::uniform((int)total);
      __syncthreads();
    } else if (few) {
#pragma unroll
      for (int i = 0; i < (kLine ? kBounds : 0); i += kThreads)
        if (i + tid <= S) {
          s_ptr[i + tid] = a.indptr[i + tid];
          s_last[i + tid] = a.last_len[min(i + tid, S - 1)];
        }
      __syncthreads();
      first = vtx::uniform(s_ptr[0]);
      total = table_pages(a, first, vtx::uniform(s_ptr[S]));
    } else if (a.pitch > 0) {
      total = (uint32_t)S * (uint32_t)a.pitch;  // (the host sees to it that this fits)
    } else {
      first = a.indptr[0];
      total = table_pages(a, first, a.indptr[S]);
    }
    const Division dv = divide_pages(a, total);
    chunk = dv.chunk;
    if (kLine && chunk == 0) {
      const uint64_t at = (uint64_t)blockIdx.x * dv.per;
      if (at >= total) return;  // uniform
      v0 = (uint32_t)at;
      v1 = total - v0 < dv.per ? total : v0 + dv.per;
    }
    if (!kLine || chunk > 0) {
      if (seg >= S) {  // uniform: the (seg - S)-th part behind the segments' first ones
        const uint32_t want = (uint32_t)(seg - S);
        if constexpr (!kLine) {  // mostly none is cut: a look at the table first
          bool any = false;
#pragma unroll 8
          for (int j = lane; j < S; j += vtx::kWave) {
            const int p0 = a.indptr[j], p1 = a.indptr[j + 1];
            any |= p1 > p0 && (uint32_t)p1 - (uint32_t)p0 > chunk;
          }
          if (!__any(any)) return;  // uniform
        }
        const int each = (S + kThreads - 1) / kThreads, j0 = min(tid * each, S), j1 = min(j0 + each, S);
        uint32_t mine = 0, cut = 0;  // such parts of this thread's segments, and how many segments have them
        for (int j = j0; j < j1; ++j) {
          const uint32_t n = parts_at(a, j, chunk);
          mine = add_parts(mine, n - 1u);
          cut += n > 1u ? 1u : 0u;
        }
        uint32_t before = vtx::wave_prefix_sum(mine) - mine, rows = vtx::wave_prefix_sum(cut) - cut, all = 0;
        if (lane == vtx::kWave - 1) {
          s_m[wave][0] = __uint_as_float(before + mine);
          s_m[wave][1] = __uint_as_float(rows + cut);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kWaves; ++i) {
          const uint32_t x = __float_as_uint(s_m[i][0]);
          before += i < wave ? x : 0u;
          rows += i < wave ? __float_as_uint(s_m[i][1]) : 0u;
          all += x;
        }
        if (want >= all) return;  // uniform
        if (want >= before && want < before + mine) {
          int j = j0;
          for (uint32_t n; want >= before + (n = parts_at(a, j, chunk) - 1u); ++j) {
            before += n;
            rows += n > 0u ? 1u : 0u;
          }
          s_l[0][0] = __int_as_float(j);
          s_l[0][1] = __uint_as_float(want - before + 1u);
          s_l[0][2] = __uint_as_float(want + 1u + rows);
        }
        __syncthreads();
        seg = vtx::uniform(__float_as_int(s_l[0][0]));
        nth = vtx::uniform(__float_as_int(s_l[0][1]));
        part_row = vtx::uniform(__float_as_int(s_l[0][2]));
        __syncthreads();
      }
    } else if (few) seg = segments_before(S, first, v0, [&](int j) { return s_ptr[j]; });
    else if (a.pitch > 0) seg = (int)divide(v0, a.by_pitch);
    else seg = segments_before(S, first, v0, [&](int j) { return a.indptr[j]; });
  }

  const bool alone = !kLine || whole || chunk > 0;  // this workgroup has one piece
  // What this workgroup has of a segment: pages pa .. pb of those that count.
  struct Piece {
    Segment s;
    uint32_t at;
    int seg, pa, pb;  // seg S: none
    bool part;        // of a segment that lies in other ranges too
  };
  int base_seg = -vtx::kWave - 1;  // the 64 segments whose bounds the lanes hold
  int b0 = 0, b1 = 0, bl = 0;
  const bool bounds_here = few && !packed;
  auto hold = [&](int s) {
    if (s - base_seg >= vtx::kWave) {  // uniform
      base_seg = s;
      const int j = min(s + lane, S - 1);
      bl = bounds_here ? s_last[j] : a.last_len[j];
      b0 = bounds_here ? s_ptr[j] : a.indptr[j];
      b1 = bounds_here ? s_ptr[j + 1] : a.indptr[j + 1];
    }
  };
  auto piece_from = [&](int s) {  // the first from segment s on
    Piece p;
    p.seg = S;
    for (; s < S; ++s) {
      hold(s);
      const int p0 = (int)vtx::lane_value((uint32_t)b0, s - base_seg);
      p.s = segment_of(a, p0, (int)vtx::lane_value((uint32_t)b1, s - base_seg),
                       (int)vtx::lane_value((uint32_t)bl, s - base_seg));
      if (alone) {
        const int n = whole ? 1 : (int)parts_of(p.s.pages, chunk), each = (p.s.pages + n - 1) / n;
        p.at = 0;
        p.seg = s;
        p.pa = min(nth * each, p.s.pages);
        p.pb = min(p.pa + each, p.s.pages);
        p.part = n > 1;
        break;
      }
      const bool laid = packed || a.pitch > 0;  // elsewhere than in the table
      const uint32_t begin = packed ? (uint32_t)vtx::uniform(s_ptr[s])
                                    : (laid ? (uint32_t)s * (uint32_t)a.pitch : (uint32_t)p0 - (uint32_t)first);
      if (begin >= v1 && (laid || p0 > first)) break;
      const Place l = place_of(p.s, laid ? begin : (uint32_t)p.s.start - (uint32_t)first, total);
      const uint32_t x = l.at > v0 ? l.at : v0, y = l.end < v1 ? l.end : v1;
      if (x >= y) continue;  // (the join writes an empty segment's zeros)
      p.at = l.at;
      p.seg = s;
      p.pa = (int)(x - l.at);
      p.pb = (int)(y - l.at);
      p.part = l.at < v0 || l.end > v1;
      break;
    }
    return p;
  };
  // the page rows of places staged .. staged_end, as far as they lie on the line
  uint32_t staged = 0, staged_end = 0;
  auto stage = [&](const Piece& p, uint32_t from, uint32_t end) {
    staged = from;
    staged_end = min(end, from + (uint32_t)kStage);
    int s = p.seg;
    for (uint32_t v = from + tid; v < staged_end; v += kThreads) {
      int64_t at = alone ? (int64_t)p.s.start + v : (int64_t)first + v;
      if (!alone && (packed || a.pitch > 0)) {
        while (packed && s + 1 < S && (uint32_t)s_ptr[s + 1] <= v) ++s;
        if (!packed) s = (int)divide(v, a.by_pitch);
        const Segment g = s == p.seg ? p.s : segment_of(a, a.indptr[s], a.indptr[s + 1], a.last_len[s]);
        at = (int64_t)g.start + (v - (packed ? (uint32_t)s_ptr[s] : (uint32_t)s * (uint32_t)a.pitch));
      }
      const int r = at >= 0 && at < a.indices_len ? a.indices[at] : -1;
      s_rows[v - from] = r >= 0 && r < a.rows ? r : -1;
    }
    __syncthreads();
  };
  // the staged pages of a piece from page pc on: tokens numbered from the first of them
  struct Stretch {
    const int32_t* rows;
    int pages, n;
  };
  auto stretch_of = [&](const Piece& p, int pc) {
    const uint32_t v = p.at + (uint32_t)pc;
    Stretch t{s_rows, 0, 0};
    if (v >= staged && v < staged_end) {
      t.rows += v - staged;
      t.pages = min(p.pb - pc, (int)(staged_end - v));
      t.n = (pc + t.pages == p.s.pages ? p.s.tokens : (pc + t.pages) * P) - pc * P;
    }
    return t;
  };

  // a tile's 16 tokens of one page (P % 16 == 0): their pool row, and how many of
  // them there are (uniform); the tile whose codes are on their way
  struct Half {
    long long row;
    int tokens;
  };
  auto half_of = [&](const Stretch& t, int i, int hf) {
    const int t0 = i * kTile + hf * 16;
    const int pg = a.p_shift >= 0 ? t0 >> a.p_shift : t0 / P;
    const int r = vtx::uniform(t.rows[t0 < t.n ? pg : 0]);
    return Half{(long long)r * P + (t0 - pg * P), t0 < t.n && r >= 0 ? min(t.n - t0, 16) : 0};
  };

  Half half[2];  // of the tile on its way
  Keys<kD> keys;
  Values<kD> values;
  auto aim = [&](const Stretch& t, int i) {
    half[0] = half_of(t, i, 0);
    half[1] = half_of(t, i, 1);
  };
  auto load_keys = [&]() {
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const auto r = buffer_of(a.k + half[hf].row * kD, (uint32_t)half[hf].tokens * kD);
#pragma unroll
      for (int j = 0; j < kD / 64; ++j) {
        uint32_t x[4];
        load_words<4>(r, c16 * kD + g4 * 16 + j * 64, x);
        keys.k[hf][j] = vtx::U4{x[0], x[1], x[2], x[3]};
      }
    }
  };
  auto load_values = [&]() {
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      uint32_t x[2];
      // (all 16 slots': a load that reaches past the end gives nothing at all)
      load_words<2>(buffer_of(a.scales + half[hf].row * 2, half[hf].tokens > 0 ? 32u : 0u), g4 * 8, x);
      values.sc[hf] = uint2{x[0], x[1]};
      const auto r = buffer_of(a.v + half[hf].row * kD, (uint32_t)half[hf].tokens * kD);
#pragma unroll
      for (int u = 0; u < 4; ++u) load_words<kD / 64>(r, 4 * g4 * kD + c16 * (kD / 16) + u * kD, values.v[hf][u]);
    }
  };
  // a segment's query rows; heads past G take head 0's, and nobody takes their results
  Queries<kD, kHalf, kWaves> own;
  float slope = 0.f;
  auto load_queries = [&](int s) {
    const int b = (int)divide((uint32_t)s, a.by_heads), h = s - b * a.H;
    const uint16_t* q = a.q + b * a.q_batch + h * a.q_kv + (c16 < G ? c16 : 0) * a.q_head + g4 * 16;
#pragma unroll
    for (int i = 0; i < Queries<kD, kHalf, kWaves>::kOwn; ++i) {
      const int j = kHalf ? min(i * kWaves + wave, kD / 32 - 1) : i;
      own.raw[i] = vtx::ld16(q + (j / 2) * 64 + (j % 2) * 8);
    }
    if (a.slopes) slope = a.slopes[h * G + (c16 < G ? c16 : 0)] * kLog2e;
  };

  Piece cur = piece_from(seg);
  if (cur.seg >= S) return;  // uniform
  if (alone && cur.part && nth == 0) {  // uniform: behind the parts of the cut segments before this
    part_row = (int)parts_before<kThreads>(a, seg, chunk, &s_l[0][0]);
    __syncthreads();
  }
  load_queries(cur.seg);
  bool ready = false;  // this wave's first tile of the segment is on its way
  while (true) {
    if constexpr (kHalf) {  // fp16 values as two bf16 ones, to LDS
#pragma unroll
      for (int i = 0; i < Queries<kD, kHalf, kWaves>::kOwn; ++i) {
        const int j = i * kWaves + wave;
        if (j >= kD / 32) break;  // uniform
        typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
        const f16x8 f = __builtin_bit_cast(f16x8, own.raw[i]);
        uint32_t x[4], y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float u = (float)f[2 * e], v = (float)f[2 * e + 1];
          // (under a cap an infinity leaves nothing, so that its scores become +-cap;
          // without one they are no weights, and its NaN says so)
          x[e] = vtx::bf16_pair(u, v);
          y[e] = vtx::bf16_pair(a.cap != 0.f && fabsf(u) == INFINITY ? 0.f : u - vtx::bf16_lo(x[e]),
                                a.cap != 0.f && fabsf(v) == INFINITY ? 0.f : v - vtx::bf16_hi(x[e]));
        }
        sh.q[0][j][lane] = vtx::U4{x[0], x[1], x[2], x[3]};
        sh.q[1][j][lane] = vtx::U4{y[0], y[1], y[2], y[3]};
      }
      // (where no staging with its barrier comes before the tiles)
      if (stretch_of(cur, cur.pa).pages > 0) __syncthreads();
    }
    Heads<kD> w;
    w.m = -INFINITY;
    w.l = 0.f;
#pragma unroll
    for (int d = 0; d < kD / 16; ++d) w.o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int pc = cur.pa; pc < cur.pb;) {
      Stretch st = stretch_of(cur, pc);
      if (st.pages == 0) {  // uniform
        if (staged_end > 0) __syncthreads();  // (the staged rows are done with)
        stage(cur, cur.at + (uint32_t)pc, alone ? (uint32_t)cur.pb : v1);
        st = stretch_of(cur, pc);
      }
      const int skip = pc == 0 ? cur.s.skip : 0;
      const int tiles = (st.n + kTile - 1) / kTile;
      const float far0 = (float)(cur.s.tokens - 1 - pc * P - 4 * g4);
      pc += st.pages;

      if constexpr (kPages16) {
        if (!ready) {  // uniform
          aim(st, wave);
          load_keys();
          load_values();
        }
        ready = false;
        for (int i = wave; i < tiles; i += kWaves) {
          f32x4 sc[2];
          score<kD, kCodes>(sh, own, keys, sc);
          const int n0 = half[0].tokens, n1 = half[1].tokens;
          aim(st, i + kWaves);  // (none past the last: no loads)
          load_keys();
          const int out = skip - i * kTile;  // tokens before the window
          uint32_t bad = 0;
          const bool masked = n0 + n1 < kTile || out > 0;
          if (masked) {  // uniform
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              bad |= 4 * g4 + x >= n0 || 4 * g4 + x < out ? 1u << x : 0u;
              bad |= 4 * g4 + x >= n1 || 16 + 4 * g4 + x < out ? 16u << x : 0u;
            }
          }
          attend<kD, kCodes>(a, w, sc, values, masked, bad, far0 - (float)(i * kTile), slope);
          load_values();
        }
      } else {
        // the pool row of a token, and whether it counts (row 0 where not)
        auto token_row = [&](int tok, bool& ok) {
          ok = tok < st.n;
          const int pg = ok ? tok / P : 0;
          const int r = st.rows[pg];
          ok = ok && r >= 0;
          return ok ? (long long)r * P + (tok - pg * P) : 0LL;
        };
        for (int i = wave; i < tiles; i += kWaves) {
          uint32_t bad = 0;
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            bool ok;
            const unsigned char* kp = a.k + token_row(i * kTile + hf * 16 + c16, ok) * kD + g4 * 16;
#pragma unroll
            for (int j = 0; j < kD / 64; ++j) keys.k[hf][j] = vtx::ld16_stream(kp + j * 64);
            uint32_t two[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int tok = i * kTile + hf * 16 + 4 * g4 + x;
              const long long row = token_row(tok, ok);
              load_v<kD>(a.v + row * kD + c16 * (kD / 16), values.v[hf][x]);
              two[x] = *reinterpret_cast<const uint16_t*>(a.scales + row * 2);
              bad |= ok && tok >= skip ? 0u : 1u << (4 * hf + x);
            }
            values.sc[hf] = uint2{two[0] | (two[1] << 16), two[2] | (two[3] << 16)};
          }
          f32x4 sc[2];
          score<kD, kCodes>(sh, own, keys, sc);
          attend<kD, kCodes>(a, w, sc, values, __ballot(bad != 0) != 0, bad, far0 - (float)(i * kTile), slope);
        }
      }
    }

    // the next segment's queries and first tiles, requested before this one's end
    Piece nxt;
    nxt.seg = S;
    if (!alone) nxt = piece_from(cur.seg + 1);
    if (nxt.seg < S) {  // uniform
      load_queries(nxt.seg);
      if constexpr (kPages16) {
        const Stretch t = stretch_of(nxt, nxt.pa);
        ready = t.pages > 0;
        if (ready) {
          aim(t, wave);
          load_keys();
          load_values();
        }
      }
    }

    // the waves' results joined in LDS: the segment's, or this part of it
    float l = w.l + vtx::xshfl(w.l, 16);
    l += vtx::xshfl(l, 32);
    // (a maximum passes NaN scores by; where nothing else was seen it is still
    // -inf, which the joins take for no tokens)
    const float m = l != l ? 0.f : w.m;
    if constexpr (kHalf) __syncthreads();  // (the queries are done with)
    if (c16 < G) {
      if (g4 == 0) {
        s_m[wave][c16] = m;
        s_l[wave][c16] = l;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int x4 = 0; x4 < kD / 64; ++x4)
          *reinterpret_cast<float4*>(&sh.o[wave][c16][(4 * g4 + i) * (kD / 16) + 4 * x4]) =
              float4{w.o[4 * x4][i], w.o[4 * x4 + 1][i], w.o[4 * x4 + 2][i], w.o[4 * x4 + 3][i]};
    }
    __syncthreads();
    for (int x = tid; x < G * (kD / 4); x += kThreads) {
      const int g = x / (kD / 4), d = (x % (kD / 4)) * 4;
      float M = -INFINITY, L = 0.f;
      float4 O{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < kWaves; ++i) M = fmaxf(M, s_m[i][g]);
      if (M != -INFINITY) {
#pragma unroll
        for (int i = 0; i < kWaves; ++i) {
          const float f = __builtin_amdgcn_exp2f(s_m[i][g] - M);
          const float4 y = *reinterpret_cast<const float4*>(&sh.o[i][g][d]);
          L = fmaf(s_l[i][g], f, L);
          O = float4{fmaf(y.x, f, O.x), fmaf(y.y, f, O.y), fmaf(y.z, f, O.z), fmaf(y.w, f, O.w)};
        }
      }
      if (cur.part) {  // uniform
        const int at = alone ? part_row : 2 * (int)blockIdx.x + (cur.at + (uint32_t)cur.pa == v0 ? 0 : 1);
        const long long row = (long long)at * G + g;
        if (at >= 2 * a.slots) break;  // (a table that decreases, if at all)
        *reinterpret_cast<float4*>(a.acc + row * kD + d) = O;
        if (d == 0) a.ml[row] = float2{M, L};
      } else {
        const float f = cur.s.over ? NAN : inverse_sum(L);
        *reinterpret_cast<uint2*>(a.o + ((long long)cur.seg * G + g) * kD + d) =
            uint2{round2<kHalf>(O.x * f, O.y * f), round2<kHalf>(O.z * f, O.w * f)};
      }
    }
    if (nxt.seg >= S) return;  // uniform
    __syncthreads();           // (the next segment's results go to the same place)
    cur = nxt;
  }
}

// The parts of a segment that lies in several ranges, joined; zeros for one
// without tokens.  Threads = (part of the parts, head, four columns), each with a
// running maximum of its own; a workgroup takes `join_items` of a segment's (head,
// four columns): 256, or as many fewer (32, a row's 512 bytes, at least) as let its
// threads take the parts that there are, on average, in one trip.  All by one
// workgroup / so, 128 columns: 8 segments of up to 20k tokens and 16 heads 36.4 / 21.5
// us, one of 32k and 8 heads 38.6 / 15.1, 13 of up to 30k and 8 heads 35.0 / 24.6.
constexpr int kJoinThreads = 256, kJoinAhead = 8;  // parts of a thread in flight
inline int join_items(long long segments, long long slots) {
  int n = kJoinThreads;
  while (n > 32 && n * slots > (long long)kJoinThreads * kJoinAhead * segments) n /= 2;
  return n;
}
template <int kD, bool kHalf>
__global__ __launch_bounds__(kJoinThreads) void quant_attention_join_kernel(QAttnArgs a) {
  constexpr int kAhead = kJoinAhead;
  __shared__ alignas(16) float s_o[kJoinThreads][4];
  __shared__ float2 s_ml[kJoinThreads];
  const int seg = blockIdx.x, tid = threadIdx.x, G = a.G, S = a.segments;
  const bool packed = S < kBounds && a.window > 0;
  const int first = a.indptr[0];
  const uint32_t total = packed ? (uint32_t)a.places[S]
                                : (a.pitch > 0 ? (uint32_t)S * (uint32_t)a.pitch : table_pages(a, first, a.indptr[S]));
  const Segment sg = segment_of(a, a.indptr[seg], a.indptr[seg + 1], a.last_len[seg]);
  const uint32_t begin = packed        ? (uint32_t)a.places[seg]
                         : a.pitch > 0 ? (uint32_t)seg * (uint32_t)a.pitch
                                       : (uint32_t)sg.start - (uint32_t)first;
  const Place at = place_of(sg, begin, total);
  const Division dv = divide_pages(a, total);
  uint32_t w0 = 0;
  int n = 0;
  bool second = false;  // the first part lies behind another segment's
  if (dv.chunk > 0) {
    n = (int)parts_of(sg.pages, dv.chunk);
    if (n == 1) return;  // uniform: written by its workgroup, zeros too
    w0 = parts_before<kJoinThreads>(a, seg, dv.chunk, &s_o[0][0]);
    if ((uint64_t)w0 + (uint32_t)n > 2u * (uint32_t)a.slots) n = 0;  // (a table that decreases, if at all)
  } else if (at.end > at.at) {
    w0 = at.at / dv.per;
    if (at.end <= (w0 + 1) * dv.per) return;  // uniform: written by its workgroup
    n = (int)((at.end - 1) / dv.per - w0) + 1;
    second = at.at > w0 * dv.per;
  }
  const int items = G * (kD / 4), x0 = (int)blockIdx.y * a.join;
  const int here = min(items - x0, a.join);
  const int most = kJoinThreads / here, groups = n < most * 2 ? (n + 1) / 2 : most;
  const int grp = tid / here, x = tid - grp * here;
  const int g = (x0 + x) / (kD / 4), d = ((x0 + x) % (kD / 4)) * 4;
  float M = -INFINITY, L = 0.f;
  float4 O{0.f, 0.f, 0.f, 0.f};
  if (grp < groups) {
    // part i of a cut segment is row w0 + i; of one in several ranges 2 (w0 + i), one
    // more for the first where that lies behind another segment's
    const int step = dv.chunk > 0 ? 1 : 2, row1 = second ? 1 : 0;
    const long long row0 = (long long)w0 * step;
    const float2* ml = a.ml + row0 * G + g;
    const float* acc = a.acc + (row0 * G + g) * kD + d;
    for (int i0 = grp; i0 < n; i0 += groups * kAhead) {
      float2 z[kAhead];
      float4 y[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int i = i0 + u * groups, row = (i == 0 ? row1 : step * i) * G;
        z[u] = float2{-INFINITY, 0.f};
        y[u] = float4{0.f, 0.f, 0.f, 0.f};
        if (i < n) {
          z[u] = ml[row];
          y[u] = *reinterpret_cast<const float4*>(acc + (long long)row * kD);
        }
      }
      float nm = M;
#pragma unroll
      for (int u = 0; u < kAhead; ++u) nm = fmaxf(nm, z[u].x);
      if (nm == -INFINITY) continue;
      const float f = __builtin_amdgcn_exp2f(M - nm);
      L *= f;
      O = float4{O.x * f, O.y * f, O.z * f, O.w * f};
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const float e = __builtin_amdgcn_exp2f(z[u].x - nm);
        L = fmaf(z[u].y, e, L);
        O = float4{fmaf(y[u].x, e, O.x), fmaf(y[u].y, e, O.y), fmaf(y[u].z, e, O.z), fmaf(y[u].w, e, O.w)};
      }
      M = nm;
    }
  }
  if (groups > 1) {  // uniform
    __syncthreads();
    s_ml[tid] = float2{M, L};
    *reinterpret_cast<float4*>(s_o[tid]) = O;
    __syncthreads();
  }
  if (grp == 0) {
    for (int i = 1; i < groups; ++i) {
      const float2 z = s_ml[i * here + x];
      const float4 y = *reinterpret_cast<const float4*>(s_o[i * here + x]);
      const float nm = fmaxf(M, z.x);
      if (nm == -INFINITY) continue;
      const float f = __builtin_amdgcn_exp2f(M - nm), e = __builtin_amdgcn_exp2f(z.x - nm);
      L = L * f + z.y * e;
      O = float4{O.x * f + y.x * e, O.y * f + y.y * e, O.z * f + y.z * e, O.w * f + y.w * e};
      M = nm;
    }
    const float f = sg.over ? NAN : inverse_sum(L);
    *reinterpret_cast<uint2*>(a.o + ((long long)seg * G + g) * kD + d) =
        uint2{round2<kHalf>(O.x * f, O.y * f), round2<kHalf>(O.z * f, O.w * f)};
  }
}

template <int kD, int kCodes, bool kHalf>
int launch_one(const QAttnArgs& a, hipStream_t s) {
  const int grid = a.workers > 0 ? a.workers : a.segments;
  constexpr int all = kAllWaves, threads = all * vtx::kWave;
  if (a.P % 16 != 0) quant_attention_kernel<kD, kCodes, kHalf, false, all><<<grid, threads, 0, s>>>(a);
  else if (a.tiny) quant_attention_kernel<kD, kCodes, kHalf, true, 1><<<grid, vtx::kWave, 0, s>>>(a);
  else quant_attention_kernel<kD, kCodes, kHalf, true, all><<<grid, threads, 0, s>>>(a);
  if (a.workers > 0)
    quant_attention_join_kernel<kD, kHalf>
        <<<dim3(a.segments, (a.G * (kD / 4) + a.join - 1) / a.join), kJoinThreads, 0, s>>>(a);
  return vtx::check_launch("quant_decode_attention");
}

template <int kD>
int launch_types(const QAttnArgs& a, int codes, bool half, hipStream_t s) {
  if (codes == VTX_CODES_E4M3)
    return half ? launch_one<kD, VTX_CODES_E4M3, true>(a, s) : launch_one<kD, VTX_CODES_E4M3, false>(a, s);
  return half ? launch_one<kD, VTX_CODES_INT8, true>(a, s) : launch_one<kD, VTX_CODES_INT8, false>(a, s);
}

// Ranges of a call: as many workgroups as the card holds at once, and no more
// than the buffer's pages can fill; or none, a workgroup per segment and one
// launch, where no segment can be long.  known: tokens that no segment exceeds
// (the window, the caller's word; 0: unknown).
//
// Segments of up to `few` tokens, by the buffer's size if all heads of a request
// are alike: ranges / segments, 8 segments of 128 columns, 128 tokens 9.0 / 6.1 us,
// 512 10.9 / 10.3, 768 11.1 / 13.1; 64 columns, 512 10.2 / 8.6, 768 10.4 / 10.7; 256
// columns, 256 12.0 / 9.2, 512 12.3 / 13.3.
//
// Known bounds, of fewer segments than compute units: with a window the line costs
// more to lay out (128 of 1024 22 / 19, of 2048 27 / 30; 256 columns, 64 of 768 22 / 20,
// of 1024 22 / 24).  Of more, which fill the card by themselves, it depends on the
// table.  Ranges / segments, all equal; between an eighth of the bound and it; anything
// under it; one in eight as long, the others a sixteenth:
//   128 columns, 256 of 1024  21 / 18, 24 / 17, 39 / 15, 18 / 16
//                256 of 2048  33 / 31, 31 / 29, 56 / 28, 18 / 27
//                512 of 2048  52 / 50, 49 / 42, 39 / 40, 36 / 38
//                512 of 4096  95 / 93, 68 / 76, 93 / 73, 39 / 71
//               1024 of 4096  184 / 181, 114 / 150, 121 / 124, 69 / 105
//   64 columns,  512 of 2048  34 / 30, 30 / 27, 62 / 27, 25 / 27
//                512 of 4096  57 / 54, 41 / 49, 71 / 48, 28 / 48
//   256 columns, 512 of 1024  50 / 47, 41 / 39, 38 / 36, 39 / 36
//                512 of 2048  90 / 88, 65 / 73, 71 / 66, 62 / 66
//                320 of 2048  64 / 77, 47 / 65, 46 / 62, 42 / 65
// (ranges lose where a few requests of a page or two share one, whose segments a
// workgroup takes one by one, segments where a few long ones come last).  So up to 2048
// tokens, or 1024 of 256 columns, where segments lose less than ranges would; past that
// divide_pages looks at the table.  With windows of a spaced line, whose places are all
// alike, that comes to segments as well, and the second launch on top (1024 of 4096 183
// / 180, 126 / 124): up to 4096.
//
// Tiny segments, more than workgroups that the card holds: a wave each, since four
// share a tile or two and then wait for each other (by the longest they can have or,
// unknown, by the buffer's size; those that are long all the same are cut from 64
// tokens x 8 on).  Four waves / one, 128 columns, 1024 segments of 16 tokens 13.6 /
// 7.7 us, 2048 of 64 25.8 / 14.8, of 128 29.8 / 20.7, of 256 38.5 / 32.7, of 512 57.5
// / 56.3, of up to 1000 74.0 / 83.6; 64 columns, 2048 of 64 20.1 / 11.7, of 256 26.8 /
// 23.3, of up to 500 30.8 / 33.2; 256 columns, 1024 of 64 21.4 / 12.5, of 256 33.5 /
// 29.1.
struct Ranges {
  long long workers, slots, least, cus, pitch;
  bool tiny;
};
Ranges ranges_of(long long segments, int32_t num_kv_heads, int32_t head_dim, int32_t page_size, int32_t window,
                 int32_t longest, long long indices_len) {
  Ranges r{0, 0, 1, 1, 0, false};
  r.cus = vtx::device_cu_count() > 0 ? vtx::device_cu_count() : 256;
  const long long few = 640 - head_dim;
  const long long known = longest > 0 && (window == 0 || longest < window) ? longest : window;
  const long long most = segments < r.cus ? (window == 0 ? few : (head_dim == 256 ? 768 : 1024))
                         : window > 0 && segments >= kBounds ? 4096
                                                             : (head_dim == 256 ? 1024 : 2048);
  const int per_cu = head_dim == 256 ? kPerCu<256> : (head_dim == 128 ? kPerCu<128> : kPerCu<64>);
  r.tiny = page_size % 16 == 0 && segments > r.cus * per_cu &&
           ((known > 0 && known <= kTiny) || (window == 0 && indices_len * page_size <= kTiny * segments));
  if (indices_len * page_size <= few * num_kv_heads || (known > 0 && known <= most)) return r;
  r.least = ((r.tiny ? kMinTokens / 2 : kMinTokens) + (long long)page_size - 1) / page_size;
  r.slots = r.cus * per_cu * (r.tiny ? kAllWaves : 1);
  if (r.tiny) r.slots = std::min(r.slots, segments);
  r.pitch = 0;
  if (window > 0 && segments >= kBounds) {
    const long long most = ((long long)window + page_size - 1) / page_size + 1;  // pages that a window touches
    if (most * segments <= 0x7fffffffLL) r.pitch = most;
  }
  const long long need = std::max(segments, (indices_len + r.least - 1) / r.least);
  if (r.slots > need) r.slots = need;
  // (a workgroup per segment, and no more parts behind them than chunks, of twice a
  // workgroup's share and of eight times the least)
  r.workers = std::max(r.slots, segments + std::min(r.slots / 2, indices_len / (8 * r.least)) + 1);
  return r;
}
// Floats of scratch: two parts a range, and a packed line's places.
long long scratch_of(const Ranges& r, long long segments, int32_t group_size, int32_t head_dim, int32_t window) {
  if (r.workers == 0) return 0;
  return 2 * r.slots * group_size * (head_dim + 2) + (window > 0 && segments < kBounds ? segments + 1 : 0);
}

}  // namespace

extern "C" int vtx_quant_decode_attention_supported(int32_t head_dim, int32_t group_size) {
  return (head_dim == 64 || head_dim == 128 || head_dim == 256) && group_size >= 1 && group_size <= kHeads;
}

extern "C" int64_t vtx_quant_decode_attention_workspace_len(int32_t batch_size, int32_t num_kv_heads,
                                                            int32_t group_size, int32_t head_dim, int32_t page_size,
                                                            int32_t window, int32_t longest, int64_t kv_indices_len) {
  if (batch_size < 1 || num_kv_heads < 1 || page_size < 1 || window < 0 || longest < 0 || kv_indices_len < 0 ||
      !vtx_quant_decode_attention_supported(head_dim, group_size))
    return 0;
  const long long segments = (long long)batch_size * num_kv_heads;
  return scratch_of(ranges_of(segments, num_kv_heads, head_dim, page_size, window, longest, kv_indices_len), segments,
                    group_size, head_dim, window);
}

extern "C" int vtx_quant_decode_attention(const void* q, const int64_t* q_strides, void* o, const void* k_cache,
                                          const void* v_cache, const void* scales, int64_t cache_rows,
                                          const int32_t* kv_indptr, const int32_t* kv_indices, int64_t kv_indices_len,
                                          const int32_t* kv_last_page_len, int32_t batch_size, int32_t num_kv_heads,
                                          int32_t group_size, int32_t head_dim, int32_t page_size, int32_t dtype,
                                          int32_t codes, float sm_scale, float soft_cap, int32_t window,
                                          const float* slopes, int32_t longest, float* workspace,
                                          int64_t workspace_len, void* stream) {
  vtx::clear_error();
  if (batch_size < 0 || num_kv_heads < 1 || page_size < 1 || cache_rows < 0 || kv_indices_len < 0 || window < 0 ||
      longest < 0)
    return vtx::fail(VTX_E_INVALID, "quant_decode_attention: bad sizes");
  if (!vtx_quant_decode_attention_supported(head_dim, group_size))
    return vtx::fail(VTX_E_INVALID, "quant_decode_attention: head_dim %d with %d query heads per kv head not supported",
                     head_dim, group_size);
  if (dtype != VTX_DTYPE_BF16 && dtype != VTX_DTYPE_F16)
    return vtx::fail(VTX_E_INVALID, "quant_decode_attention: unknown element type %d", dtype);
  if (codes != VTX_CODES_E4M3 && codes != VTX_CODES_INT8)
    return vtx::fail(VTX_E_INVALID, "quant_decode_attention: unknown codes %d", codes);
  if (!(soft_cap >= 0.f) || !(soft_cap < INFINITY))
    return vtx::fail(VTX_E_INVALID, "quant_decode_attention: the cap must be finite and not negative");
  const long long segments = (long long)batch_size * num_kv_heads;
  if (segments == 0) return VTX_OK;
  if (segments > (1LL << 23) || kv_indices_len > 0x7fffffffLL)  // (a launch has under 2^32 threads)
    return vtx::fail(VTX_E_INVALID, "quant_decode_attention: too many segments or table entries");
  if (!q || !q_strides || !o || !k_cache || !v_cache || !scales || !kv_indptr || !kv_last_page_len ||
      (kv_indices_len > 0 && !kv_indices))
    return vtx::fail(VTX_E_INVALID, "quant_decode_attention: null pointer");
  if (!vtx::aligned16(q) || !vtx::aligned16(k_cache) || !vtx::aligned16(v_cache) ||
      ((q_strides[0] | q_strides[1] | q_strides[2]) % 8) != 0 || reinterpret_cast<uintptr_t>(o) % 8 != 0 ||
      reinterpret_cast<uintptr_t>(scales) % 8 != 0)
    return vtx::fail(VTX_E_INVALID, "quant_decode_attention: query rows, k_cache and v_cache must be 16-byte aligned, "
                                    "the output and the scales 8-byte");
  QAttnArgs a;
  a.q = static_cast<const uint16_t*>(q);
  a.o = static_cast<uint16_t*>(o);
  a.k = static_cast<const unsigned char*>(k_cache);
  a.v = static_cast<const unsigned char*>(v_cache);
  a.scales = static_cast<const unsigned char*>(scales);
  a.rows = cache_rows;
  a.indptr = kv_indptr;
  a.indices = kv_indices;
  a.indices_len = kv_indices_len;
  a.last_len = kv_last_page_len;
  a.slopes = slopes;
  a.q_batch = q_strides[0];
  a.q_kv = q_strides[1];
  a.q_head = q_strides[2];
  a.segments = (int32_t)segments;
  a.H = num_kv_heads;
  a.G = group_size;
  a.P = page_size;
  a.p_shift = vtx::log2_exact(page_size);
  a.window = window;
  a.c = sm_scale * kLog2e;
  a.cap = std::min(soft_cap * kLog2e, FLT_MAX);
  a.by_cap = soft_cap > 0.f ? std::min(1.f / a.cap, FLT_MAX) : 0.f;
  a.workers = 0;
  a.tiny = false;
  a.least = 1;
  a.join = kJoinThreads;
  a.by_segments = divisor(segments);
  a.by_heads = divisor(num_kv_heads);
  a.slots = 0;
  a.balanced = false;
  a.by_slots = a.by_cus = a.by_least = a.by_pitch = divisor(1);
  a.pitch = 0;
  a.acc = nullptr;
  a.ml = nullptr;
  a.places = nullptr;
  const Ranges r = ranges_of(segments, num_kv_heads, head_dim, page_size, window, longest, kv_indices_len);
  a.tiny = r.tiny && (workspace || r.workers == 0);
  if (workspace) {
    const long long parts = 2 * r.slots * group_size, need = scratch_of(r, segments, group_size, head_dim, window);
    if (workspace_len < need || !vtx::aligned16(workspace))
      return vtx::fail(VTX_E_INVALID,
                       "quant_decode_attention: workspace of %lld floats (16-byte aligned) needed, got %lld", need,
                       (long long)workspace_len);
    a.workers = (int32_t)r.workers;  // (0: as without a workspace)
    a.least = (int32_t)r.least;
    a.join = join_items(segments, r.slots);
    a.slots = (int32_t)r.slots;
    a.balanced = 20 * ((segments + r.cus - 1) / r.cus * r.cus) <= 23 * segments;
    a.by_slots = divisor(r.slots > 0 ? r.slots : 1);
    a.by_cus = divisor(r.cus);
    a.by_least = divisor(r.least);
    a.pitch = (int32_t)r.pitch;
    if (r.pitch > 0) a.by_pitch = divisor(r.pitch);
    a.acc = workspace;
    a.ml = reinterpret_cast<float2*>(workspace + parts * head_dim);
    a.places = reinterpret_cast<int32_t*>(workspace + parts * (head_dim + 2));
  }
  hipStream_t s = vtx::as_stream(stream);
  const bool half = dtype == VTX_DTYPE_F16;
  switch (head_dim) {
    case 64: return launch_types<64>(a, codes, half, s);
    case 128: return launch_types<128>(a, codes, half, s);
    default: return launch_types<256>(a, codes, half, s);
  }
}
