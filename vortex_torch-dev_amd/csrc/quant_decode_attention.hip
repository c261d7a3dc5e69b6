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
// 4 waves per workgroup, 32 tokens of a wave at a time.  The table's pages, all
// segments after one another, are cut into equal ranges, a workgroup each, so
// that ragged lengths and any number of segments fill the card evenly; a
// workgroup meets the segments of its range one after another.  A segment inside
// its range is finished there; the others' parts (at most two per workgroup) are
// joined by a second launch.
#include "vtx_device.h"
#include "vtx_host.h"
#include "vtx_quant.h"

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / vtx::kWave;
constexpr int kHeads = 16;       // query heads of a matrix tile
constexpr int kTile = 32;        // tokens of a wave at a time
constexpr int kStage = 1024;     // page rows staged in LDS at a time
constexpr int kMinTokens = 128;  // tokens of a range at least: a tile per wave
constexpr float kLog2e = 1.4426950408889634f;

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
  int32_t window;  // the last tokens that count; 0: all
  int32_t pitch;   // pages of a segment's place on the line of pages; 0: its own pages
  float c;         // scale log2 e; with a cap 2 scale log2 e / cap
  float cap;       // cap log2 e, or 0
  int32_t workers, least;  // ranges at most, pages of one at least; workers 0: a segment each, whole
  float* acc;      // [2 workers, G, D]
  float2* ml;      // [2 workers, G]
};

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// The line of pages and its ranges.
struct Line {
  uint32_t total, per;  // pages, pages of a range
};
__device__ __forceinline__ Line line_of(const QAttnArgs& a, long long first, long long end) {
  Line l;
  if (a.pitch > 0) {
    l.total = (uint32_t)a.segments * (uint32_t)a.pitch;  // (the host sees to it that this fits)
  } else {
    const long long all = end - first;
    l.total = all < 0 ? 0u : (uint32_t)(all < a.indices_len ? all : a.indices_len);
  }
  const uint32_t even = (l.total + (uint32_t)a.workers - 1u) / (uint32_t)a.workers;
  l.per = even > (uint32_t)a.least ? even : (uint32_t)a.least;
  return l;
}

// A segment: its pages that count, and its place on the line.
struct Segment {
  long long start;     // of the pages that count, in the table
  int pages, tokens;   // that count (tokens of the last page included), from the first of these pages on
  int skip;            // tokens of the first page that the window leaves out
  uint32_t at, end;    // on the line
};
__device__ __forceinline__ Segment segment_of(const QAttnArgs& a, int s, long long first, long long p0, long long p1,
                                              int last, uint32_t total) {
  Segment g;
  g.start = p0;
  g.pages = g.tokens = g.skip = 0;
  const long long m = p1 - p0;
  if (m > 0 && p0 >= 0 && p1 <= a.indices_len && a.rows > 0) {
    last = last < 0 ? 0 : (last > a.P ? a.P : last);
    const long long n = (m - 1) * a.P + last;
    if (n > 0 && n < (1LL << 30)) {
      g.pages = (int)m;
      g.tokens = (int)n;
      if (a.window > 0 && n > a.window) {
        const int lo = (int)n - a.window, pg = lo / a.P;
        g.start += pg;
        g.pages -= pg;
        g.tokens -= pg * a.P;
        g.skip = lo - pg * a.P;
      }
    }
  }
  if (a.pitch > 0) {
    g.at = (uint32_t)s * (uint32_t)a.pitch;
    const uint32_t used = (uint32_t)g.pages < (uint32_t)a.pitch ? (uint32_t)g.pages : (uint32_t)a.pitch;
    g.end = g.at + used;
  } else {
    const long long x = g.start - first, y = p1 - first;
    const bool ok = x >= 0 && y >= x && y <= (long long)total && g.pages > 0;
    g.at = ok ? (uint32_t)x : 0u;
    g.end = ok ? (uint32_t)y : 0u;
  }
  return g;
}

// What a wave holds of 16 query heads: their fragments, running maximum (base 2),
// sum (of this lane's tokens) and output.
template <int kD, bool kHalf>
struct Heads {
  vtx::U4 q[kD / 32];
  vtx::U4 ql[kHalf ? kD / 32 : 1];  // what bf16 left of fp16 queries
  float m, l;
  f32x4 o[kD / 16];
};

// 32 tokens' codes and factors on their way.
template <int kD>
struct Tile {
  vtx::U4 k[2][kD / 64];
  uint32_t v[2][4][kD / 64];  // 16-token half, token, codes
  uint2 sc[2];                // (K, V) bytes of this lane's four tokens of a half
  bool ok[2];                 // the half lies in the pool (P % 16 == 0)
  uint32_t bad;               // tokens of this lane that do not count (otherwise): bit 4 half + i
};

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

template <int kD, int kCodes, bool kHalf>
__device__ __forceinline__ void attend(const QAttnArgs& a, Heads<kD, kHalf>& w, Tile<kD>& t, bool masked,
                                       uint32_t bad, float far, float slope) {
  f32x4 s[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    s[h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < kD / 64; ++j) {
      vtx::U4 f0, f1;
      vtx::decode_pairs<kCodes>(t.k[h][j].x, f0.x, f0.y);
      vtx::decode_pairs<kCodes>(t.k[h][j].y, f0.z, f0.w);
      vtx::decode_pairs<kCodes>(t.k[h][j].z, f1.x, f1.y);
      vtx::decode_pairs<kCodes>(t.k[h][j].w, f1.z, f1.w);
      auto mul = [&](const vtx::U4& k, const vtx::U4& q) {
        s[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, k), __builtin_bit_cast(bf16x8, q),
                                                       s[h], 0, 0, 0);
      };
      mul(f0, w.q[2 * j]);
      mul(f1, w.q[2 * j + 1]);
      if constexpr (kHalf) {
        mul(f0, w.ql[2 * j]);
        mul(f1, w.ql[2 * j + 1]);
      }
    }
  }
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
    for (int i = 0; i < 8; ++i)  // cap tanh(y / cap), the argument doubled and in base 2
      x[i] = a.cap - 2.f * a.cap * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x[i]));
  }
  if (a.slopes) {  // uniform; far: the distance of this lane's first token
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

template <int kD, int kCodes, bool kHalf, bool kPages16>
__global__ __launch_bounds__(kThreads, kD == 256 ? 2 : (kD == 128 ? 3 : 4)) void quant_attention_kernel(QAttnArgs a) {
  constexpr int kOut = kD + 4;  // floats of a head's outputs in LDS: 16 heads' pieces in all banks
  __shared__ int32_t s_rows[kStage];
  __shared__ float s_m[kWaves][kHeads], s_l[kWaves][kHeads];
  __shared__ alignas(16) float s_o[kWaves][kHeads][kOut];
  __shared__ uint32_t s_count[kWaves];

  const int tid = threadIdx.x, lane = vtx::lane_id();
  const int wave = vtx::uniform(tid / vtx::kWave);
  const int c16 = lane % 16, g4 = lane / 16;
  const int S = a.segments, G = a.G, P = a.P;

  // this workgroup's range of the line, and its first segment
  long long first = 0;
  uint32_t total = 0, v0 = 0, v1 = 1;
  int seg = (int)blockIdx.x;
  const bool whole = a.workers == 0;  // uniform
  if (!whole) {
    first = a.indptr[0];
    const Line l = line_of(a, first, a.indptr[S]);
    total = l.total;
    const unsigned long long at = (unsigned long long)blockIdx.x * l.per;
    if (at >= total) return;  // uniform
    v0 = (uint32_t)at;
    v1 = total - v0 < l.per ? total : v0 + l.per;
    if (a.pitch > 0) {
      seg = (int)(v0 / (uint32_t)a.pitch);
    } else {
      // the segments that end at or before v0, of as many evenly spaced ones as
      // there are threads first where they are many
      const int step = S > 4 * kThreads ? (S + kThreads - 1) / kThreads : 1;
      seg = 0;
      for (int round = step > 1 ? 0 : 1; round < 2; ++round) {
        const int n = round == 0 ? kThreads : (step > 1 ? step - 1 : S);
        uint32_t mine = 0;
        for (int i = tid; i < n; i += kThreads) {
          const int j = round == 0 ? (i + 1) * step : seg + i + 1;  // ends of segment j - 1
          mine += j <= S && (long long)a.indptr[j] - first <= (long long)v0 ? 1u : 0u;
        }
        mine = vtx::wave_sum(mine);
        if (lane == 0) s_count[wave] = mine;
        __syncthreads();
        uint32_t all = 0;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) all += s_count[i];
        seg = vtx::uniform(seg + (int)all * (round == 0 ? step : 1));
        __syncthreads();
      }
    }
  }

  int base_seg = -vtx::kWave - 1;  // the 64 segments whose bounds the lanes hold
  int b0 = 0, b1 = 0, bl = 0;
  for (; seg < S; ++seg) {
    if (seg - base_seg >= vtx::kWave || seg < base_seg) {  // uniform
      base_seg = seg;
      const int j = seg + lane < S ? seg + lane : S - 1;
      b0 = a.indptr[j];
      b1 = a.indptr[j + 1];
      bl = a.last_len[j];
    }
    const int at = seg - base_seg;
    const Segment sg =
        segment_of(a, seg, first, (int)vtx::lane_value((uint32_t)b0, at), (int)vtx::lane_value((uint32_t)b1, at),
                   (int)vtx::lane_value((uint32_t)bl, at), total);
    int pa = 0, pb = sg.pages;  // this workgroup's pages of the segment
    bool part = false;
    int slot = 0;
    if (!whole) {
      // (an empty segment's place may lie anywhere: the bounds of the next decide)
      if (a.pitch > 0 ? (unsigned long long)seg * (uint32_t)a.pitch >= v1
                      : (long long)(int)vtx::lane_value((uint32_t)b0, at) - first >= (long long)v1)
        break;
      const uint32_t x = sg.at > v0 ? sg.at : v0, y = sg.end < v1 ? sg.end : v1;
      if (x >= y) continue;  // (the join writes an empty segment's zeros)
      pa = (int)(x - sg.at);
      pb = (int)(y - sg.at);
      part = sg.at < v0 || sg.end > v1;
      slot = x == v0 ? 0 : 1;
    }

    Heads<kD, kHalf> w;
    w.m = -INFINITY;
    w.l = 0.f;
#pragma unroll
    for (int d = 0; d < kD / 16; ++d) w.o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int b = seg / a.H, h = seg - b * a.H;
    {
      // heads past G take head 0's queries, and nobody takes their results
      const uint16_t* q = a.q + b * a.q_batch + h * a.q_kv + (c16 < G ? c16 : 0) * a.q_head + g4 * 16;
#pragma unroll
      for (int j = 0; j < kD / 32; ++j) {
        const vtx::U4 raw = vtx::ld16(q + (j / 2) * 64 + (j % 2) * 8);
        if constexpr (kHalf) {
          typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
          const f16x8 f = __builtin_bit_cast(f16x8, raw);
          uint32_t x[4], y[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float u = (float)f[2 * e], v = (float)f[2 * e + 1];
            x[e] = vtx::bf16_pair(u, v);
            y[e] = vtx::bf16_pair(u - vtx::bf16_lo(x[e]), v - vtx::bf16_hi(x[e]));
          }
          w.q[j] = vtx::U4{x[0], x[1], x[2], x[3]};
          w.ql[j] = vtx::U4{y[0], y[1], y[2], y[3]};
        } else {
          w.q[j] = raw;
        }
      }
    }
    const float slope = a.slopes ? a.slopes[h * G + (c16 < G ? c16 : 0)] * kLog2e : 0.f;

    for (int pc = pa; pc < pb; pc += kStage) {
      const int np = min(kStage, pb - pc);
      __syncthreads();  // (the staged rows before are done with)
      for (int i = tid; i < np; i += kThreads) {
        const int r = a.indices[sg.start + pc + i];
        s_rows[i] = r >= 0 && r < a.rows ? r : -1;
      }
      __syncthreads();
      // tokens of these pages, numbered from the first of them
      const int n = (pc + np == sg.pages ? sg.tokens : (pc + np) * P) - pc * P;
      const int skip = pc == 0 ? sg.skip : 0;
      const int tiles = (n + kTile - 1) / kTile;
      const float far0 = (float)(sg.tokens - 1 - pc * P - 4 * g4);

      auto load = [&](int i, Tile<kD>& t) {
        if constexpr (kPages16) {
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            const int t0 = i * kTile + hf * 16;  // uniform
            const int pg = a.p_shift >= 0 ? t0 >> a.p_shift : t0 / P;
            const int r = vtx::uniform(s_rows[pg < np ? pg : 0]);
            t.ok[hf] = pg < np && r >= 0;
            const long long row = (long long)(r >= 0 ? r : 0) * P + (pg < np ? t0 - pg * P : 0);
            const unsigned char* kp = a.k + row * kD;
            const unsigned char* vp = a.v + row * kD;
#pragma unroll
            for (int j = 0; j < kD / 64; ++j) t.k[hf][j] = vtx::ld16_stream(kp + (c16 * kD + j * 64 + g4 * 16));
#pragma unroll
            for (int x = 0; x < 4; ++x) load_v<kD>(vp + ((4 * g4 + x) * kD + c16 * (kD / 16)), t.v[hf][x]);
            t.sc[hf] = *reinterpret_cast<const uint2*>(a.scales + row * 2 + 8 * g4);
          }
        } else {
          t.bad = 0;
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            auto row_of = [&](int tok, bool& ok) {
              ok = tok < n;
              const int pg = ok ? tok / P : 0;
              const int r = s_rows[pg];
              ok = ok && r >= 0;
              return ok ? (long long)r * P + (tok - pg * P) : 0LL;
            };
            bool ok;
            const unsigned char* kp = a.k + row_of(i * kTile + hf * 16 + c16, ok) * kD;
#pragma unroll
            for (int j = 0; j < kD / 64; ++j) t.k[hf][j] = vtx::ld16_stream(kp + (j * 64 + g4 * 16));
            uint32_t two[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const long long row = row_of(i * kTile + hf * 16 + 4 * g4 + x, ok);
              load_v<kD>(a.v + row * kD + c16 * (kD / 16), t.v[hf][x]);
              two[x] = *reinterpret_cast<const uint16_t*>(a.scales + row * 2);
              t.bad |= ok ? 0u : 1u << (4 * hf + x);
            }
            t.sc[hf] = uint2{two[0] | (two[1] << 16), two[2] | (two[3] << 16)};
          }
        }
      };
      auto compute = [&](int i, Tile<kD>& t) {
        uint32_t bad = 0;
        bool masked = i * kTile + kTile > n || i * kTile < skip;
        if constexpr (kPages16) masked = masked || !t.ok[0] || !t.ok[1];
        else masked = masked || __ballot(t.bad != 0) != 0;
        if (masked) {  // uniform
          if constexpr (kPages16) bad = (t.ok[0] ? 0u : 0xfu) | (t.ok[1] ? 0u : 0xf0u);
          else bad = t.bad;
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            const int tok = i * kTile + 16 * (x / 4) + 4 * g4 + x % 4;
            bad |= tok >= n || tok < skip ? 1u << x : 0u;
          }
        }
        attend<kD, kCodes, kHalf>(a, w, t, masked, bad, far0 - (float)(i * kTile), slope);
      };
      for (int i = wave; i < tiles; i += kWaves) {
        Tile<kD> t;
        load(i, t);
        compute(i, t);
      }
    }

    // the waves' results joined in LDS: the segment's, or this part of it
    float l = w.l + vtx::xshfl(w.l, 16);
    l += vtx::xshfl(l, 32);
    // (a maximum passes NaN scores by; where nothing else was seen it is still
    // -inf, which the joins take for no tokens)
    const float m = l != l ? 0.f : w.m;
    if (c16 < G) {
      if (g4 == 0) {
        s_m[wave][c16] = m;
        s_l[wave][c16] = l;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int x4 = 0; x4 < kD / 64; ++x4)
          *reinterpret_cast<float4*>(&s_o[wave][c16][(4 * g4 + i) * (kD / 16) + 4 * x4]) =
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
          const float4 y = *reinterpret_cast<const float4*>(&s_o[i][g][d]);
          L = fmaf(s_l[i][g], f, L);
          O = float4{fmaf(y.x, f, O.x), fmaf(y.y, f, O.y), fmaf(y.z, f, O.z), fmaf(y.w, f, O.w)};
        }
      }
      if (part) {  // uniform
        const long long row = (2LL * blockIdx.x + slot) * G + g;
        *reinterpret_cast<float4*>(a.acc + row * kD + d) = O;
        if (d == 0) a.ml[row] = float2{M, L};
      } else {
        const float f = inverse_sum(L);
        *reinterpret_cast<uint2*>(a.o + ((long long)seg * G + g) * kD + d) =
            uint2{round2<kHalf>(O.x * f, O.y * f), round2<kHalf>(O.z * f, O.w * f)};
      }
    }
    if (whole) return;  // uniform
    __syncthreads();  // (the next segment's results go to the same place)
  }
}

// The parts of a segment that lies in several ranges, joined; zeros for one
// without tokens.  A workgroup per segment: threads = (part of the parts, head,
// four columns), each with a running maximum of its own.
constexpr int kJoinThreads = 512;
template <int kD, bool kHalf>
__global__ __launch_bounds__(kJoinThreads) void quant_attention_join_kernel(QAttnArgs a) {
  constexpr int kAhead = 8;  // parts in flight
  __shared__ alignas(16) float s_o[kJoinThreads][4];
  __shared__ float2 s_ml[kJoinThreads];
  const int seg = blockIdx.x, tid = threadIdx.x, G = a.G, S = a.segments;
  const long long first = a.indptr[0];
  const Line l = line_of(a, first, a.indptr[S]);
  const Segment sg = segment_of(a, seg, first, a.indptr[seg], a.indptr[seg + 1], a.last_len[seg], l.total);
  int w0 = 0, n = 0;
  bool second = false;  // the first part lies behind another segment's
  if (sg.end > sg.at) {
    w0 = (int)(sg.at / l.per);
    n = (int)((sg.end - 1) / l.per) - w0 + 1;
    second = sg.at > (uint32_t)w0 * l.per;
    if (n == 1) return;  // uniform: written by its workgroup
  }
  const int items = G * (kD / 4);
  for (int x0 = 0; x0 < items; x0 += kJoinThreads) {
    // (items a multiple of 16: a group's size is a power of two times a head count)
    const int here = min(items - x0, kJoinThreads), groups = kJoinThreads / here;
    const int x = tid % here, grp = tid / here;
    const int g = (x0 + x) / (kD / 4), d = ((x0 + x) % (kD / 4)) * 4;
    float M = -INFINITY, L = 0.f;
    float4 O{0.f, 0.f, 0.f, 0.f};
    if (grp < groups) {
      for (int i0 = grp; i0 < n; i0 += groups * kAhead) {
        float2 ml[kAhead];
        float4 y[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int i = i0 + u * groups < n ? i0 + u * groups : i0;
          const long long row = (2LL * (w0 + i) + (i == 0 && second ? 1 : 0)) * G + g;
          ml[u] = a.ml[row];
          y[u] = *reinterpret_cast<const float4*>(a.acc + row * kD + d);
        }
        float nm = M;
#pragma unroll
        for (int u = 0; u < kAhead; ++u) nm = fmaxf(nm, ml[u].x);
        if (nm == -INFINITY) continue;
        const float f = __builtin_amdgcn_exp2f(M - nm);
        L *= f;
        O = float4{O.x * f, O.y * f, O.z * f, O.w * f};
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const float e = i0 + u * groups < n ? __builtin_amdgcn_exp2f(ml[u].x - nm) : 0.f;
          if (i0 + u * groups < n) {
            L = fmaf(ml[u].y, e, L);
            O = float4{fmaf(y[u].x, e, O.x), fmaf(y[u].y, e, O.y), fmaf(y[u].z, e, O.z), fmaf(y[u].w, e, O.w)};
          }
        }
        M = nm;
      }
    }
    __syncthreads();
    s_ml[tid] = float2{M, L};
    *reinterpret_cast<float4*>(s_o[tid]) = O;
    __syncthreads();
    if (grp == 0) {
      for (int i = 1; i < groups; ++i) {
        const float2 ml = s_ml[i * here + x];
        const float4 y = *reinterpret_cast<const float4*>(s_o[i * here + x]);
        const float nm = fmaxf(M, ml.x);
        if (nm == -INFINITY) continue;
        const float f = __builtin_amdgcn_exp2f(M - nm), e = __builtin_amdgcn_exp2f(ml.x - nm);
        L = L * f + ml.y * e;
        O = float4{O.x * f + y.x * e, O.y * f + y.y * e, O.z * f + y.z * e, O.w * f + y.w * e};
        M = nm;
      }
      const float f = inverse_sum(L);
      *reinterpret_cast<uint2*>(a.o + ((long long)seg * G + g) * kD + d) =
          uint2{round2<kHalf>(O.x * f, O.y * f), round2<kHalf>(O.z * f, O.w * f)};
    }
  }
}

template <int kD, int kCodes, bool kHalf>
int launch_one(const QAttnArgs& a, hipStream_t s) {
  const int grid = a.workers > 0 ? a.workers : a.segments;
  if (a.P % 16 == 0) quant_attention_kernel<kD, kCodes, kHalf, true><<<grid, kThreads, 0, s>>>(a);
  else quant_attention_kernel<kD, kCodes, kHalf, false><<<grid, kThreads, 0, s>>>(a);
  if (a.workers > 0) quant_attention_join_kernel<kD, kHalf><<<a.segments, kJoinThreads, 0, s>>>(a);
  return vtx::check_launch("quant_decode_attention");
}

template <int kD>
int launch_types(const QAttnArgs& a, int codes, bool half, hipStream_t s) {
  if (codes == VTX_CODES_E4M3)
    return half ? launch_one<kD, VTX_CODES_E4M3, true>(a, s) : launch_one<kD, VTX_CODES_E4M3, false>(a, s);
  return half ? launch_one<kD, VTX_CODES_INT8, true>(a, s) : launch_one<kD, VTX_CODES_INT8, false>(a, s);
}

// Ranges of a call: as many workgroups as the card holds at once, and no more
// than the buffer's pages can fill.
struct Ranges {
  long long workers, least, pitch;
};
Ranges ranges_of(long long segments, int32_t head_dim, int32_t page_size, int32_t window, long long indices_len) {
  const int cus = vtx::device_cu_count() > 0 ? vtx::device_cu_count() : 256;
  Ranges r;
  r.least = (kMinTokens + (long long)page_size - 1) / page_size;
  r.pitch = window > 0 ? ((long long)window + page_size - 1) / page_size + 1 : 0;
  if (r.pitch * segments > 0x7fffffffLL) r.pitch = 0;  // (a window past any segment: the pages as they are)
  const long long line = r.pitch > 0 ? r.pitch * segments : indices_len;
  r.workers = (long long)cus * (head_dim == 256 ? 2 : (head_dim == 128 ? 3 : 4));
  const long long need = (line + r.least - 1) / r.least;
  if (r.workers > need) r.workers = need;
  if (r.workers < 1) r.workers = 1;
  return r;
}

}  // namespace

extern "C" int vtx_quant_decode_attention_supported(int32_t head_dim, int32_t group_size) {
  return (head_dim == 64 || head_dim == 128 || head_dim == 256) && group_size >= 1 && group_size <= kHeads;
}

extern "C" int64_t vtx_quant_decode_attention_workspace_len(int32_t batch_size, int32_t num_kv_heads,
                                                            int32_t group_size, int32_t head_dim, int32_t page_size,
                                                            int32_t window, int64_t kv_indices_len) {
  if (batch_size < 1 || num_kv_heads < 1 || page_size < 1 || window < 0 || kv_indices_len < 0 ||
      !vtx_quant_decode_attention_supported(head_dim, group_size))
    return 0;
  const Ranges r = ranges_of((long long)batch_size * num_kv_heads, head_dim, page_size, window, kv_indices_len);
  return 2 * r.workers * group_size * (head_dim + 2);
}

extern "C" int vtx_quant_decode_attention(const void* q, const int64_t* q_strides, void* o, const void* k_cache,
                                          const void* v_cache, const void* scales, int64_t cache_rows,
                                          const int32_t* kv_indptr, const int32_t* kv_indices, int64_t kv_indices_len,
                                          const int32_t* kv_last_page_len, int32_t batch_size, int32_t num_kv_heads,
                                          int32_t group_size, int32_t head_dim, int32_t page_size, int32_t dtype,
                                          int32_t codes, float sm_scale, float soft_cap, int32_t window,
                                          const float* slopes, float* workspace, int64_t workspace_len, void* stream) {
  vtx::clear_error();
  if (batch_size < 0 || num_kv_heads < 1 || page_size < 1 || cache_rows < 0 || kv_indices_len < 0 || window < 0)
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
  if (segments > 0x3fffffffLL || kv_indices_len > 0x7fffffffLL)
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
  a.c = soft_cap > 0.f ? 2.f * kLog2e * (sm_scale / soft_cap) : sm_scale * kLog2e;
  a.cap = soft_cap * kLog2e;
  a.pitch = 0;
  a.workers = 0;
  a.least = 1;
  a.acc = nullptr;
  a.ml = nullptr;
  if (workspace) {
    const Ranges r = ranges_of(segments, head_dim, page_size, window, kv_indices_len);
    const long long parts = 2 * r.workers * group_size;
    if (workspace_len < parts * (head_dim + 2) || !vtx::aligned16(workspace))
      return vtx::fail(VTX_E_INVALID,
                       "quant_decode_attention: workspace of %lld floats (16-byte aligned) needed, got %lld",
                       parts * (long long)(head_dim + 2), (long long)workspace_len);
    a.workers = (int32_t)r.workers;
    a.least = (int32_t)r.least;
    a.pitch = (int32_t)r.pitch;
    a.acc = workspace;
    a.ml = reinterpret_cast<float2*>(workspace + parts * head_dim);
  }
  hipStream_t s = vtx::as_stream(stream);
  const bool half = dtype == VTX_DTYPE_F16;
  switch (head_dim) {
    case 64: return launch_types<64>(a, codes, half, s);
    case 128: return launch_types<128>(a, codes, half, s);
    default: return launch_types<256>(a, codes, half, s);
  }
}
