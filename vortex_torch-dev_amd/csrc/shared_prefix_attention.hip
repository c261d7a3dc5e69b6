// Decode attention for requests that share leading pages, for gfx950: the
// result of paged decode attention over the same block table, with a shared
// page read once for all requests of its run instead of once for each.
//
// For a query row and the tokens t of its segment,
//   o = sum_t p_t V[t] / sum_t p_t,  p_t = 2^(c q.K[t] - m),  c = scale log2 e
// over any partition of the tokens into chunks, each with its own m, the joint
// sums follow from the chunks' (m, sum p, sum p V) weighted by 2^(m - max m).
// So the plan's items (vtx_shared_prefix.h) are independent: the rows of a run
// against a chunk of its shared pages, or those of a request against a chunk
// of its own; a second launch joins the partial results (fp32).
//
// Both products run on the matrix cores (v_mfma_f32_32x32x16_bf16), transposed
// so that a lane holds one query row: S^T = K Q^T (32 tokens x 32 rows per
// step, fp32) leaves lane l with row l % 32 and half of the 32 tokens, so the
// softmax is in the lane but for one exchange of halves; rounded to bf16, those
// registers are the B operand of O^T = V^T P^T as they stand, if V^T's tokens
// are taken in the same order, which is the transposing LDS read's addressing.
// P is rounded to bf16 for the matrix cores; the sums are taken of the rounded
// values, so the weights sum to one and a mean of V is not shifted.
//
// 4 waves.  Up to 32 rows (a request's own pages): every wave takes tiles of 32
// tokens of its own, through registers, or all tiles of a short request of its
// own.  More: tiles of 64 tokens for all waves, of which each takes 32 rows (or
// 32 rows and 32 tokens where there are up to 64 rows), two buffers, copied
// straight to LDS one tile ahead.
//
// Bound by HBM up to about 150 rows (5.7 TB/s in 32 runs of 8 requests behind 4k
// tokens), by the matrix cores, what feeds them and the exponentials beyond (886
// TFLOP/s over both launches for 2048 rows and 8 heads behind 16k tokens, 155 us).
#include "vtx_shared_prefix.h"

#include <type_traits>

#include "vtx_device.h"
#include "vtx_host.h"

namespace {

using namespace vtx_prefix;

struct SharedArgs {
  const uint16_t* q;
  uint16_t* o;
  const uint16_t* k;
  const uint16_t* v;
  int64_t rows;  // pool rows (page * H + h)
  uint32_t pool_bytes;  // 0: over 4 GiB
  const int32_t* indices;
  int64_t indices_len;
  const int32_t* last_len;
  const int32_t* counts;   // items of a head
  const Item* items;
  const int32_t* combine;  // [segments][kCombineInts]
  int32_t most_items;
  int32_t B, H, G, P, p_shift;
  float c;          // |scale| log2 e, or 1 for a scale of 0
  uint32_t q_sign;  // flips the queries' signs for a negative scale
  uint32_t q_keep;  // 0 for a scale of 0: no scores
  float* acc;       // [max_rows, D]
  float2* ml;       // [max_rows]
  int64_t max_rows;  // of all heads
  bool join_four;
};

constexpr int kThreads = 256;
constexpr int kWaves = 4;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s16x4 lds4;

// Classes of instructions for the scheduler's groups.
constexpr int kSchedValu = 0x2, kSchedMfma = 0x8, kSchedRead = 0x100;
constexpr int kWeighOps = 24;  // instructions of a step's weights

// LDS rows of a tile are kD bf16 in 16-byte pieces; piece c of token t lies at
// c ^ swizzle(t), so that the 8 (or 16) tokens of a K read, at one c, and the
// 8 tokens x 4 pieces of a transposing V read spread over all banks.
template <int kD>
__device__ __forceinline__ int swizzle(int t) {
  if constexpr (kD == 64) return (((t >> 1) & 1) << 2) | (((t >> 2) & 1) << 1) | ((t >> 3) & 1);
  return ((t & 3) << 2) | ((t >> 2) & 3);
}

// Orders a wave's LDS accesses around it (its lanes read what others wrote;
// the hardware keeps a wave's LDS operations in order).
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Copies from a pool straight to LDS, 16 bytes per lane: lane l's, `at` elements
// into the pool, to `to` (uniform) + 16 l.  Pools of up to 4 GiB (kFar false) take
// buffer loads: 32-bit offsets, and LDS reads behind a copy in flight are waited
// for one by one; behind the other form, which counts as an LDS operation too, the
// compiler waits for all of them (256 requests of 8 heads each behind 16k tokens:
// 155 us a layer, 159 by the other form).
template <bool kFar>
struct Pool {
  const uint16_t* base;
  __amdgpu_buffer_rsrc_t buffer;
  __device__ __forceinline__ Pool(const uint16_t* p, uint32_t bytes) : base(p) {
    if constexpr (!kFar) buffer = __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, (int)bytes, 0x27000);
  }
  __device__ __forceinline__ void copy(uint32_t row, int log2_row, uint32_t within, void* to) const {
    auto* lds = (__attribute__((address_space(3))) void*)to;
    if constexpr (kFar) {
      const uint16_t* from = base + (((uint64_t)row << log2_row) + within);
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from, lds, 16, 0, 0);
    } else {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(buffer, lds, 16, (int)(((row << log2_row) + within) * 2u), 0, 0, 0);
    }
  }
};
// Waits for this wave's copies (and other loads).
__device__ __forceinline__ void copies_done() { __builtin_amdgcn_s_waitcnt(0x0f70); }

// Output columns of a wave: all, or half of 256 (two waves share 32 rows and
// both compute their scores: with all columns a lane's outputs and queries leave
// no registers for more).
template <int kD>
constexpr int kCols = kD == 256 ? 128 : kD;
// Tokens of a tile that all waves share.
template <int kD>
constexpr int kTile = kD == 256 ? 32 : 64;

// A wave's 32 query rows: their fragments, running maximum (scaled, base 2),
// sum (this lane's half of the tokens) and output.
template <int kD>
struct Rows {
  vtx::U4 q[kD / 16];
  float m, l;
  f32x16 o[kCols<kD> / 32];
};

// The running maximum follows the scores only when they outgrow it by so much
// (base 2): until then weights up to 2^8 are as exact as weights up to 1, and
// most tiles leave the outputs as they are (256 requests of 8 heads each behind
// 16k tokens 155 us a layer, following every maximum 159).
constexpr float kGrowth = 8.f;

// kN x 32 tokens at kt / vt in LDS; bit i of mask: token i counts.  kAhead: the
// LDS reads are kept ahead of the products that take them (registers allowing).
// col: the wave's first output column / 8.
template <int kD, int kN, bool kAhead>
__device__ __forceinline__ void attend(Rows<kD>& w, const unsigned char* kt, const unsigned char* vt, uint64_t mask,
                                       float c, int col) {
  constexpr int kRow = kD * 2, kBlocks = kCols<kD> / 32;
  const int lane = vtx::lane_id(), r = lane % 32, half = lane / 32;
  f32x16 s[kN];
#pragma unroll
  for (int n = 0; n < kN; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) s[n][i] = 0.f;
  const int ksw = swizzle<kD>(r);
#pragma unroll
  for (int kk = 0; kk < kD / 16; ++kk)
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      const vtx::U4 f = vtx::ld16(kt + (n * 32 + r) * kRow + (((2 * kk + half) ^ ksw) << 4));
      s[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, f), __builtin_bit_cast(bf16x8, w.q[kk]),
                                                     s[n], 0, 0, 0);
    }
  // V^T of the first 16 tokens, on the way during the softmax: 16 lanes take 4
  // tokens x 16 columns per read
  const int g16 = lane / 16, i16 = lane % 16;
  const int vrow = 4 * half + i16 / 4;
  const int vcol = col + (g16 & 1) * 2 + (i16 % 4) / 2;
  constexpr int kSteps = 2 * kN;  // 16 tokens each
  s16x4 f[kAhead ? 2 : 1][kBlocks][2];
  auto read_v = [&](int k, s16x4 (&to)[kBlocks][2]) {
#pragma unroll
    for (int d = 0; d < kBlocks; ++d)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int t = vrow + 8 * e;  // (+ 16 k, which the swizzle does not see)
        const unsigned char* at =
            vt + (k * 16 + t) * kRow + (((d * 4 + vcol) ^ swizzle<kD>(t)) << 4) + (i16 % 2) * 8;
        to[d][e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)at);
      }
  };
  if constexpr (kAhead) {
    read_v(0, f[0]);
    constexpr int kReads = kN * (kD / 16), kLead = kReads < 8 ? kReads : 8;
    __builtin_amdgcn_sched_group_barrier(kSchedRead, kLead, 0);
#pragma unroll
    for (int i = 0; i < kReads; ++i) {
      __builtin_amdgcn_sched_group_barrier(kSchedMfma, 1, 0);
      __builtin_amdgcn_sched_group_barrier(kSchedRead, 1, 0);
    }
  }
  constexpr uint64_t kAll = kN == 2 ? ~0ull : 0xffffffffull;
  if ((mask & kAll) != kAll) {  // uniform
    const uint64_t mine = mask >> (4 * half);
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      const uint32_t bits = (uint32_t)(mine >> (32 * n));
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (!(bits & (1u << (8 * (i / 4) + i % 4)))) s[n][i] = -INFINITY;
    }
    asm volatile("" : "+v"(s[0][0]));  // (a branch, not selects in every tile)
  }
  float mx = s[0][0];
#pragma unroll
  for (int n = 0; n < kN; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[n][i]);
  mx = fmaxf(mx, vtx::xshfl(mx, 32)) * c;
  if (__ballot(mx > w.m + kGrowth)) {  // uniform
    const float nm = fmaxf(w.m, mx);
    const float f = nm == -INFINITY ? 1.f : exp2_fast(w.m - nm);
    w.l *= f;
#pragma unroll
    for (int d = 0; d < kBlocks; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) w.o[d][i] *= f;
    w.m = nm;
  }
  const float base = w.m == -INFINITY ? 0.f : w.m;
  // P of step k: 16 tokens
  auto weigh = [&](int k) {
    uint32_t p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int x = 8 * (k & 1) + 2 * i;
      p[i] = vtx::bf16_pair(exp2_fast(fmaf(s[k / 2][x], c, -base)), exp2_fast(fmaf(s[k / 2][x + 1], c, -base)));
      w.l = vtx::dot2_bf16(p[i], 0x3f803f80u, w.l);
    }
    return vtx::U4{p[0], p[1], p[2], p[3]};
  };
  auto product = [&](const vtx::U4& b, const s16x4 (&f)[kBlocks][2]) {
#pragma unroll
    for (int d = 0; d < kBlocks; ++d) {
      const s16x8 a = __builtin_shufflevector(f[d][0], f[d][1], 0, 1, 2, 3, 4, 5, 6, 7);
      w.o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b),
                                                       w.o[d], 0, 0, 0);
    }
  };
  if constexpr (kAhead) {
    // The weights of a step between the products of the one before, its V reads
    // before them.
    if (kSteps > 1) read_v(1, f[1]);
    vtx::U4 b = weigh(0);
    __builtin_amdgcn_sched_group_barrier(kSchedRead, kSteps > 1 ? 2 * kBlocks : 0, 1);
    __builtin_amdgcn_sched_group_barrier(kSchedValu, kWeighOps, 1);
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      product(b, f[k & 1]);
      if (k + 1 < kSteps) b = weigh(k + 1);
      if (k + 2 < kSteps) read_v(k + 2, f[k & 1]);
#pragma unroll
      for (int d = 0; d < kBlocks; ++d) {
        __builtin_amdgcn_sched_group_barrier(kSchedMfma, 1, 1);
        if (k + 1 < kSteps) __builtin_amdgcn_sched_group_barrier(kSchedValu, kWeighOps / kBlocks, 1);
      }
      if (k + 2 < kSteps) __builtin_amdgcn_sched_group_barrier(kSchedRead, 2 * kBlocks, 1);
    }
  } else {
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      read_v(k, f[0]);
      product(weigh(k), f[0]);
    }
  }
}

// The tokens of an item: where they lie in the table, and how many.
struct Tokens {
  const int32_t* pages;
  int count;
};

// Pool token row (page row * P + slot) of token t, and whether it exists and
// lies inside the pool; 0 (a valid row) where it does not.  In two steps, the
// table entry requested a tile before it is needed.
struct Entry {
  int page, slot;  // page: the table's entry, -1 past the last token
};
__device__ __forceinline__ Entry entry_of(const SharedArgs& a, const Tokens& tk, int t) {
  Entry e{-1, 0};
  if (t < tk.count) {
    const int pg = a.p_shift >= 0 ? t >> a.p_shift : t / a.P;
    e.slot = t - pg * a.P;
    e.page = tk.pages[pg];
  }
  return e;
}
__device__ __forceinline__ bool resolve(const SharedArgs& a, const Entry& e, uint32_t& row) {
  const bool ok = e.page >= 0 && e.page < a.rows;
  row = ok ? (uint32_t)e.page * (uint32_t)a.P + (uint32_t)e.slot : 0u;
  return ok;
}

// A result row: four columns of it from sums O and L.
__device__ __forceinline__ uint2 result4(const float4& O, float L) {
  const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : NAN);
  return uint2{vtx::bf16_pair(O.x * inv, O.y * inv), vtx::bf16_pair(O.z * inv, O.w * inv)};
}

// A wave's maximum and sum, whole, as they leave it.  A maximum passes NaN scores
// by, so rows of which nothing else was seen still have -inf, which the joins
// take for "no tokens": they get a finite one, and their NaN stays in every sum.
struct Stats {
  float m, l;
};
template <int kD>
__device__ __forceinline__ Stats stats_of(const Rows<kD>& w) {
  const float l = w.l + vtx::xshfl(w.l, 32);
  return Stats{l != l ? 0.f : w.m, l};
}

// A wave's output to its stretch of LDS: row r's 16-byte piece x at x ^ r.
template <int kD>
__device__ __forceinline__ void spread(const Rows<kD>& w, float* to) {
  constexpr int kOut = kCols<kD> / 4;
  const int r = vtx::lane_id() % 32, half = vtx::lane_id() / 32;
#pragma unroll
  for (int d = 0; d < kCols<kD> / 32; ++d)
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int pc = (d * 8 + x * 2 + half) ^ (r % kOut);
      *reinterpret_cast<float4*>(to + (r * kOut + pc) * 4) =
          float4{w.o[d][4 * x], w.o[d][4 * x + 1], w.o[d][4 * x + 2], w.o[d][4 * x + 3]};
    }
}

// The result of a wave that has a request of its own: its `rows` rows to
// partial rows `out`, or finished to query rows q0 .. (out < 0).
template <int kD>
__device__ __forceinline__ void leave_apart(const SharedArgs& a, const Rows<kD>& w, float* lds, int rows, int out,
                                            long long q0) {
  constexpr int kOut = kD / 4;
  const int lane = vtx::lane_id();
  const Stats st = stats_of(w);
  spread<kD>(w, lds);
  wave_lds_fence();
  if (out >= 0 && (long long)out + rows > a.max_rows) return;
  for (int x0 = 0; x0 < rows * kOut; x0 += vtx::kWave) {
    const int x = x0 + lane, r = x / kOut, pc = x % kOut;
    const float L = __shfl(st.l, r % 32);
    if (r >= rows) continue;
    const float4 O = reinterpret_cast<const float4*>(lds)[r * kOut + (pc ^ (r % kOut))];
    if (out < 0) *reinterpret_cast<uint2*>(a.o + (q0 + r) * kD + pc * 4) = result4(O, L);
    else *reinterpret_cast<float4*>(a.acc + ((long long)out + r) * kD + pc * 4) = O;
  }
  if (out >= 0 && lane < rows) a.ml[(long long)out + lane] = float2{st.m, st.l};
}

template <int kD, bool kFar>
__global__ __launch_bounds__(kThreads, kD == 64 ? 3 : 2) void shared_prefix_attention_kernel(SharedArgs a) {
  constexpr int kRow = kD * 2;
  constexpr int kPieces = kD / 8;
  constexpr int kBlocks = kCols<kD> / 32;
  constexpr int kShare = kD / kCols<kD>;  // waves that share rows
  constexpr int kGroups = kWaves / kShare;
  // Two buffers of a tile (its K and V), or every wave's 32 tokens; then the waves'
  // outputs.  Arrays of their own, so that the compiler sees which of them a copy
  // in flight writes and lets the reads of the others pass it.
  __shared__ alignas(16) unsigned char s_k0[kTile<kD> * kRow], s_v0[kTile<kD> * kRow], s_k1[kTile<kD> * kRow],
      s_v1[kTile<kD> * kRow];
  auto part = [&](int i) -> unsigned char* { return i == 0 ? s_k0 : (i == 1 ? s_v0 : (i == 2 ? s_k1 : s_v1)); };
  __shared__ float s_m[kWaves][32];
  __shared__ float s_l[kWaves][32];

  const int h = blockIdx.x % (uint32_t)a.H, nth = blockIdx.x / (uint32_t)a.H;
  const Item it = a.items[(int64_t)h * a.most_items + nth];  // (past the head's last one not used)
  if (nth >= a.counts[h]) return;  // uniform
  const int tid = threadIdx.x, lane = vtx::lane_id();
  const int wave = vtx::uniform(tid / vtx::kWave);
  const int seg = vtx::uniform(it.segment), S = a.B * a.H;
  if (seg < 0 || seg >= S) return;
  const bool apart = it.last == kApart;  // uniform
  int b0 = seg / a.H, rows = min(max(it.rows, 0), tile_rows(kD)), out = it.out;
  int start = it.start, pages = it.pages, last_of = it.last ? seg : -1;
  if (apart) {  // this wave's request
    b0 += wave;
    if (wave >= pages || b0 >= a.B) return;  // (no barriers on this way)
    last_of = b0 * a.H + h;
    const int32_t* info = a.combine + (long long)kCombineInts * last_of;
    if (vtx::uniform(info[4]) == 0) return;
    out = info[1] == 0 ? -1 : info[3];
    start = vtx::uniform(info[5]);
    pages = vtx::uniform(info[6]);
  }

  // the item's tokens
  Tokens tk{nullptr, 0};
  if (start >= 0 && pages > 0 && (long long)start + pages <= a.indices_len && a.rows > 0) {
    int last = a.P;
    if (last_of >= 0) last = min(max(a.last_len[last_of], 0), a.P);
    const long long t = (long long)(pages - 1) * a.P + last;
    tk.pages = a.indices + start;
    tk.count = (int)(t < 0x3fffffff ? t : 0x3fffffff);
  }

  // blocks of 32 rows, a power of two; this wave's, its tokens among the waves
  // that have the same rows, and its columns
  const int wr = rows > 64 ? 4 : (rows > 32 ? 2 : 1);
  const int half_col = wave % kShare, rb = (wave / kShare) % wr, tb = (wave / kShare) / wr, wt = kGroups / wr;
  Rows<kD> w;
  w.m = -INFINITY;
  w.l = 0.f;
#pragma unroll
  for (int d = 0; d < kBlocks; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) w.o[d][i] = 0.f;
  {
    const int r = rb * 32 + lane % 32, at = (int)((uint32_t)it.row0 + r);
    const int b = (int)((uint32_t)b0 + (uint32_t)(at / a.G)), g = at % a.G;
    const bool ok = r < rows && at >= 0 && (uint32_t)b < (uint32_t)a.B;
    const uint16_t* q = a.q + (((long long)(ok ? b : b0) * a.H + h) * a.G + (ok ? g : 0)) * kD + (lane / 32) * 8;
    const uint32_t keep = ok ? a.q_keep : 0u;
#pragma unroll
    for (int kk = 0; kk < kD / 16; ++kk) {
      const vtx::U4 x = vtx::ld16(q + kk * 16);
      w.q[kk] = vtx::U4{(x.x & keep) ^ a.q_sign, (x.y & keep) ^ a.q_sign, (x.z & keep) ^ a.q_sign,
                        (x.w & keep) ^ a.q_sign};
    }
  }

  // tiles of 32 tokens, wave w those of index w, w + 4, ...; or all, of its own request
  bool alone = false;
  if constexpr (kShare == 1) alone = wr == 1;
  if (alone) {  // uniform
    constexpr int kPass = vtx::kWave / kPieces;  // tokens per wave-wide load
    constexpr int kLoads = 32 / kPass;
    unsigned char* kt = part(wave);
    unsigned char* vt = kt + 32 * kRow;
    const int piece = lane % kPieces, sub = lane / kPieces;
    const int t0 = apart ? 0 : wave * 32, step = apart ? 32 : kWaves * 32;
    const int n = tk.count > t0 ? (tk.count - t0 + step - 1) / step : 0;
    vtx::U4 kr[kLoads], vr[kLoads];
    uint64_t next_mask = 0;
    Entry e = entry_of(a, tk, t0 + lane % 32);
    auto request = [&](int j) __attribute__((always_inline)) {  // tile j's rows, and the entries of tile j + 1
      uint32_t row;
      const bool ok = resolve(a, e, row);
      next_mask = __ballot(ok) & 0xffffffffull;
      e = entry_of(a, tk, t0 + (j + 1) * step + lane % 32);
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const uint32_t tr = (uint32_t)__shfl((int)row, i * kPass + sub);
        kr[i] = vtx::ld16_stream(a.k + (uint64_t)tr * kD + piece * 8);
        vr[i] = vtx::ld16_stream(a.v + (uint64_t)tr * kD + piece * 8);
      }
    };
    if (n > 0) request(0);
    for (int j = 0; j < n; ++j) {
      const uint64_t mask = next_mask;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int t = i * kPass + sub;
        const int at = t * kRow + ((piece ^ swizzle<kD>(t)) << 4);
        const uint32_t live = (mask >> t) & 1 ? ~0u : 0u;  // (what lies in a masked row may be NaN)
        vtx::st16(kt + at, kr[i]);
        vtx::st16(vt + at, vtx::U4{vr[i].x & live, vr[i].y & live, vr[i].z & live, vr[i].w & live});
      }
      wave_lds_fence();
      if (j + 1 < n) request(j + 1);
      attend<kD, 1, false>(w, kt, vt, mask, a.c, 0);
      wave_lds_fence();
    }
  } else {  // uniform: tiles of kTile tokens for all waves
    constexpr int kT = kTile<kD>;
    constexpr uint64_t kFull = kT == 64 ? ~0ull : (1ull << kT) - 1;
    constexpr int kPass = vtx::kWave / kPieces;  // tokens per wave-wide copy
    constexpr int kCopies = kT / (kPass * kWaves);
    constexpr int kLog2 = kD == 64 ? 6 : (kD == 128 ? 7 : 8);
    const Pool<kFar> pool_k(a.k, a.pool_bytes), pool_v(a.v, a.pool_bytes);
    const int tiles = (tk.count + kT - 1) / kT;
    const int col = half_col * (kCols<kD> / 8);
    const bool busy = rb * 32 < rows && tb * 32 < kT;
    uint64_t next_mask = 0;
    Entry e = entry_of(a, tk, lane % kT);
    // Requests tile j: copies straight to LDS, every lane 16 bytes to its place in
    // the wave's stretch, so it is the piece it reads that follows the swizzle.
    auto request = [&](int j, unsigned char* kt, unsigned char* vt) __attribute__((always_inline)) {
      uint32_t row;
      const bool ok = resolve(a, e, row);
      next_mask = __ballot(ok) & kFull;
      e = entry_of(a, tk, (j + 1) * kT + lane % kT);
#pragma unroll
      for (int i = 0; i < kCopies; ++i) {
        const int t0 = (i * kWaves + wave) * kPass, t = t0 + lane / kPieces;
        const uint32_t from = (uint32_t)__shfl((int)row, t), within = ((lane % kPieces) ^ swizzle<kD>(t)) * 8;
        pool_k.copy(from, kLog2, within, kt + t0 * kRow);
        pool_v.copy(from, kLog2, within, vt + t0 * kRow);
      }
    };
    // The requested tile has arrived, this wave's part of it: what its copies left
    // in masked rows of V may be NaN.
    auto arrived = [&](unsigned char* vt) __attribute__((always_inline)) {
      copies_done();
      if (next_mask != kFull) {  // uniform
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
          const int t0 = (i * kWaves + wave) * kPass;
          if (!((next_mask >> (t0 + lane / kPieces)) & 1))
            vtx::st16(vt + t0 * kRow + lane * 16, vtx::U4{0u, 0u, 0u, 0u});
        }
      }
      __syncthreads();
    };
    auto tile = [&](auto all, uint64_t mask, unsigned char* kt, unsigned char* vt) __attribute__((always_inline)) {
      if (busy) {  // uniform over the wave
        if constexpr (decltype(all)::value) attend<kD, kT / 32, true>(w, kt, vt, mask, a.c, col);
        else attend<kD, 1, true>(w, kt + tb * 32 * kRow, vt + tb * 32 * kRow, mask >> (tb * 32), a.c, col);
      }
    };
    // all: every wave takes all tokens of a tile, for 32 rows of its own (or shared).
    auto all_tiles = [&](auto all) __attribute__((always_inline)) {
      request(0, s_k0, s_v0);
      arrived(s_v0);
      for (int j = 0; j < tiles; j += 2) {
        uint64_t mask = next_mask;
        if (j + 1 < tiles) request(j + 1, s_k1, s_v1);
        tile(all, mask, s_k0, s_v0);
        arrived(s_v1);  // (past the last tile: a barrier, and at most zeros)
        if (j + 1 < tiles) {
          mask = next_mask;
          if (j + 2 < tiles) request(j + 2, s_k0, s_v0);
          tile(all, mask, s_k1, s_v1);
          arrived(s_v0);
        }
      }
    };
    if (tiles > 0) {  // (loops of their own: each one's registers)
      if (kShare > 1 || wr == 4) all_tiles(std::true_type{});
      else if constexpr (kShare == 1) all_tiles(std::false_type{});
    }
  }

  if constexpr (kShare == 1)
    if (apart) {  // uniform
      leave_apart(a, w, reinterpret_cast<float*>(part(wave)), rows, out, ((long long)b0 * a.H + h) * a.G);
      return;
    }

  // The waves' results meet in LDS (rows in 16-byte pieces, piece x of row r at
  // x ^ r), and leave it joined and in whole rows.
  __syncthreads();
  constexpr int kOut = kCols<kD> / 4;  // pieces of a wave's part of an output row
  {
    const int r = lane % 32;
    const Stats st = stats_of(w);
    if (lane < 32) {
      s_m[wave][r] = st.m;
      s_l[wave][r] = st.l;
    }
    spread<kD>(w, reinterpret_cast<float*>(part(wave)));
  }
  __syncthreads();
  const bool direct = out < 0;
  if (!direct && (long long)out + rows > a.max_rows) return;  // uniform
  if (wt == 1) {  // uniform: nothing to join (and never direct: more than G rows)
    auto leave = [&](const unsigned char* from, int v) __attribute__((always_inline)) {
      const int r0 = (v / kShare) * 32, c0 = (v % kShare) * kCols<kD>;
      if (direct || r0 >= rows) return;  // uniform
      constexpr int kEach = 32 * kOut / kThreads;
      float4 y[kEach];
#pragma unroll
      for (int u = 0; u < kEach; ++u) {
        const int x = u * kThreads + tid, rl = x / kOut, pw = x % kOut;
        y[u] = reinterpret_cast<const float4*>(from)[rl * kOut + (pw ^ (rl % kOut))];
      }
#pragma unroll
      for (int u = 0; u < kEach; ++u) {
        const int x = u * kThreads + tid, rl = x / kOut, pw = x % kOut;
        if (r0 + rl < rows)
          *reinterpret_cast<float4*>(a.acc + ((long long)out + r0 + rl) * kD + c0 + pw * 4) = y[u];
      }
    };
    leave(s_k0, 0);
    leave(s_v0, 1);
    leave(s_k1, 2);
    leave(s_v1, 3);
    if (!direct && tid < rows)
      a.ml[(long long)out + tid] = float2{s_m[tid / 32 * kShare][tid % 32], s_l[tid / 32 * kShare][tid % 32]};
    return;
  }
  for (int x = tid; x < rows * (kD / 4); x += kThreads) {
    const int r = x / (kD / 4), pc = x - r * (kD / 4), rl = r % 32, blk = r / 32;
    const int share = pc / kOut, pw = pc % kOut;
    float M = -INFINITY;
    for (int i = 0; i < wt; ++i) M = fmaxf(M, s_m[(i * wr + blk) * kShare + share][rl]);
    float L = 0.f;
    float4 O{0.f, 0.f, 0.f, 0.f};
    if (M != -INFINITY) {
      for (int i = 0; i < wt; ++i) {
        const int v = (i * wr + blk) * kShare + share;
        const float f = exp2_fast(s_m[v][rl] - M);
        const float4 y = reinterpret_cast<const float4*>(part(v))[rl * kOut + (pw ^ (rl % kOut))];
        L = fmaf(s_l[v][rl], f, L);
        O.x = fmaf(y.x, f, O.x);
        O.y = fmaf(y.y, f, O.y);
        O.z = fmaf(y.z, f, O.z);
        O.w = fmaf(y.w, f, O.w);
      }
    }
    if (direct) {
      const int at = (int)((uint32_t)it.row0 + r), b = (int)((uint32_t)b0 + (uint32_t)(at / a.G)), g = at % a.G;
      if (at < 0 || (uint32_t)b >= (uint32_t)a.B) continue;
      *reinterpret_cast<uint2*>(a.o + (((long long)b * a.H + h) * a.G + g) * kD + pc * 4) = result4(O, L);
    } else {
      *reinterpret_cast<float4*>(a.acc + ((long long)out + r) * kD + pc * 4) = O;
      if (pc == 0) a.ml[(long long)out + r] = float2{M, L};
    }
  }
}

// A query row's partial results, weighted: by one wave, or by four that take
// every fourth batch of them and meet in LDS.  A partial row is read in 16-byte
// pieces, kAtOnce rows side by side in the wave; before it reads them, lane i
// weighs the i-th of up to 64 rows.  Four waves pay where a row has many (a layer
// by one / four: 48 requests of one behind 32k, D 64, 65 each, 31.4 / 29.1 us; 17
// behind 5k, D 256, 25 each, 24.3 / 22.0) and cost where not (64 of 4 behind 8k
// 27.6 / 28.6; 16 of 4 behind 4k, D 64, 12.8 / 14.4).
constexpr int kJoinFour = 5120;  // partial rows x columns from which on
constexpr int kJoinWaves = 4;
template <int kD, bool kFour>
__global__ __launch_bounds__(kJoinWaves* vtx::kWave) void shared_prefix_join_kernel(SharedArgs a) {
  constexpr int kPieces = kD / 4, kAtOnce = vtx::kWave / kPieces;
  constexpr int kAhead = kFour ? 8 : 4;  // loads in flight
  constexpr int kBatch = kFour ? kAtOnce * kAhead : vtx::kWave;
  __shared__ float s_ml[kFour ? kJoinWaves : 1][2];
  __shared__ float4 s_o[kFour ? kJoinWaves : 1][kPieces];
  const int wave = vtx::uniform(threadIdx.x / vtx::kWave), lane = vtx::lane_id();
  const int row = kFour ? blockIdx.x : blockIdx.x * kJoinWaves + wave;
  if (row >= a.B * a.H * a.G) return;  // uniform over the waves that meet
  const int seg = row / a.G, g = row - seg * a.G;
  const int32_t* info = a.combine + (long long)kCombineInts * seg;
  const int run_row = info[0], run_step = info[2], own_row = info[3];
  const int run_n = min(max(info[1], 0), a.most_items), own_n = min(max(info[4], 0), a.most_items);
  if (run_n == 0 && own_n == 1) return;  // written by its item
  const int n = run_n + own_n, sub = lane / kPieces, piece = lane % kPieces;
  auto at = [&](int i) -> long long {
    const long long r = i < run_n ? run_row + (long long)i * run_step + g : own_row + (long long)(i - run_n) * a.G + g;
    return r >= 0 && r < a.max_rows ? r : 0;
  };
  float M = -INFINITY, L = 0.f;
  float4 O{0.f, 0.f, 0.f, 0.f};
  for (int i0 = kFour ? wave * kBatch : 0; i0 < n; i0 += kFour ? kJoinWaves * kBatch : kBatch) {
    const int live = min(n - i0, kBatch);
    float4 x[kAhead];
    auto read = [&](int c) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        x[u] = reinterpret_cast<const float4*>(a.acc)[at(i0 + min(c + u * kAtOnce + sub, live - 1)) * kPieces + piece];
    };
    const float2 ml = a.ml[at(i0 + min(lane, live - 1))];
    read(0);
    float mx = ml.x;
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) mx = fmaxf(mx, vtx::xshfl(mx, d));
    const float nm = fmaxf(M, mx);
    if (nm == -INFINITY) continue;
    const float f = exp2_fast(M - nm);
    const float wgt = lane < live ? exp2_fast(ml.x - nm) : 0.f;
    L = fmaf(L, f, vtx::wave_sum(wgt * ml.y));
    O.x *= f;
    O.y *= f;
    O.z *= f;
    O.w *= f;
    M = nm;
    for (int c = 0; c < live; c += kAtOnce * kAhead) {
      if (c > 0) read(c);
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int i = c + u * kAtOnce + sub;
        const float wu = __shfl(wgt, min(i, vtx::kWave - 1));
        const bool on = i < live;  // (an unwritten row may hold anything)
        O.x = on ? fmaf(x[u].x, wu, O.x) : O.x;
        O.y = on ? fmaf(x[u].y, wu, O.y) : O.y;
        O.z = on ? fmaf(x[u].z, wu, O.z) : O.z;
        O.w = on ? fmaf(x[u].w, wu, O.w) : O.w;
      }
    }
  }
#pragma unroll
  for (int d = kPieces; d < vtx::kWave; d <<= 1) {
    O.x += vtx::xshfl(O.x, d);
    O.y += vtx::xshfl(O.y, d);
    O.z += vtx::xshfl(O.z, d);
    O.w += vtx::xshfl(O.w, d);
  }
  if constexpr (kFour) {
    if (lane == 0) {
      s_ml[wave][0] = M;
      s_ml[wave][1] = L;
    }
    if (lane < kPieces) s_o[wave][lane] = O;
    __syncthreads();
    if (threadIdx.x >= kPieces) return;
    M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kJoinWaves; ++w) M = fmaxf(M, s_ml[w][0]);
    L = 0.f;
    O = float4{0.f, 0.f, 0.f, 0.f};
    if (M != -INFINITY) {
#pragma unroll
      for (int w = 0; w < kJoinWaves; ++w) {
        const float f = exp2_fast(s_ml[w][0] - M);
        const float4 y = s_o[w][threadIdx.x];
        L = fmaf(s_ml[w][1], f, L);
        O.x = fmaf(y.x, f, O.x);
        O.y = fmaf(y.y, f, O.y);
        O.z = fmaf(y.z, f, O.z);
        O.w = fmaf(y.w, f, O.w);
      }
    }
  } else {
    if (lane >= kPieces) return;
  }
  reinterpret_cast<uint2*>(a.o + (long long)row * kD)[kFour ? threadIdx.x : lane] = result4(O, L);
}

template <int kD>
int launch(const SharedArgs& a, hipStream_t s) {
  if (a.pool_bytes) shared_prefix_attention_kernel<kD, false><<<a.H * a.most_items, kThreads, 0, s>>>(a);
  else shared_prefix_attention_kernel<kD, true><<<a.H * a.most_items, kThreads, 0, s>>>(a);
  const int rows = a.B * a.H * a.G;
  if (a.join_four)
    shared_prefix_join_kernel<kD, true><<<rows, kJoinWaves * vtx::kWave, 0, s>>>(a);
  else
    shared_prefix_join_kernel<kD, false><<<(rows + kJoinWaves - 1) / kJoinWaves, kJoinWaves * vtx::kWave, 0, s>>>(a);
  return vtx::check_launch("shared_prefix_decode_attention");
}

}  // namespace

extern "C" int64_t vtx_shared_prefix_workspace_len(int32_t batch_size, int32_t num_kv_heads, int32_t group_size,
                                                   int32_t head_dim) {
  const int cus = vtx::device_cu_count();
  if (batch_size < 0 || num_kv_heads < 1 || cus <= 0 || !vtx_paged_decode_attention_supported(head_dim, group_size))
    return 0;
  if ((int64_t)batch_size * num_kv_heads > kMaxSegments) return 0;
  return layout_of(batch_size, num_kv_heads, group_size, head_dim, cus).most_rows * num_kv_heads * (head_dim + 2);
}

extern "C" int vtx_shared_prefix_decode_attention(const uint16_t* q, uint16_t* o, const uint16_t* k_cache,
                                                  const uint16_t* v_cache, int64_t cache_rows,
                                                  const int32_t* kv_indptr, const int32_t* kv_indices,
                                                  int64_t kv_indices_len, const int32_t* kv_last_page_len,
                                                  const int32_t* plan, int64_t plan_len, int32_t batch_size,
                                                  int32_t num_kv_heads, int32_t group_size, int32_t head_dim,
                                                  int32_t page_size, float sm_scale, float* workspace,
                                                  int64_t workspace_len, void* stream) {
  vtx::clear_error();
  const char* what = "shared_prefix_decode_attention";
  if (batch_size < 0 || num_kv_heads < 1 || page_size < 1 || cache_rows < 0 || kv_indices_len < 0)
    return vtx::fail(VTX_E_INVALID, "%s: bad sizes", what);
  if (!vtx_paged_decode_attention_supported(head_dim, group_size))
    return vtx::fail(VTX_E_INVALID, "%s: head_dim %d with %d query heads per kv head not supported", what, head_dim,
                     group_size);
  const int64_t S = (int64_t)batch_size * num_kv_heads;
  if (S > kMaxSegments) return vtx::fail(VTX_E_INVALID, "%s: too many segments", what);
  if (S == 0) return VTX_OK;
  if (cache_rows > 0x7fffffffLL || cache_rows * page_size > 0xffffffffLL)
    return vtx::fail(VTX_E_INVALID, "%s: pools of more than 2^32 tokens x heads", what);
  if (!q || !o || !k_cache || !v_cache || !kv_indptr || !kv_last_page_len || !plan || !workspace ||
      (kv_indices_len > 0 && !kv_indices))
    return vtx::fail(VTX_E_INVALID, "%s: null pointer", what);
  if (!vtx::aligned16(q) || !vtx::aligned16(o) || !vtx::aligned16(k_cache) || !vtx::aligned16(v_cache))
    return vtx::fail(VTX_E_INVALID, "%s: q, o, k_cache and v_cache must be 16-byte aligned", what);
  const int cus = vtx::device_cu_count();
  if (cus <= 0) return vtx::fail(VTX_E_DEVICE, "%s: device query failed", what);
  const Layout at = layout_of(batch_size, num_kv_heads, group_size, head_dim, cus);
  if (plan_len < at.size || reinterpret_cast<uintptr_t>(plan) % 32)
    return vtx::fail(VTX_E_INVALID, "%s: plan of %lld int32 (32-byte aligned) needed, got %lld", what,
                     (long long)at.size, (long long)plan_len);
  const int64_t rows = at.most_rows * num_kv_heads;
  if (workspace_len < rows * (head_dim + 2) || !vtx::aligned16(workspace))
    return vtx::fail(VTX_E_INVALID, "%s: workspace of %lld floats (16-byte aligned) needed, got %lld", what,
                     (long long)(rows * (head_dim + 2)), (long long)workspace_len);
  SharedArgs a;
  a.q = q;
  a.o = o;
  a.k = k_cache;
  a.v = v_cache;
  a.rows = cache_rows;
  const int64_t bytes = cache_rows * page_size * head_dim * 2;
  a.pool_bytes = bytes <= 0xffffffffLL ? (uint32_t)bytes : 0u;
  a.indices = kv_indices;
  a.indices_len = kv_indices_len;
  a.last_len = kv_last_page_len;
  a.counts = plan + at.counts;
  a.items = reinterpret_cast<const Item*>(plan + at.items);
  a.combine = plan + at.combine;
  a.most_items = (int32_t)at.most_items;
  a.B = batch_size;
  a.H = num_kv_heads;
  a.G = group_size;
  a.P = page_size;
  a.p_shift = vtx::log2_exact(page_size);
  const float log2e = 1.44269504088896340736f;
  a.c = sm_scale == 0.f ? 1.f : (sm_scale < 0.f ? -sm_scale : sm_scale) * log2e;
  a.q_sign = sm_scale < 0.f ? 0x80008000u : 0u;
  a.q_keep = sm_scale == 0.f ? 0u : ~0u;
  a.acc = workspace;
  a.ml = reinterpret_cast<float2*>(workspace + rows * head_dim);
  a.max_rows = rows;
  // A row's partial results, by what the host knows: one run's chunks, a slot each,
  // or the segments' mean length, were the table's buffer full, in chunks of
  // kMinChunk tokens.  A guess: a row of an uneven table can have more, one of a table
  // with room behind it fewer (16 of 4 behind 4k, D 64, in a buffer for 128k tokens
  // each 14.4 us a layer, 12.7 in one that fits).  Either join is right for any count;
  // the order of its sums, and so a result's last bits, follow the buffer's length.
  const int64_t tiles = ((int64_t)batch_size * group_size + tile_rows(head_dim) - 1) / tile_rows(head_dim);
  const int64_t parts = at.slots / tiles, longest = kv_indices_len * page_size / (S * kMinChunk) + 1;
  a.join_four = (parts < longest ? parts : longest) * head_dim > kJoinFour;
  hipStream_t s = vtx::as_stream(stream);
  switch (head_dim) {
    case 64: return launch<64>(a, s);
    case 128: return launch<128>(a, s);
    default: return launch<256>(a, s);
  }
}
