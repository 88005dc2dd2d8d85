// Linear attention with a decay for each head, forward and backward, on MFMA.
//
//   S_t = l S_{t-1} + k_t v_t^T,   o_t = scale q_t S_t,   l = exp(log_decay[h]).
//
// Rows go in chunks of 64.  With S the state before a chunk of n rows,
//   O  = scale ((Q K^T . M) V + diag(l^{i+1}) Q S),   M_ij = l^{i-j} (j <= i),
//   S' = l^n S + sum_j l^{n-1-j} k_j v_j^T:
// four matrix products a chunk instead of one rank-one update a row.
//
// The backward is the same operator three times:
//   dq: (q, k, v) -> (dO, v, k), state transposed, time forward;
//   dv: (k, q, dO) and dk: (v, dO, q), time reversed, where the carried state
//   has its decay taken already (a row sees l^i of it instead of l^{i+1}, and
//   the update's weights are l^{n-j}); its last value of the dv pass is the
//   gradient of the initial state.  dk's state is dv's transposed: a segment of dk
//   starts from dv's.
// One kernel runs all of them ("passes"), in one launch.
//
// Work split: a workgroup holds one (sequence, head, segment)'s state in
// registers and walks its chunks; each wave owns 16 of the state's columns (D / 16
// waves).  On a CU: three workgroups at head_dim 64 (registers, 41 KB of LDS), one at
// 128 (two to three LDS buffers, 150 KB) and one at 256 (16 waves of 128 registers).  Where
// sequences x heads are too few for the GPU, sequences are cut into segments: one
// launch forms every segment's own state, and the main launch starts each segment
// from the states of those before it, which it adds up itself (few segments) or finds
// joined by linear_scan_kernel.
//
// What bounds it: the chunks of a workgroup follow each other, and a chunk's phases
// (operand reads, products, the split, barriers) hardly overlap.  At head_dim 128 a
// chunk takes 4.0 us with 256 workgroups (16 chunks, 68 us, 4.1 TB/s); of its 8420
// cycles LDS is busy 49%, the matrix cores 29%, and the waves wait 43%.
// [4, 2048, 16, 128] bf16: forward 43 us after 23 us for the segments' states,
// the three gradients 128 us.
//
// Registers and LDS: the state's accumulators (row d in the registers, column e
// in the lane) are, rounded, the A operand of O^T = S^T Q^T as they stand: S never
// leaves its registers.  The chunk's Q, K and V rows go through LDS; V^T and K^T
// operands come from transposing LDS reads.
//
// Rounding: P = Q K^T . M and the copy of S that meets Q are rounded to the inputs'
// type, once each, as the attention kernels round P.  The state itself is fp32,
// and its update is kept exact to it: l^{n-1-j} v_j is split into NT terms of the
// input type whose products with k are exact (three of bf16's 8 bits or two of
// fp16's 11 make up fp32's 24; two of bf16's, where no state is returned, would save
// 8% at head_dim 128 (115 -> 105 us in one segment), and outputs would then differ with
// what is asked for).  fp16's terms would leave its range below 2^-14: there a wave
// holds its columns of S times a power of two that keeps the largest weighted value
// near 2^13, and takes it out at every use.
#include "fa_common.h"
#include "fa_fwd_d128.h"
#include "fa_internal.h"

namespace fa {

namespace {

constexpr int kChunk = 64;

// One of q, k, v in a pass; head h of the pass reads head h / div.
struct LinTensor {
  const uint16_t* p;
  int64_t s[3];  // batch, seq, head
  int32_t div;
};

struct LinPass {
  LinTensor q, k, v;
  void* out;
  int64_t os[3];
  const float* init;  // [d][e] at d * ird + e * icd, nullptr: zero
  float* fin;         // [d][e] contiguous, nullptr: not kept
  int64_t is[2], fs[2];
  int32_t ird, icd;
  int32_t reverse, out_f32;
  float p_scale, inter_scale, upd_scale;
};

struct LinParams {
  LinPass pass[3];
  const float* log_decay;
  const int32_t* starts;  // packed form
  const int32_t* prefix;
  const int32_t* slots;
  float* ws;  // [pass][slot][head][D][D]: the segments' states (of two passes at most)
  int32_t batch, seqlen, heads, npass;
  int32_t nseg;    // dense: segments of a sequence; packed: slots in all
  int32_t seglen;  // rows of a segment, a multiple of kChunk
  int32_t nstates;
  int32_t join;
};

// How a segment comes by the state before it: there is one segment; from the
// initial state and the states of those before it, which the main kernel adds up; or
// linear_scan_kernel has put it into its slot.  (The main launch writes final states
// where a pool's initial ones stand: with several segments it reads the copies that the
// states' launch left in the last segments' slots.)
enum { kWhole = 0, kAdded = 1, kScanned = 2 };
// Passes: the forward alone, or dq, dv and dk, whose states are dv's transposed.
constexpr int kTwin = 2;
// Segments up to which they are added up (none at head_dim 256, whose kernel has no
// registers for it).  One sequence: [2, 8192, 8, 64] in 16 takes 38 us added and 41
// joined, [1, 16384, 4, 128] in 32 takes 68 and 63.  Packed sequences share the count,
// which bounds each one's: eight of 600 to 4096 rows, 16 heads, head_dim 128, in 18
// take 167 and 175 us; one of 17000 among single tokens, in 34, 194 and 196.
constexpr int max_added(int D, bool shared) { return D == 256 ? 1 : (shared ? 32 : 16); }

struct Segment {
  int b, seg, nseg;  // sequence, segment, segments of the sequence; b < 0: none
  int start, len;    // the sequence's first row and rows
};

// The packed sequence b, kept inside the rows there are whatever the offsets say.
__device__ __forceinline__ void packed_rows(const LinParams& p, int b, int& start, int& len) {
  const int s0 = min(max(p.starts[b], 0), p.seqlen);
  const int s1 = min(max(p.starts[b + 1], s0), p.seqlen);
  start = s0;
  len = s1 - s0;
}

// Slot -> segment: dense slots are (sequence, segment); packed ones are handed
// out in order, ceil(len / seglen) to a sequence, found by a wave scan.
__device__ __forceinline__ Segment find_segment(const LinParams& p, int slot) {
  Segment r;
  if (!p.starts) {
    r.b = slot / p.nseg;
    r.seg = slot - r.b * p.nseg;
    r.nseg = p.nseg;
    r.start = 0;
    r.len = p.seqlen;
    if (r.seg * p.seglen >= r.len) r.b = -1;
    return r;
  }
  r.b = -1;
  const int lane = threadIdx.x & 63;
  int base = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 64) {
    const int b = b0 + lane;
    int start = 0, len = 0;
    if (b < p.batch) packed_rows(p, b, start, len);
    const int n = (len + p.seglen - 1) / p.seglen;
    const int end = base + wave_scan(n);
    const uint64_t hit = __ballot(slot >= end - n && slot < end);
    if (hit) {
      const int src = __ffsll((unsigned long long)hit) - 1;
      r.b = b0 + src;
      r.nseg = __shfl(n, src);
      r.seg = slot - (__shfl(end, src) - r.nseg);
      r.start = __shfl(start, src);
      r.len = __shfl(len, src);
      break;
    }
    base = __shfl(end, 63);
  }
  r.b = __builtin_amdgcn_readfirstlane(r.b);
  r.nseg = __builtin_amdgcn_readfirstlane(r.nseg);
  r.seg = __builtin_amdgcn_readfirstlane(r.seg);
  r.start = __builtin_amdgcn_readfirstlane(r.start);
  r.len = __builtin_amdgcn_readfirstlane(r.len);
  return r;
}

// The state slot of sequence b, or -1: it starts from zero and keeps nothing.
__device__ __forceinline__ int state_slot(const LinParams& p, int b) {
  const int s = p.slots ? p.slots[b] : b;
  return s >= 0 && s < p.nstates ? s : -1;
}
__device__ __forceinline__ const float* init_of(const LinParams& p, const LinPass& a, int b, int h) {
  const int s = state_slot(p, b);
  if (!a.init || s < 0 || (p.prefix && p.prefix[b] <= 0)) return nullptr;
  return a.init + s * a.is[0] + h * a.is[1];
}
__device__ __forceinline__ float* fin_of(const LinParams& p, const LinPass& a, int b, int h) {
  const int s = state_slot(p, b);
  return a.fin && s >= 0 ? a.fin + s * a.fs[0] + h * a.fs[1] : nullptr;
}

// log_decay[h], with -inf as a number whose product with 0 is 0.
__device__ __forceinline__ float decay_of(const LinParams& p, int h) {
  const float g = p.log_decay[h];
  return g < -1e30f ? -1e30f : g;
}

// LDS rows of `W` 16-bit elements, 32 bytes (8 banks) further apart than they are
// long: the operand reads (16 bytes of 16 rows) and the transposing reads (32 bytes
// of 16 rows) then have no bank conflicts (3.9 and 2.6 cycles a wave; 6.4 and 3.8 at
// 16 or 64 bytes), and every address is one lane register plus an immediate (an XOR
// swizzle took some 40 address registers).
template <int W>
struct Rows16 {
  static constexpr int kStride = 2 * W + 32;
  static constexpr int kBytes = kChunk * kStride;
  __device__ static __forceinline__ int at(int r) { return r * kStride; }
};

template <int D>
struct LinShape {
  static constexpr int NW = D / 16;        // waves
  static constexpr int THREADS = 64 * NW;
  static constexpr int CPR = D / 8;        // 16-byte chunks of a row
  static constexpr int RPT = THREADS / CPR;  // rows the workgroup moves at a time: 32
  static constexpr int DT = D / 16;        // 16-row tiles of the state
  using Tile = Rows16<D>;
  using Scores = Rows16<kChunk>;
};

// Q's rows and P's are kept with their 4-element groups of each 32 in the order 0,
// 4, 1, 5, 2, 6, 3, 7.  A lane quarter l then finds in one 16-byte read the 8
// components (keys) that it has in the other operand: 4 l + 0..3 and 16 + 4 l + 0..3,
// from two of the state's 16-row tiles or two transposing reads of V.  Byte offset
// of group g of a row:
__device__ __forceinline__ int group_at(int g) {
  return 64 * (g >> 3) + 16 * (g & 3) + 8 * ((g >> 2) & 1);
}

// A chunk's rows of one tensor on the way to LDS, 16 bytes x 2 a thread: row
// 32 u + tid / CPR.  Rows at or behind n are zeros.
struct Staged {
  u32x4 x[2];
};
// Byte offset of row r of a chunk of n rows from its lowest address: rows go up
// from it (step 1) or down to it (step -1); out of any range behind n.
__device__ __forceinline__ uint32_t row_offset(int r, int n, int step, uint32_t row, uint32_t at) {
  return r < n ? (uint32_t)(step > 0 ? r : n - 1 - r) * row + at : 0xffffffffu;
}
template <int D>
__device__ __forceinline__ void load_rows(Staged& s, const uint16_t* lowest, int64_t stride,
                                          int step, int n, int tid) {
  using L = LinShape<D>;
  const rsrc_t rs = make_rsrc(lowest, (uint32_t)((n - 1) * stride + D) * 2u);
#pragma unroll
  for (int u = 0; u < 2; ++u)
    s.x[u] = __builtin_amdgcn_raw_buffer_load_b128(
        rs,
        row_offset(L::RPT * u + tid / L::CPR, n, step, 2 * (uint32_t)stride, 16 * (tid % L::CPR)),
        0, 0);
}
// Where a thread's 16 bytes of row tid / CPR stand in LDS.
template <int D>
__device__ __forceinline__ int place_of(int tid) {
  using L = LinShape<D>;
  return L::Tile::at(tid / L::CPR) + 16 * (tid % L::CPR);
}
template <int D>
__device__ __forceinline__ void store_grouped(const Staged& s, char* lds, int tid) {
  using L = LinShape<D>;
  char* p = lds + L::Tile::at(tid / L::CPR) + group_at(2 * (tid % L::CPR));
#pragma unroll
  for (int u = 0; u < 2; ++u, p += L::Tile::at(L::RPT)) {
    st8(p, u32x2{s.x[u][0], s.x[u][1]});
    st8(p + 16, u32x2{s.x[u][2], s.x[u][3]});
  }
}
template <int D>
__device__ __forceinline__ void store_rows(const Staged& s, char* lds, int tid) {
  using L = LinShape<D>;
#pragma unroll
  for (int u = 0; u < 2; ++u) st16(lds + place_of<D>(tid) + u * L::Tile::at(L::RPT), s.x[u]);
}

// Operand with row or column lane % 16 and k = 32 s + 4 (lane / 16) + 0..3 and the
// same + 16, from 16 columns of a row-major [k][column] tile in LDS; p: the tile,
// transposed_at of the lane, and the 16 columns' place.
template <class Tile>
__device__ __forceinline__ u32x4 read_transposed(const char* p, int s) {
  const u32x2 lo = lds_read_tr(p + s * Tile::at(32));
  const u32x2 hi = lds_read_tr(p + s * Tile::at(32) + Tile::at(16));
  return u32x4{lo[0], lo[1], hi[0], hi[1]};
}
template <class Tile>
__device__ __forceinline__ int transposed_at() {
  const int lane = threadIdx.x & 63;
  return Tile::at(4 * (lane >> 4) + ((lane & 15) >> 2)) + 8 * (lane & 3);
}

// x as the sum of NT terms of the input type, each the rounding of what is left.
template <class T, int NT>
__device__ __forceinline__ void split_terms(float (&x)[8], u32x4 (&term)[NT]) {
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // One rounding for the term and for what is left of it: the compiler may
      // otherwise round the product that x is to the term in one step, and x in
      // two for the difference, which then differ by a whole step of the type.
      asm("" : "+v"(x[2 * i]), "+v"(x[2 * i + 1]));
      uint32_t w = T::pack(x[2 * i], x[2 * i + 1]);
      asm("" : "+v"(w));
      term[n][i] = w;
      if (n + 1 < NT) {
        x[2 * i] -= T::lo(w);
        x[2 * i + 1] -= T::hi(w);
      }
    }
}

template <class T>
constexpr int kTerms = T::kId == 0 ? 2 : 3;

__device__ __forceinline__ float pow2(int e) {
  return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23);
}
__device__ __forceinline__ int exponent(float x) {
  return (int)((__builtin_bit_cast(uint32_t, x) >> 23) & 255) - 127;
}

// Exponent of the wave's largest |value| in fp16 words, or kNone where all are zero.
constexpr int kNone = -1000;
template <int N>
__device__ __forceinline__ int max_exponent(const u32x4 (&w)[N]) {
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  u16x2 m = {0, 0};
#pragma unroll
  for (int s = 0; s < N; ++s)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w[s][i] & 0x7fff7fffu));
  const int top = wave_max_nonneg(max((int)m[0], (int)m[1]));
  return top ? exponent(Half::lo((uint32_t)top)) : kNone;
}

// Where a wave keeps its part of a segment's state in the workspace: the
// accumulators as they are, 16 bytes a lane.
template <int D>
__device__ __forceinline__ int state_image(int wave, int dt, int lane) {
  return ((wave * (D / 16) + dt) * 64 + lane) * 4;
}

// A wave's part of a segment's state; transposed: u is the state of the pass whose
// states are this one's transposed.
template <int D>
__device__ __forceinline__ void load_state(f32x4 (&x)[D / 16], const float* u, int wave, int lane,
                                           bool transposed) {
  if (transposed) {
    // Row 16 dt + 4 lq + i and column 16 wave + lc here are that column and row there.
    const int quad = 16 * ((lane & 15) >> 2) + 4 * (lane >> 4);
    const float* t = u + state_image<D>(0, wave, quad) + (lane & 3);
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i) x[dt][i] = t[state_image<D>(dt, 0, i)];
  } else {
    const float* t = u + state_image<D>(wave, 0, lane);
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt)
      x[dt] = *reinterpret_cast<const f32x4*>(t + state_image<D>(0, dt, 0));
  }
}

// One segment of one head.  STATE_ONLY: forms the segment's own state (from
// zero) into the workspace and no output.
template <class T, int D, bool STATE_ONLY>
__global__ __launch_bounds__(LinShape<D>::THREADS, D == 256 ? 4 : 2) void linear_kernel(LinParams p) {
  using L = LinShape<D>;
  using Tile = typename L::Tile;
  using Scores = typename L::Scores;
  constexpr int NT = kTerms<T>;
  // Whether registers hold what a chunk does not change (head_dim 256 has 128 of them
  // for a wave, and spills 20 to 36 as it is).
  constexpr bool kKeep = D < 256;
  // Buffers of a chunk's rows: with two, the next chunk's rows go to LDS while this
  // one is worked on, and one barrier of three goes: [2, 8192, 16, 128] forward 119 ->
  // 108 us.  head_dim 256 has no LDS for it; at 64 a third workgroup on the CU is
  // worth more ([4, 2048, 16, 64] backward 54 us, 62 us with two buffers).
  constexpr int NB = D == 128 ? 2 : 1;
  __shared__ __align__(16) char lds_q[STATE_ONLY ? 16 : NB * Tile::kBytes];
  __shared__ __align__(16) char lds_k[NB * Tile::kBytes];
  // With two, a chunk's P meets V while the next chunk is worked on, which leaves one
  // barrier a chunk: P has two buffers, and V, whose places take O's rows, three.  [32,
  // 2048, 16, 128] backward 865 -> 844 us.  (Half of the waves with the state's products
  // first and the rows and P after them: 872 us, 252 registers.)
  constexpr bool kLate = NB == 2 && !STATE_ONLY;
  constexpr int VB = kLate ? 3 : NB;
  __shared__ __align__(16) char lds_v[VB * Tile::kBytes];
  __shared__ __align__(16) char lds_p[STATE_ONLY ? 16 : NB * Scores::kBytes];
  __shared__ __align__(16) float weight[NB * kChunk];  // of row j in the state's update
  __shared__ float powers[STATE_ONLY ? 1 : kChunk + 17];

  const int h = blockIdx.x % p.heads, slot = blockIdx.x / p.heads;
  const LinPass& a = p.pass[blockIdx.y];
  const Segment sg = find_segment(p, slot);
  if (sg.b < 0) return;
  // (No segment starts from the last one's state.)
  if (STATE_ONLY && sg.seg == sg.nseg - 1 && (p.join != kAdded || sg.nseg == 1)) return;
  const int row0 = sg.seg * p.seglen;
  const int nrows = min(p.seglen, sg.len - row0);

  const int lane = threadIdx.x & 63, wave = wave_id();
  const int lc = lane & 15, lq = lane >> 4;
  const float g = decay_of(p, h), g2 = g * kLog2e;
  const int sh = a.reverse ? 1 : 0;

  const int batch = p.starts ? 0 : sg.b;
  const int step = a.reverse ? -1 : 1;
  // The token with the lowest address among rows c .. c + n - 1 of the segment.
  auto lowest = [&](int c, int n) {
    return (int64_t)(sg.start + (a.reverse ? sg.len - row0 - c - n : row0 + c));
  };
  auto base_of = [&](const LinTensor& t) {
    return t.p + batch * t.s[0] + (h / t.div) * t.s[2];
  };
  const uint16_t* qp = base_of(a.q);
  const uint16_t* kp = base_of(a.k);
  const uint16_t* vp = base_of(a.v);
  Staged sq, sk, sv;
  auto load_chunk = [&](int c, int tid) {
    const int n = min(kChunk, nrows - c);
    const int64_t t = lowest(c, n);
    if (!STATE_ONLY) load_rows<D>(sq, qp + t * a.q.s[1], a.q.s[1], step, n, tid);
    load_rows<D>(sk, kp + t * a.k.s[1], a.k.s[1], step, n, tid);
    load_rows<D>(sv, vp + t * a.v.s[1], a.v.s[1], step, n, tid);
  };
  // State column 16 wave + lc, rows 16 dt + 4 lq + (0..3).
  f32x4 S[L::DT];
  const bool twin = blockIdx.y == kTwin;
  const int64_t slots = (int64_t)p.nseg * (p.starts ? 1 : p.batch);
  float* seg_state =
      p.ws + ((min((int)blockIdx.y, kTwin - 1) * slots + slot) * p.heads + h) * D * D;
  const int col = 16 * wave + lc;
  const float* init = init_of(p, a, sg.b, h);
  auto load_init = [&]() {
#pragma unroll
    for (int dt = 0; dt < L::DT; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        S[dt][i] = init[(16 * dt + 4 * lq + i) * a.ird + col * a.icd];
  };
  if (STATE_ONLY && sg.seg == sg.nseg - 1) {
    if (!init) return;
    load_init();
#pragma unroll
    for (int dt = 0; dt < L::DT; ++dt)
      *reinterpret_cast<f32x4*>(seg_state + state_image<D>(wave, dt, lane)) = S[dt];
    return;
  }
  load_chunk(0, threadIdx.x);

#pragma unroll
  for (int dt = 0; dt < L::DT; ++dt) S[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (!STATE_ONLY) {
    const int64_t next = (int64_t)p.heads * D * D;
    if (p.join == kScanned) {
      load_state<D>(S, seg_state, wave, lane, twin);
    } else if (!kKeep || sg.nseg == 1) {
      if (init) load_init();
    } else {
      // The initial state and those of the segments before, in order.  (Offsets that
      // overlap would give more segments than there are slots.)
      const int last = min(slot + sg.nseg - 1 - sg.seg, (int)slots - 1);
      if (init) load_state<D>(S, seg_state + (last - slot) * next, wave, lane, twin);
      const float decay = expm1f(g * (float)p.seglen);
      for (int s = sg.seg; s > 0; --s) {
        f32x4 x[L::DT];
        load_state<D>(x, seg_state - s * next, wave, lane, twin);
#pragma unroll
        for (int dt = 0; dt < L::DT; ++dt)
#pragma unroll
          for (int i = 0; i < 4; ++i) S[dt][i] = fmaf(S[dt][i], decay, S[dt][i]) + x[dt][i];
      }
    }
  }

  // P^T tiles (16 keys j x 16 rows i) on and below the diagonal, dealt to the waves
  // in the order (row tile, key tile) = (0, 0), (1, 0), (1, 1), (2, 0), ...
  constexpr int NP = (10 + L::NW - 1) / L::NW;
  static_assert(L::THREADS >= kChunk + 17, "a thread for each power");
  // l^e for e = 0..64, and 0 for e = -16..-1 (keys behind their row).  At head_dim
  // 256 the factors of P and of O's rows are read from it where they are used: a
  // wave's 128 registers have no room for them.
  const float* power = powers + 16;
  if (!STATE_ONLY && threadIdx.x < kChunk + 17) {
    const int e = (int)threadIdx.x - 16;
    powers[threadIdx.x] = e < 0 ? 0.f : fast_exp2(g2 * (float)e);
  }

  const int op_at = Tile::at(lc) + 16 * lq;  // operand reads of Q and K rows
  const int tr_at = transposed_at<Tile>();   // transposing reads of K and V rows
  const int p_at = Scores::at(lc);

  // The two tiles above the diagonal that O's 32-key steps take in.
  if (!STATE_ONLY && threadIdx.x < 64) {
    const int t = threadIdx.x >> 5, r = (threadIdx.x & 31) >> 1;
    for (int g = 0; g < 2 * NB; ++g)
      st8(lds_p + (g >> 1) * Scores::kBytes + Scores::at(32 * t + r) + group_at(4 * (2 * t + 1) + 2 * (threadIdx.x & 1) + (g & 1)),
          u32x2{0, 0});
  }

  float dm1 = 0.f;  // l^n - 1 for the chunk's n rows
  int held = 0;       // S is held times 2^held (fp16)
  const float p_scale = a.p_scale, inter_scale = a.inter_scale;
  auto p_factor = [&](int tile, int i) {
    const int it = (tile >= 1) + (tile >= 3) + (tile >= 6), jt = tile - it * (it + 1) / 2;
    return p_scale * power[16 * (it - jt) + lc - 4 * lq - i];  // row - key of acc[i]
  };
  auto row_factor = [&](int it) { return power[16 * it + lc + 1 - sh]; };
  float pf[NP][4], rowf[4];
  if constexpr (!STATE_ONLY && kKeep) {
    __syncthreads();
#pragma unroll
    for (int np = 0; np < NP; ++np)
#pragma unroll
      for (int i = 0; i < 4; ++i) pf[np][i] = p_factor(min(wave + L::NW * np, 9), i);
#pragma unroll
    for (int it = 0; it < 4; ++it) rowf[it] = row_factor(it);
  }
  // |weight| < 2^weight_top (upd_scale 0 or not finite: no scaling to speak of)
  const int weight_top = min(max(exponent(a.upd_scale), -60), 60) + 1;

  // The rows of O that chunk c left in V's place, 16 bytes x 2 a thread (at the
  // places where the thread puts its part of a later V).
  auto write_rows = [&](int c, int vbuf, int tid) {
    const int n = min(kChunk, nrows - c);
    const rsrc_t rs = make_rsrc(static_cast<uint16_t*>(a.out) + batch * a.os[0] +
                                    lowest(c, n) * a.os[1] + h * a.os[2],
                                (uint32_t)((n - 1) * a.os[1] + D) * 2u);
#pragma unroll
    for (int u = 0; u < 2; ++u)
      __builtin_amdgcn_raw_buffer_store_b128(
          ld16(lds_v + vbuf * Tile::kBytes + place_of<D>(tid) + u * Tile::at(L::RPT)), rs,
          row_offset(L::RPT * u + tid / L::CPR, n, step, 2 * (uint32_t)a.os[1],
                     16 * (tid % L::CPR)),
          0, 0);
  };
  // Chunk c's rows, which have been loaded, and its weights into their buffers.
  auto stage = [&](int c, int buf, int vbuf, int tid) {
    if (!STATE_ONLY) store_grouped<D>(sq, lds_q + buf * Tile::kBytes, tid);
    store_rows<D>(sk, lds_k + buf * Tile::kBytes, tid);
    store_rows<D>(sv, lds_v + vbuf * Tile::kBytes, tid);
    // Rows at or behind n are zeros: their weight only has to be finite.
    const int n = min(kChunk, nrows - c);
    if (tid < kChunk)
      weight[buf * kChunk + tid] = a.upd_scale * fast_exp2(g2 * (float)max(n - 1 - tid + sh, 0));
  };
  const bool out16 = !STATE_ONLY && !a.out_f32;
  u32x4 vt[kChunk / 32];  // the wave's columns of V, for O and for the update
  f32x4 o[4];
  auto read_values = [&](const char* v_rows) {
#pragma unroll
    for (int s = 0; s < kChunk / 32; ++s)
      vt[s] = read_transposed<Tile>(v_rows + tr_at + 32 * wave, s);
  };
  auto scores = [&](const char* q_rows, const char* k_rows, char* p_rows) {
    // P^T = K Q^T with the decay, rounded, as P's rows in LDS.
#pragma unroll
    for (int np = 0; np < NP; ++np) {
      const int tile = wave + L::NW * np;
      if (tile < 10) {
        const int it = (tile >= 1) + (tile >= 3) + (tile >= 6), jt = tile - it * (it + 1) / 2;
        const char* kq = k_rows + Tile::at(16 * jt + lc) + 8 * lq;
        const char* qq = q_rows + op_at + it * Tile::at(16);
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < D / 32; ++kk) {
          const u32x2 x = ld8(kq + 64 * kk), y = ld8(kq + 64 * kk + 32);
          acc = T::mma16(u32x4{x[0], x[1], y[0], y[1]}, ld16(qq + 64 * kk), acc);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] *= kKeep ? pf[np][i] : p_factor(tile, i);
        st8(p_rows + p_at + it * Scores::at(16) + group_at(4 * jt + lq),
            u32x2{T::pack(acc[0], acc[1]), T::pack(acc[2], acc[3])});
      }
    }
  };
  auto from_state = [&](const char* q_rows) {
    // O^T = S^T Q^T, then the rows' decay.  fp16: S meets Q scaled by a power of
    // two (its largest value to 2^14), so that neither a long memory's sums nor
    // small ones leave the type's range.
    float up = inter_scale, down = 1.f;
    if constexpr (T::kId == 0) {
      float m = 0.f;
#pragma unroll
      for (int dt = 0; dt < L::DT; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) m = fmaxf(m, fabsf(S[dt][i]));
      m = __builtin_bit_cast(float, wave_max_nonneg(__builtin_bit_cast(int, m)));
      const int e = m > 0.f && m < __builtin_inff() ? min(max(exponent(m), -100), 100) : 14;
      down = pow2(14 - e);
      up *= pow2(e - 14) * pow2(-held);
    }
#pragma unroll
    for (int it = 0; it < 4; ++it) o[it] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int dt = 0; dt < L::DT; dt += 2) {
      u32x4 sf;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        sf[i] = T::pack(S[dt + i / 2][2 * (i & 1)] * down, S[dt + i / 2][2 * (i & 1) + 1] * down);
#pragma unroll
      for (int it = 0; it < 4; ++it)
        o[it] = T::mma16(sf, ld16(q_rows + op_at + it * Tile::at(16) + 32 * dt), o[it]);
    }
#pragma unroll
    for (int it = 0; it < 4; ++it) o[it] *= up * (kKeep ? rowf[it] : row_factor(it));
  };
  // The rest of chunk c's O, and O on its way out.
  auto finish = [&](int c, const char* p_rows, char* v_rows) {
    const int n = min(kChunk, nrows - c);
    // O^T += V^T P^T
#pragma unroll
    for (int s = 0; s < kChunk / 32; ++s)
#pragma unroll
      for (int it = 2 * s; it < 4; ++it)
        o[it] = T::mma16(vt[s], ld16(p_rows + p_at + it * Scores::at(16) + 64 * s + 16 * lq), o[it]);
    if (a.out_f32) {
      const rsrc_t rs = make_rsrc(static_cast<float*>(a.out) + batch * a.os[0] +
                                      lowest(c, n) * a.os[1] + h * a.os[2],
                                  (uint32_t)((n - 1) * a.os[1] + D) * 4u);
#pragma unroll
      for (int it = 0; it < 4; ++it)
        __builtin_amdgcn_raw_buffer_store_b128(
            __builtin_bit_cast(u32x4, o[it]), rs,
            row_offset(16 * it + lc, n, step, 4 * (uint32_t)a.os[1], 4 * (16 * wave + 4 * lq)), 0,
            0);
    } else {
      // Into V's columns of this wave, which no other wave reads.
#pragma unroll
      for (int it = 0; it < 4; ++it)
        st8(v_rows + Tile::at(16 * it + lc) + 32 * wave + 8 * lq,
            u32x2{T::pack(o[it][0], o[it][1]), T::pack(o[it][2], o[it][3])});
    }
  };
  auto update = [&](const char* k_rows, int buf) {
    // S = l^n S + K^T (weight V).  The decay as S + S (l^n - 1): the factor's own
    // rounding, which a slow decay would compound over hundreds of chunks, is then
    // relative to the small difference.
#pragma unroll
    for (int dt = 0; dt < L::DT; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i) S[dt][i] = fmaf(S[dt][i], dm1, S[dt][i]);
    if constexpr (T::kId == 0) {
      const int e = max_exponent(vt);
      const int want = 13 - e - weight_top;
      // Down where a term would overflow, up where eight bits would be lost.
      if (e != kNone && (want < held || want > held + 8)) {
        const float f = pow2(want - held);
#pragma unroll
        for (int dt = 0; dt < L::DT; ++dt) S[dt] *= f;
        held = want;
      }
    }
    const float hold = T::kId == 0 ? pow2(held) : 1.f;
#pragma unroll
    for (int s = 0; s < kChunk / 32; ++s) {
      float x[8];
      const float* w = weight + buf * kChunk + 32 * s + 4 * lq;
      const f32x4 w0 = *reinterpret_cast<const f32x4*>(w) * hold;
      const f32x4 w1 = *reinterpret_cast<const f32x4*>(w + 16) * hold;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[2 * i] = T::lo(vt[s][i]) * (i < 2 ? w0[2 * i] : w1[2 * i - 4]);
        x[2 * i + 1] = T::hi(vt[s][i]) * (i < 2 ? w0[2 * i + 1] : w1[2 * i - 3]);
      }
      u32x4 term[NT];
      split_terms<T, NT>(x, term);
#pragma unroll
      for (int dt = 0; dt < L::DT; ++dt) {
        const u32x4 kt = read_transposed<Tile>(k_rows + tr_at + 32 * dt, s);
#pragma unroll
        for (int t = 0; t < NT; ++t) S[dt] = T::mma16(kt, term[t], S[dt]);
      }
    }
  };

  if constexpr (NB == 2) {
    stage(0, 0, 0, threadIdx.x);
    if (kChunk < nrows) load_chunk(kChunk, threadIdx.x);
    __syncthreads();
  }
  int vbuf = 0;  // V's buffer of the chunk
  for (int c = 0; c < nrows; c += kChunk) {
    const int n = min(kChunk, nrows - c);
    const int buf = NB == 2 ? c / kChunk & 1 : 0;
    // At head_dim 256 addresses are formed anew in every chunk: kept, they are the
    // registers that no longer fit, and a reload from scratch waits for the rows on
    // their way.
    int tid = threadIdx.x;
    if constexpr (!kKeep) asm volatile("" : "+v"(tid));
    if (c == 0 || n < kChunk) dm1 = expm1f(g * (float)n);
    const char* q_rows = lds_q + buf * Tile::kBytes;
    const char* k_rows = lds_k + buf * Tile::kBytes;
    char* p_rows = lds_p + (STATE_ONLY ? 0 : buf * Scores::kBytes);
    if constexpr (kLate) {
      const int next = vbuf == 2 ? 0 : vbuf + 1, before = vbuf == 0 ? 2 : vbuf - 1;
      if (c > 0)
        finish(c - kChunk, lds_p + (buf ^ 1) * Scores::kBytes, lds_v + before * Tile::kBytes);
      // The next chunk's rows, into buffers whose readers were done before the last
      // barrier; in V's stands the O of two chunks ago.
      if (out16 && c > kChunk) write_rows(c - 2 * kChunk, next, tid);
      if (c + kChunk < nrows) stage(c + kChunk, buf ^ 1, next, tid);
      if (c + 2 * kChunk < nrows) load_chunk(c + 2 * kChunk, tid);
      read_values(lds_v + vbuf * Tile::kBytes);
      scores(q_rows, k_rows, p_rows);
      from_state(q_rows);
      update(k_rows, buf);
      vbuf = next;
      __syncthreads();  // P and the next chunk are there, and O of the chunk before
    } else if constexpr (STATE_ONLY) {
      if constexpr (NB == 2) {
        if (c + kChunk < nrows) stage(c + kChunk, buf ^ 1, buf ^ 1, tid);
        if (c + 2 * kChunk < nrows) load_chunk(c + 2 * kChunk, tid);
      } else {
        __syncthreads();  // the last chunk's LDS reads are done
        stage(c, 0, 0, tid);
        __syncthreads();
        if (c + kChunk < nrows) load_chunk(c + kChunk, tid);
      }
      read_values(lds_v + buf * Tile::kBytes);
      update(k_rows, buf);
      if constexpr (NB == 2) __syncthreads();  // the next chunk is there
    } else {
      __syncthreads();  // the last chunk's LDS reads are done, and its O is there
      if (out16 && c > 0) write_rows(c - kChunk, 0, tid);
      stage(c, 0, 0, tid);
      __syncthreads();
      if (c + kChunk < nrows) load_chunk(c + kChunk, tid);
      read_values(lds_v);
      scores(q_rows, k_rows, p_rows);
      from_state(q_rows);
      // The update stands before the barrier that P's readers need, where the waves
      // that formed P's tiles are behind the others; at head_dim 256 there are no
      // registers to keep O through it.
      if constexpr (kKeep) update(k_rows, 0);
      __syncthreads();  // P is there
      finish(c, p_rows, lds_v);
      if constexpr (!kKeep) update(k_rows, 0);
    }
  }

  const float out = pow2(-held);
  if (STATE_ONLY) {
#pragma unroll
    for (int dt = 0; dt < L::DT; ++dt)
      *reinterpret_cast<f32x4*>(seg_state + state_image<D>(wave, dt, lane)) = S[dt] * out;
    return;
  }
  const int c = (nrows - 1) / kChunk * kChunk;
  if constexpr (kLate) {
    vbuf = vbuf == 0 ? 2 : vbuf - 1;
    finish(c, lds_p + (c / kChunk & 1) * Scores::kBytes, lds_v + vbuf * Tile::kBytes);
    if (out16 && c > 0) write_rows(c - kChunk, vbuf == 0 ? 2 : vbuf - 1, threadIdx.x);
  }
  if (out16) {
    __syncthreads();
    write_rows(c, vbuf, threadIdx.x);
  }
  float* fin = sg.seg == sg.nseg - 1 ? fin_of(p, a, sg.b, h) : nullptr;
  if (fin) {
#pragma unroll
    for (int dt = 0; dt < L::DT; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i) fin[(16 * dt + 4 * lq + i) * D + col] = S[dt][i] * out;
  }
}

// Joins the segments' states in order: each slot's own state becomes the state
// before it.  A thread holds four components, in the workspace's layout
// (state_image): rows d .. d + 3 of column e.  Bound by the states' memory: 9 us for
// eight packed prompts of 16 heads at head_dim 128 (before those were added up).
template <int D>
__global__ __launch_bounds__(256) void linear_scan_kernel(LinParams p) {
  constexpr int PARTS = D * D / 1024;
  const int unit = blockIdx.x / PARTS, h = unit % p.heads, b = unit / p.heads;
  const LinPass& a = p.pass[blockIdx.y];
  const int at = 4 * ((int)(blockIdx.x % PARTS) * 256 + (int)threadIdx.x);
  int first = b * p.nseg, len = p.seqlen;
  if (p.starts) {
    int start, n = 0;
    for (int i = threadIdx.x & 63; i < b; i += 64) {
      packed_rows(p, i, start, len);
      n += (len + p.seglen - 1) / p.seglen;
    }
    first = wave_total(n);
    packed_rows(p, b, start, len);
  }
  const int64_t total = (int64_t)p.nseg * (p.starts ? 1 : p.batch);
  // (Offsets that overlap would give more segments than there are slots.)
  const int nseg = min((len + p.seglen - 1) / p.seglen, (int)max(total - first, (int64_t)0));
  if (nseg == 0) return;
  float* state = p.ws + ((blockIdx.y * total + first) * p.heads + h) * D * D + at;
  const int64_t next = (int64_t)p.heads * D * D;
  const float* init = init_of(p, a, b, h);
  const float decay = expm1f(decay_of(p, h) * (float)p.seglen);
  f32x4 S = {0.f, 0.f, 0.f, 0.f};
  const int lane = at / 4 % 64, dt = at / 256 % (D / 16);
  const int d = 16 * dt + 4 * (lane >> 4), e = 16 * (at / (16 * D)) + (lane & 15);
  if (init) {
#pragma unroll
    for (int i = 0; i < 4; ++i) S[i] = init[(d + i) * a.ird + e * a.icd];
  }
  for (int s = 0; s < nseg; ++s, state += next) {
    f32x4 u = {0.f, 0.f, 0.f, 0.f};
    if (s < nseg - 1) u = *reinterpret_cast<const f32x4*>(state);
    *reinterpret_cast<f32x4*>(state) = S;
#pragma unroll
    for (int i = 0; i < 4; ++i) S[i] = fmaf(S[i], decay, S[i]) + u[i];
  }
}

// Gradients of shared heads: the fp32 parts of a KV head's query heads, in order.
template <class T>
__global__ __launch_bounds__(256) void linear_group_sum_kernel(const float* part, uint16_t* out,
                                                               int64_t s0, int64_t s1, int64_t s2,
                                                               int64_t total, int seqlen, int heads_k,
                                                               int group, int D) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= total) return;
  const int cpr = D / 8;
  const int c = (int)(i % cpr);
  const int64_t row = i / cpr;  // (b, s, kv head)
  const int hk = (int)(row % heads_k);
  const int64_t t = row / heads_k;
  const float* src = part + (row * group) * D + 8 * c;
  f32x4 x = {0.f, 0.f, 0.f, 0.f}, y = x;
  for (int n = 0; n < group; ++n, src += D) {
    x += *reinterpret_cast<const f32x4*>(src);
    y += *reinterpret_cast<const f32x4*>(src + 4);
  }
  uint16_t* dst = out + (t / seqlen) * s0 + (t % seqlen) * s1 + hk * s2 + 8 * c;
  st16(dst, u32x4{T::pack(x[0], x[1]), T::pack(x[2], x[3]), T::pack(y[0], y[1]),
                  T::pack(y[2], y[3])});
}

// ------------------------------------------------------------------ decode

// One token for each sequence: the state is read, updated and written once.
// Bound by that memory (8 D^2 bytes a sequence and head; D^2 * 5 flops).  A
// workgroup takes COLS columns of one head's state: every load is issued before
// the first use, and a column's sum over d stays inside the workgroup.  64 x 32 states
// at head_dim 128: 56 us, 4.8 TB/s (a large copy: 5.2); 4 x 16: 4.6 us.
template <class T, int D, int COLS>
__global__ __launch_bounds__(256) void linear_decode_kernel(fa_linear_decode_args a) {
  constexpr int LANES = COLS / 4, ROWS = 256 / LANES, N = D / ROWS, SLICES = D / COLS;
  __shared__ float qs[D], ks[D];
  __shared__ __align__(16) float part[ROWS][COLS];
  const int slice = blockIdx.x % SLICES;
  const int h = (blockIdx.x / SLICES) % a.num_heads, b = blockIdx.x / SLICES / a.num_heads;
  const int hk = h / (a.num_heads / a.num_heads_k);
  const int slot = a.state_indices ? a.state_indices[b] : b;
  const bool kept = slot >= 0 && slot < a.num_states;
  const int e = slice * COLS + 4 * (threadIdx.x % LANES), r0 = threadIdx.x / LANES;
  float* st = a.state + (kept ? slot * a.s_stride[0] + h * a.s_stride[1] : 0) + e;
  f32x4 S[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    S[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (kept) S[i] = *reinterpret_cast<const f32x4*>(st + (r0 + i * ROWS) * D);
  }
  const uint16_t* q = static_cast<const uint16_t*>(a.q) + b * a.q_stride[0] + h * a.q_stride[1];
  const uint16_t* k = static_cast<const uint16_t*>(a.k) + b * a.k_stride[0] + hk * a.k_stride[1];
  const uint16_t* v = static_cast<const uint16_t*>(a.v) + b * a.v_stride[0] + hk * a.v_stride[1];
  if (threadIdx.x < D) {
    qs[threadIdx.x] = T::lo(q[threadIdx.x]);
    ks[threadIdx.x] = T::lo(k[threadIdx.x]);
  }
  const u32x2 vw = ld8(v + e);
  const f32x4 vv = {T::lo(vw[0]), T::hi(vw[0]), T::lo(vw[1]), T::hi(vw[1])};
  const float decay = expf(a.log_decay[h]);
  __syncthreads();
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int d = r0 + i * ROWS;
    const float kd = ks[d], qd = qs[d];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      S[i][j] = fmaf(kd, vv[j], S[i][j] * decay);
      o[j] = fmaf(qd, S[i][j], o[j]);
    }
    if (kept) *reinterpret_cast<f32x4*>(st + d * D) = S[i];
  }
  *reinterpret_cast<f32x4*>(&part[r0][4 * (threadIdx.x % LANES)]) = o;
  __syncthreads();
  if (threadIdx.x < COLS / 2) {
    float x = 0.f, y = 0.f;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      x += part[r][2 * threadIdx.x];
      y += part[r][2 * threadIdx.x + 1];
    }
    uint16_t* out = static_cast<uint16_t*>(a.out) + b * a.o_stride[0] + h * a.o_stride[1];
    *reinterpret_cast<uint32_t*>(out + slice * COLS + 2 * threadIdx.x) =
        T::pack(x * a.scale, y * a.scale);
  }
}

// ------------------------------------------------------------------ host

// Microseconds of a launch whose `groups` workgroups walk `chunks` chunks each,
// `per_cu` of them on a CU at a time: a chunk takes `lat` for one workgroup alone
// and `mem` for each of those on a CU.
double launch_us(int64_t groups, int64_t chunks, int per_cu, double lat, double mem) {
  const int64_t cus = device_cu_count(), full = groups / (cus * per_cu);
  const int64_t rest = groups - full * cus * per_cu;
  const double start = 4.5;
  double t = full * (start + chunks * std::max(lat, per_cu * mem));
  if (rest > 0) t += start + chunks * std::max(lat, (double)((rest + cus - 1) / cus) * mem);
  return t;
}

// Rows of a segment.  More segments fill the GPU, and each costs a state formed
// twice and carried through memory: the count with the least time by the model
// above.  Its constants (us a chunk, TB/s) are fitted to MI355X times of the forward
// and the backward of 21 shapes, one to forty heads and 1024 to 32768 rows, at 1 to 64
// segments: what it picks is within 4% of the fastest of them, 0.3% on average.
// units: sequences x heads x passes; state_units: of those, the ones whose segments'
// states are formed.  tokens: of one sequence, or of all `seqs` packed ones, which end
// in a part of a segment each.
int segment_rows(int64_t tokens, int64_t units, int64_t state_units, int64_t seqs, int D) {
  const int per_cu = D == 64 ? 3 : 1, state_per_cu = D == 64 ? 6 : (D == 128 ? 2 : 1);
  const double chunk = D == 64 ? 1.8 : (D == 128 ? 3.8 : 10.5);
  const double state_lat = D == 64 ? 0.75 : (D == 128 ? 1.5 : 4.5);
  const double state_mem = D == 64 ? 0.33 : state_lat;
  // A state once through memory; smaller ones stay in the last cache.
  const double bytes_us = 4.0 * D * D / (D < 256 ? 10e6 : 5e6);
  const int added = max_added(D, seqs > 1);
  const int64_t chunks = (tokens + kChunk - 1) / kChunk;
  double best = 0;
  int64_t rows = chunks;
  for (int64_t n = 1; n <= std::min<int64_t>(chunks, 64); ++n) {
    const int64_t c = (chunks + n - 1) / n;
    if (n > 1 && (chunks + c - 1) / c < n) continue;  // the same as fewer
    const int64_t segments = std::max(n + (seqs - 1) / 2, seqs);
    double t = launch_us(units * segments, c, per_cu, chunk, chunk);
    if (n > 1)
      t += launch_us(state_units * (segments - seqs), c, state_per_cu, state_lat, state_mem) +
           units * n * (n <= added ? 1 + n / seqs / 2 : 4) * bytes_us + (n <= added ? 0 : 5);
    if (n == 1 || t < best) {
      best = t;
      rows = c;
    }
  }
  return (int)(rows * kChunk);
}

// Passes whose segments' states are formed.
int state_passes(const LinParams& p) { return std::min<int>(p.npass, kTwin); }

// Cuts p's sequences; returns the slots in all.
int64_t set_segments(LinParams& p, int D) {
  // (Packed: the sequences' lengths are on the device.)
  const int64_t units = (int64_t)p.heads * p.npass * (p.starts ? 1 : p.batch);
  const int64_t seqs = p.starts ? p.batch : 1;
  p.seglen = segment_rows(p.seqlen, units, units / p.npass * state_passes(p), seqs, D);
  const int64_t most = ((int64_t)p.seqlen + p.seglen - 1) / p.seglen;
  p.join = most == 1 ? kWhole : (most <= max_added(D, seqs > 1) ? kAdded : kScanned);
  if (p.starts) {
    p.nseg = p.seqlen / p.seglen + p.batch;
    return p.nseg;
  }
  p.nseg = (int)most;
  return (int64_t)p.nseg * p.batch;
}

size_t state_bytes(const LinParams& p, int64_t slots, int D) {
  return p.join != kWhole ? (size_t)slots * state_passes(p) * p.heads * D * D * sizeof(float) : 0;
}

template <class T, int D>
hipError_t launch_passes(LinParams& p, int64_t slots, hipStream_t st) {
  const dim3 grid((unsigned)(slots * p.heads), p.npass), block(LinShape<D>::THREADS);
  if (p.join != kWhole)
    hipLaunchKernelGGL((linear_kernel<T, D, true>), dim3(grid.x, state_passes(p)), block, 0, st, p);
  if (p.join == kScanned)
    hipLaunchKernelGGL((linear_scan_kernel<D>),
                       dim3((unsigned)(D * D / 1024 * p.batch * p.heads), state_passes(p)),
                       dim3(256), 0, st, p);
  hipLaunchKernelGGL((linear_kernel<T, D, false>), grid, block, 0, st, p);
  return hipGetLastError();
}

template <class T>
hipError_t launch_dim(LinParams& p, int64_t slots, int D, hipStream_t st) {
  if (D == 64) return launch_passes<T, 64>(p, slots, st);
  if (D == 128) return launch_passes<T, 128>(p, slots, st);
  return launch_passes<T, 256>(p, slots, st);
}

LinTensor tensor(const void* x, const int64_t* s, int div) {
  return {static_cast<const uint16_t*>(x), {s[0], s[1], s[2]}, div};
}

LinParams fwd_params(const fa_linear_args& a) {
  LinParams p = {};
  const int group = a.num_heads / a.num_heads_k, D = a.head_dim;
  LinPass& f = p.pass[0];
  f.q = tensor(a.q, a.q_stride, 1);
  f.k = tensor(a.k, a.k_stride, group);
  f.v = tensor(a.v, a.v_stride, group);
  f.out = a.out;
  for (int i = 0; i < 3; ++i) f.os[i] = a.o_stride[i];
  f.init = a.initial_state;
  f.fin = a.final_state;
  for (int i = 0; i < 2; ++i) {
    f.is[i] = a.is_stride[i];
    f.fs[i] = a.fs_stride[i];
  }
  f.ird = D;
  f.icd = 1;
  f.p_scale = f.inter_scale = a.scale;
  f.upd_scale = 1.f;
  p.log_decay = a.log_decay;
  p.starts = a.query_start_loc;
  p.prefix = a.prefix_kv_lens;
  p.slots = a.state_indices;
  p.batch = a.batch;
  p.seqlen = a.seqlen;
  p.heads = a.num_heads;
  p.npass = 1;
  p.nstates = a.num_states;
  return p;
}

LinParams bwd_params(const fa_linear_bwd_args& a) {
  LinParams p = {};
  const int group = a.num_heads / a.num_heads_k, D = a.head_dim;
  const LinTensor q = tensor(a.q, a.q_stride, 1), k = tensor(a.k, a.k_stride, group);
  const LinTensor v = tensor(a.v, a.v_stride, group), o = tensor(a.dout, a.do_stride, 1);
  auto pass = [&](LinPass& f, const LinTensor& x, const LinTensor& y, const LinTensor& z, void* out,
                  const int64_t* os, const float* init, const int64_t* is, bool transposed) {
    f.q = x;
    f.k = y;
    f.v = z;
    f.out = out;
    for (int i = 0; i < 3; ++i) f.os[i] = os[i];
    f.init = init;
    for (int i = 0; i < 2; ++i) f.is[i] = is[i];
    f.ird = transposed ? 1 : D;
    f.icd = transposed ? D : 1;
  };
  pass(p.pass[0], o, v, k, a.dq, a.dq_stride, a.initial_state, a.is_stride, true);
  p.pass[0].p_scale = p.pass[0].inter_scale = a.scale;
  p.pass[0].upd_scale = 1.f;
  pass(p.pass[1], k, q, o, a.dv, a.dv_stride, a.d_final_state, a.fs_stride, false);
  pass(p.pass[kTwin], v, o, q, a.dk, a.dk_stride, a.d_final_state, a.fs_stride, true);
  for (int i = 1; i < 3; ++i) {
    // The carried state holds the scale (the final state's gradient has none).
    p.pass[i].reverse = 1;
    p.pass[i].p_scale = p.pass[i].upd_scale = a.scale;
    p.pass[i].inter_scale = 1.f;
  }
  p.pass[1].fin = a.d_initial_state;
  for (int i = 0; i < 2; ++i) p.pass[1].fs[i] = a.dis_stride[i];
  p.log_decay = a.log_decay;
  p.batch = p.nstates = a.batch;
  p.seqlen = a.seqlen;
  p.heads = a.num_heads;
  p.npass = 3;
  return p;
}

// fp32 parts of dk and dv for each query head, where heads share k and v.
size_t part_bytes(const fa_linear_bwd_args& a) {
  return a.num_heads == a.num_heads_k
             ? 0
             : (size_t)a.batch * a.seqlen * a.num_heads * a.head_dim * sizeof(float);
}

template <class T, int D>
hipError_t launch_decode_cols(const fa_linear_decode_args& a, hipStream_t st) {
  // Wide slices (512-byte rows) where they give every CU a workgroup, before that 32
  // columns: 4 x 32 states at head_dim 128 take 4.6 us in 32 columns and 5.3 wide, 8 x 32
  // take 8.1 and 7.0.  At head_dim 64 a whole state (4 x 16: 3.3 and 3.2 us, 64 x 32: 13.9
  // and 11.8).
  constexpr int WIDE = D < 128 ? D : 128;
  const int64_t heads = (int64_t)a.batch * a.num_heads;
  auto run = [&](auto kernel, int cols) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)(heads * (D / cols))), dim3(256), 0, st, a);
  };
  if constexpr (D > 64) {
    if (heads * (D / WIDE) < device_cu_count()) {
      run(linear_decode_kernel<T, D, 32>, 32);
      return hipGetLastError();
    }
  }
  run(linear_decode_kernel<T, D, WIDE>, WIDE);
  return hipGetLastError();
}

template <class T>
hipError_t launch_decode_dim(const fa_linear_decode_args& a, hipStream_t st) {
  if (a.head_dim == 64) return launch_decode_cols<T, 64>(a, st);
  if (a.head_dim == 128) return launch_decode_cols<T, 128>(a, st);
  return launch_decode_cols<T, 256>(a, st);
}

}  // namespace

int64_t linear_fwd_workgroups(const fa_linear_args& a) {
  LinParams p = fwd_params(a);
  return set_segments(p, a.head_dim) * p.heads;
}

size_t linear_fwd_workspace_bytes(const fa_linear_args& a) {
  LinParams p = fwd_params(a);
  const int64_t slots = set_segments(p, a.head_dim);
  return state_bytes(p, slots, a.head_dim);
}

hipError_t launch_linear_fwd(const fa_linear_args& a, void* ws, hipStream_t st) {
  LinParams p = fwd_params(a);
  const int64_t slots = set_segments(p, a.head_dim);
  p.ws = static_cast<float*>(ws);
  return a.dtype == FA_DTYPE_F16 ? launch_dim<Half>(p, slots, a.head_dim, st)
                                 : launch_dim<BFloat16>(p, slots, a.head_dim, st);
}

int64_t linear_bwd_workgroups(const fa_linear_bwd_args& a) {
  LinParams p = bwd_params(a);
  return set_segments(p, a.head_dim) * p.heads;
}

size_t linear_bwd_workspace_bytes(const fa_linear_bwd_args& a) {
  LinParams p = bwd_params(a);
  const int64_t slots = set_segments(p, a.head_dim);
  return state_bytes(p, slots, a.head_dim) + 2 * part_bytes(a);
}

hipError_t launch_linear_bwd(const fa_linear_bwd_args& a, void* ws, hipStream_t st) {
  LinParams p = bwd_params(a);
  const int64_t slots = set_segments(p, a.head_dim);
  p.ws = static_cast<float*>(ws);
  const size_t part = part_bytes(a);
  float* dk = reinterpret_cast<float*>(static_cast<char*>(ws) + state_bytes(p, slots, a.head_dim));
  float* dv = dk + part / sizeof(float);
  if (part) {
    for (int i = 1; i < 3; ++i) {
      p.pass[i].out = i == kTwin ? dk : dv;
      p.pass[i].out_f32 = 1;
      p.pass[i].os[2] = a.head_dim;
      p.pass[i].os[1] = (int64_t)a.num_heads * a.head_dim;
      p.pass[i].os[0] = p.pass[i].os[1] * a.seqlen;
    }
  }
  const bool f16 = a.dtype == FA_DTYPE_F16;
  hipError_t e = f16 ? launch_dim<Half>(p, slots, a.head_dim, st)
                     : launch_dim<BFloat16>(p, slots, a.head_dim, st);
  if (e != hipSuccess || !part) return e;
  const int64_t total = (int64_t)a.batch * a.seqlen * a.num_heads_k * (a.head_dim / 8);
  const dim3 grid((unsigned)((total + 255) / 256));
  for (int i = 0; i < 2; ++i) {
    const float* src = i ? dv : dk;
    uint16_t* dst = static_cast<uint16_t*>(i ? a.dv : a.dk);
    const int64_t* s = i ? a.dv_stride : a.dk_stride;
    auto run = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, src, dst, s[0], s[1], s[2], total,
                         a.seqlen, a.num_heads_k, a.num_heads / a.num_heads_k, a.head_dim);
    };
    if (f16)
      run(linear_group_sum_kernel<Half>);
    else
      run(linear_group_sum_kernel<BFloat16>);
  }
  return hipGetLastError();
}

hipError_t launch_linear_decode(const fa_linear_decode_args& a, hipStream_t st) {
  return a.dtype == FA_DTYPE_F16 ? launch_decode_dim<Half>(a, st)
                                 : launch_decode_dim<BFloat16>(a, st);
}

}  // namespace fa
