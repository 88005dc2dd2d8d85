// Per-head RMS norm and position rotation of queries and keys: dense with its
// backward, and the serving form that writes the keys and values of new tokens
// into the paged cache on the way.
//
// One head row x of D components: n = x r w, r = 1 / sqrt(mean(x^2) + eps), then
// components paired by the rotation turn by the token's table row:
// (a c - b s, a s + b c).  Its transpose with g = R^T dy, h = g w:
//   dx = r (h - x r mean(h x r)),   dw = sum over rows of g x r.
// Everything is fp32 from the loaded 16-bit values to the one rounding at the store.
//
// Bound by memory: 4 bytes an element forward, 6 backward (r is formed again from
// x, which dx needs anyway, so nothing is saved but the inputs).
//
// Layout: a group of LPR lanes holds one row; each lane holds two 16-byte chunks,
// the two that the rotation pairs (chunks c and c + rotary / 16, or 2c and 2c + 1
// interleaved), so rotating needs no exchange between lanes and every load and
// store is 16 bytes.  Rows of q, of k and of v are separate ranges of workgroups:
// what differs between them (pointers, weight) is then wave-uniform.
#include "fa_common.h"
#include "fa_internal.h"

namespace fa {

namespace {

constexpr int kThreads = 256;

// n / d for n < 2^31 by a multiplication.
struct FastDiv {
  uint32_t mul, shift, d;
  FastDiv() = default;
  explicit FastDiv(uint32_t div) : d(div) {
    shift = 0;
    while ((uint64_t(1) << shift) < div) ++shift;
    mul = (uint32_t)(((uint64_t(1) << 32) * ((uint64_t(1) << shift) - div)) / div + 1);
  }
  __device__ __forceinline__ uint32_t quot(uint32_t n) const {
    return (__umulhi(n, mul) + n) >> shift;
  }
};

// The rows of one tensor: row r is head r % heads of token r / heads.
struct Rows {
  const uint16_t* x;
  uint16_t* y;
  const void* w;  // nullptr: no norm
  int64_t xs[3];  // batch, seq, head
  int64_t ys[3];  // dense: as xs; cache: page, slot, head
  int64_t gs[3];  // backward: strides of dy
  const uint16_t* dy;
  uint32_t count;   // rows
  uint32_t blocks;  // workgroups
  FastDiv heads;
};

struct Params {
  Rows q, k, v;
  const float* cos;
  const float* sin;
  const int64_t* pos;
  const int64_t* slots;  // cache form: k and v rows go to their token's slot
  int64_t ts[2], ps[2];
  int64_t npos, max_slot;
  FastDiv seqlen, page;
  int32_t page_size;
  int32_t chunks, nrot;  // 16-byte chunks of a row, lanes that rotate
  int32_t interleaved, weight_f32;
  float eps, inv_d;
  float* partial;  // backward: [blocks][D] of q, then of k
};

template <int CTRL>
__device__ __forceinline__ float dpp_add(float x) {
  return x + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(
                                           0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
// Sum over the LPR lanes of a row (every lane gets it).
template <int LPR>
__device__ __forceinline__ float row_sum(float x) {
  x = dpp_add<0xB1>(x);                         // quad_perm [1, 0, 3, 2]
  x = dpp_add<0x4E>(x);                         // quad_perm [2, 3, 0, 1]
  if constexpr (LPR >= 8) x = dpp_add<0x141>(x);   // row_half_mirror
  if constexpr (LPR >= 16) x = dpp_add<0x140>(x);  // row_mirror
  if constexpr (LPR >= 32) x += __shfl_xor(x, 16);
  return x;
}

template <class T>
__device__ __forceinline__ void unpack(u32x4 v, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = T::lo(v[i]);
    f[2 * i + 1] = T::hi(v[i]);
  }
}
template <class T>
__device__ __forceinline__ u32x4 pack8(const float (&f)[8]) {
  u32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = T::pack(f[2 * i], f[2 * i + 1]);
  return v;
}

// The lane's two chunks of every row.
struct Lane {
  int ca, cb;
  bool has_a, has_b, turns;
};
__device__ __forceinline__ Lane lane_chunks(const Params& p, int c) {
  Lane l;
  l.turns = c < p.nrot;
  if (p.interleaved || !l.turns) {  // neighbours; behind the rotated part they start at 2 nrot
    l.ca = 2 * c;
    l.cb = 2 * c + 1;
  } else {
    l.ca = c;
    l.cb = c + p.nrot;
  }
  l.has_a = l.ca < p.chunks;
  l.has_b = l.cb < p.chunks;
  return l;
}

__device__ __forceinline__ void load8(const void* w, int f32, int chunk, bool there, int bf16,
                                      float (&out)[8]) {
  if (!there) {
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = 0.f;
    return;
  }
  if (f32) {
    const float* p = static_cast<const float*>(w) + 8 * chunk;
    const f32x4 x = *reinterpret_cast<const f32x4*>(p), y = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      out[i] = x[i];
      out[4 + i] = y[i];
    }
    return;
  }
  const u32x4 v = ld16(static_cast<const uint16_t*>(w) + 8 * chunk);
  if (bf16)
    unpack<BFloat16>(v, out);
  else
    unpack<Half>(v, out);
}

// Table columns 8c .. 8c + 7 of position `pos`: NaN at or beyond the table's end.
__device__ __forceinline__ void load_turn(const Params& p, int64_t pos, int c, float (&cs)[8],
                                          float (&sn)[8]) {
  if (pos < p.npos) {
    const float* cp = p.cos + pos * p.ts[0] + 8 * c;
    const float* sp = p.sin + pos * p.ts[1] + 8 * c;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(cp + 4 * h);
      const f32x4 y = *reinterpret_cast<const f32x4*>(sp + 4 * h);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        cs[4 * h + i] = x[i];
        sn[4 * h + i] = y[i];
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) cs[i] = sn[i] = __builtin_nanf("");
  }
}

// (a, b) turned in place; BACK: by the transpose.
template <bool BACK>
__device__ __forceinline__ void turn(bool interleaved, const float (&cs)[8], const float (&sn)[8],
                                     float (&a)[8], float (&b)[8]) {
  auto one = [](float c, float s, float& x, float& y) {
    if constexpr (BACK) s = -s;
    const float u = x * c - y * s, v = x * s + y * c;
    x = u;
    y = v;
  };
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      one(cs[i], sn[i], a[2 * i], a[2 * i + 1]);
      one(cs[4 + i], sn[4 + i], b[2 * i], b[2 * i + 1]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) one(cs[i], sn[i], a[i], b[i]);
  }
}

__device__ __forceinline__ float dot8(const float (&x)[8], const float (&y)[8], float acc) {
#pragma unroll
  for (int i = 0; i < 8; ++i) acc = fmaf(x[i], y[i], acc);
  return acc;
}

struct Token {
  uint32_t t, b, s, h;
};
__device__ __forceinline__ Token token_of(const Params& p, const Rows& r, uint32_t row) {
  Token k;
  k.t = r.heads.quot(row);
  k.h = row - k.t * r.heads.d;
  k.b = p.seqlen.quot(k.t);
  k.s = k.t - k.b * p.seqlen.d;
  return k;
}
__device__ __forceinline__ int64_t position_of(const Params& p, const Token& k) {
  return p.pos ? p.pos[k.b * p.ps[0] + k.s * p.ps[1]] : (int64_t)k.s;
}
__device__ __forceinline__ int64_t offset_of(const int64_t (&s)[3], const Token& k) {
  return k.b * s[0] + k.s * s[1] + k.h * s[2];
}

// One row a group of lanes.  (Two to four rows a group, their loads issued together:
// [2, 8192, 32 + 8, 128] takes 68.3 us with one and 69.6, 70.8 and 72.1 with two to
// four; the waves of a CU overlap enough.  71 us among other work, 4.7 TB/s.)
template <class T, int LPR, bool CACHE>
__global__ __launch_bounds__(kThreads) void norm_rope_kernel(Params p) {
  constexpr int G = kThreads / LPR;  // rows of a workgroup
  uint32_t blk = blockIdx.x;
  const bool is_q = blk < p.q.blocks;
  const bool is_v = CACHE && blk >= p.q.blocks + p.k.blocks;
  const Rows& R = is_q ? p.q : (is_v ? p.v : p.k);
  blk -= is_q ? 0 : (is_v ? p.q.blocks + p.k.blocks : p.q.blocks);
  const uint32_t row = blk * G + threadIdx.x / LPR;
  if (row >= R.count) return;
  const int c = threadIdx.x % LPR;
  const Lane l = lane_chunks(p, c);
  const Token k = token_of(p, R, row);
  const uint16_t* xp = R.x + offset_of(R.xs, k);
  u32x4 xa = {0, 0, 0, 0}, xb = xa;
  if (l.has_a) xa = ld16(xp + 8 * l.ca);
  if (l.has_b) xb = ld16(xp + 8 * l.cb);
  uint16_t* out;
  if (CACHE && !is_q) {
    const int64_t slot = p.slots[k.t];
    if (slot < 0 || slot >= p.max_slot) return;
    const int64_t page = p.max_slot <= 0x7fffffff ? (int64_t)p.page.quot((uint32_t)slot)
                                                  : slot / p.page_size;
    out = R.y + page * R.ys[0] + (slot - page * p.page_size) * R.ys[1] + k.h * R.ys[2];
  } else {
    out = R.y + offset_of(R.ys, k);
  }
  if (!is_v) {
    const int64_t pos = position_of(p, k);
    float a[8], b[8], cs[8], sn[8];
    if (l.turns && pos >= 0) load_turn(p, pos, c, cs, sn);
    unpack<T>(xa, a);
    unpack<T>(xb, b);
    if (R.w) {
      float wa[8], wb[8];
      load8(R.w, p.weight_f32, l.ca, l.has_a, T::kId, wa);
      load8(R.w, p.weight_f32, l.cb, l.has_b, T::kId, wb);
      const float sum = row_sum<LPR>(dot8(b, b, dot8(a, a, 0.f)));
      const float r = rsqrtf(fmaf(sum, p.inv_d, p.eps));
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        a[i] *= r * wa[i];
        b[i] *= r * wb[i];
      }
    }
    if (pos < 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] = b[i] = 0.f;
    } else if (l.turns) {
      turn<false>(p.interleaved, cs, sn, a, b);
    }
    xa = pack8<T>(a);
    xb = pack8<T>(b);
  }
  if (l.has_a) st16(out + 8 * l.ca, xa);
  if (l.has_b) st16(out + 8 * l.cb, xb);
}

// dx of every row; with a weight, the workgroup's sum of g x r over its rows goes
// to its own row of `partial` (a fixed order: the gradients repeat bit for bit).
template <class T, int LPR>
__global__ __launch_bounds__(kThreads) void norm_rope_bwd_kernel(Params p) {
  constexpr int G = kThreads / LPR;
  __shared__ float sums[G][LPR * 16];
  const bool is_q = blockIdx.x < p.q.blocks;
  const Rows& R = is_q ? p.q : p.k;
  const uint32_t blk = blockIdx.x - (is_q ? 0 : p.q.blocks);
  const int c = threadIdx.x % LPR, grp = threadIdx.x / LPR;
  const Lane l = lane_chunks(p, c);
  const bool norm = R.w != nullptr;
  float wa[8], wb[8], da[8], db[8];
  if (norm) {
    load8(R.w, p.weight_f32, l.ca, l.has_a, T::kId, wa);
    load8(R.w, p.weight_f32, l.cb, l.has_b, T::kId, wb);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) da[i] = db[i] = 0.f;
  for (uint32_t row = blk * G + grp; row < R.count; row += R.blocks * G) {
    const Token k = token_of(p, R, row);
    const uint16_t* gp = R.dy + offset_of(R.gs, k);
    const uint16_t* xp = R.x + offset_of(R.xs, k);
    const int64_t pos = position_of(p, k);
    u32x4 ga = {0, 0, 0, 0}, gb = ga, xa = ga, xb = ga;
    if (l.has_a) ga = ld16(gp + 8 * l.ca);
    if (l.has_b) gb = ld16(gp + 8 * l.cb);
    if (norm) {
      if (l.has_a) xa = ld16(xp + 8 * l.ca);
      if (l.has_b) xb = ld16(xp + 8 * l.cb);
    }
    float a[8], b[8], cs[8], sn[8];
    if (l.turns && pos >= 0) load_turn(p, pos, c, cs, sn);
    unpack<T>(ga, a);
    unpack<T>(gb, b);
    if (pos < 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] = b[i] = 0.f;
    } else if (l.turns) {
      turn<true>(p.interleaved, cs, sn, a, b);
    }
    if (norm) {
      float x[8], y[8];
      unpack<T>(xa, x);
      unpack<T>(xb, y);
      float hx = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        hx = fmaf(a[i] * wa[i], x[i], hx);
        hx = fmaf(b[i] * wb[i], y[i], hx);
      }
      hx = row_sum<LPR>(hx);
      const float r = rsqrtf(fmaf(row_sum<LPR>(dot8(y, y, dot8(x, x, 0.f))), p.inv_d, p.eps));
      // r (h - x r mean(h x r)) = r h - x (r^3 mean(h x))
      const float m = pos < 0 ? 0.f : r * r * r * (hx * p.inv_d);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (pos >= 0) {
          da[i] = fmaf(a[i], x[i] * r, da[i]);
          db[i] = fmaf(b[i], y[i] * r, db[i]);
        }
        a[i] = pos < 0 ? 0.f : r * wa[i] * a[i] - x[i] * m;
        b[i] = pos < 0 ? 0.f : r * wb[i] * b[i] - y[i] * m;
      }
    }
    uint16_t* out = R.y + offset_of(R.ys, k);
    if (l.has_a) st16(out + 8 * l.ca, pack8<T>(a));
    if (l.has_b) st16(out + 8 * l.cb, pack8<T>(b));
  }
  if (!norm) return;
  if (l.has_a)
    for (int i = 0; i < 8; ++i) sums[grp][8 * l.ca + i] = da[i];
  if (l.has_b)
    for (int i = 0; i < 8; ++i) sums[grp][8 * l.cb + i] = db[i];
  __syncthreads();
  const int D = 8 * p.chunks;
  for (int i = threadIdx.x; i < D; i += kThreads) {
    float s = 0.f;
#pragma unroll 8
    for (int g = 0; g < G; ++g) s += sums[g][i];
    p.partial[(int64_t)blockIdx.x * D + i] = s;
  }
}

// Sums the workgroups' rows of `partial`: 16 columns a workgroup, 64 strided
// parts of the rows side by side, then those in order.
__global__ __launch_bounds__(1024) void weight_grad_kernel(const float* partial, int D, int nq,
                                                           int nk, void* dqw, void* dkw, int f32,
                                                           int bf16) {
  __shared__ float sums[64][17];
  const bool is_q = blockIdx.y == 0;
  void* out = is_q ? dqw : dkw;
  if (!out) return;
  const float* src = partial + (is_q ? 0 : (int64_t)nq * D);
  const int n = is_q ? nq : nk;
  const int col = blockIdx.x * 16 + threadIdx.x % 16, part = threadIdx.x / 16;
  float s = 0.f;
  if (col < D) {
#pragma unroll 8
    for (int i = part; i < n; i += 64) s += src[(int64_t)i * D + col];
  }
  sums[part][threadIdx.x % 16] = s;
  __syncthreads();
  if (part != 0 || col >= D) return;
  s = 0.f;
#pragma unroll
  for (int i = 0; i < 64; ++i) s += sums[i][threadIdx.x];
  if (f32)
    static_cast<float*>(out)[col] = s;
  else
    static_cast<uint16_t*>(out)[col] =
        (uint16_t)(bf16 ? BFloat16::pack(s, 0.f) : Half::pack(s, 0.f));
}

int lanes_per_row(int D) {
  int n = 4;
  while (n * 16 < D) n *= 2;
  return n;
}

void set_rows(Rows& r, const void* x, const int64_t* xs, void* y, const int64_t* ys, const void* w,
              int64_t tokens, int heads, int nx, int ny) {
  r = {};
  r.x = static_cast<const uint16_t*>(x);
  r.y = static_cast<uint16_t*>(y);
  r.w = w;
  for (int i = 0; i < nx; ++i) r.xs[3 - nx + i] = xs[i];
  for (int i = 0; i < ny; ++i) r.ys[3 - ny + i] = ys[i];
  r.count = (uint32_t)(tokens * heads);
  r.heads = FastDiv((uint32_t)heads);
}

template <class Args>
void set_common(Params& p, const Args& a, int seqlen) {
  p.cos = a.cos;
  p.sin = a.sin;
  p.ts[0] = a.table_stride[0];
  p.ts[1] = a.table_stride[1];
  p.npos = a.num_positions;
  p.seqlen = FastDiv((uint32_t)std::max(seqlen, 1));
  p.page = FastDiv(1);
  p.chunks = a.head_dim / 8;
  p.nrot = a.rotary_dim / 16;
  p.interleaved = a.interleaved;
  p.weight_f32 = a.weight_f32;
  p.eps = a.eps;
  p.inv_d = 1.f / (float)a.head_dim;
}

template <class T, int LPR, bool CACHE>
hipError_t launch_rows(Params& p, hipStream_t st) {
  constexpr int G = kThreads / LPR;
  uint32_t n = 0;
  for (Rows* r : {&p.q, &p.k, &p.v}) {
    r->blocks = (uint32_t)(((uint64_t)r->count + G - 1) / G);
    n += r->blocks;
  }
  hipLaunchKernelGGL((norm_rope_kernel<T, LPR, CACHE>), dim3(n), dim3(kThreads), 0, st, p);
  return hipGetLastError();
}

template <class F>
hipError_t by_lanes(int D, F f) {
  switch (lanes_per_row(D)) {
    case 4: return f(IntC<4>{});
    case 8: return f(IntC<8>{});
    case 16: return f(IntC<16>{});
    default: return f(IntC<32>{});
  }
}

template <bool CACHE>
hipError_t launch_rope(Params& p, int D, int dtype, hipStream_t st) {
  return by_lanes(D, [&](auto lanes) {
    constexpr int LPR = decltype(lanes)::value;
    return dtype == FA_DTYPE_F16 ? launch_rows<Half, LPR, CACHE>(p, st)
                                 : launch_rows<BFloat16, LPR, CACHE>(p, st);
  });
}

// Workgroups of the backward for `rows` rows of a tensor: four a CU ([2, 8192, 32 + 8,
// 128] 104 us; one 147, two 109, eight 110, sixteen 121), fewer
// where the rows are.
uint32_t bwd_blocks(int64_t rows, int D) {
  const int64_t G = kThreads / lanes_per_row(D);
  return (uint32_t)std::min<int64_t>((rows + G - 1) / G, 4 * device_cu_count());
}

}  // namespace

hipError_t launch_norm_rope(const fa_norm_rope_args& a, hipStream_t st) {
  Params p = {};
  const int64_t tokens = (int64_t)a.batch * a.seqlen;
  set_rows(p.q, a.q, a.q_stride, a.q_out, a.qo_stride, a.q_weight, tokens, a.num_heads, 3, 3);
  set_rows(p.k, a.k, a.k_stride, a.k_out, a.ko_stride, a.k_weight, tokens, a.num_heads_k, 3, 3);
  set_common(p, a, a.seqlen);
  p.pos = a.positions;
  p.ps[0] = a.pos_stride[0];
  p.ps[1] = a.pos_stride[1];
  return launch_rope<false>(p, a.head_dim, a.dtype, st);
}

hipError_t launch_norm_rope_cache(const fa_norm_rope_cache_args& a, hipStream_t st) {
  Params p = {};
  set_rows(p.q, a.q, a.q_stride, a.q_out, a.qo_stride, a.q_weight, a.num_tokens, a.num_heads, 2, 2);
  set_rows(p.k, a.k, a.key_stride, a.k_cache, a.k_stride, a.k_weight, a.num_tokens,
           a.num_kv_heads, 2, 3);
  set_rows(p.v, a.v, a.value_stride, a.v_cache, a.v_stride, nullptr, a.num_tokens, a.num_kv_heads,
           2, 3);
  set_common(p, a, a.num_tokens);
  p.pos = a.positions;
  p.ps[1] = 1;
  p.slots = a.slot_mapping;
  p.page_size = a.page_size;
  p.max_slot = (int64_t)a.num_pages * a.page_size;
  p.page = FastDiv((uint32_t)a.page_size);
  return launch_rope<true>(p, a.head_dim, a.dtype, st);
}

size_t norm_rope_bwd_workspace_bytes(const fa_norm_rope_bwd_args& a) {
  if (!a.q_weight && !a.k_weight) return 0;
  const int64_t tokens = (int64_t)a.batch * a.seqlen;
  return ((size_t)bwd_blocks(tokens * a.num_heads, a.head_dim) +
          bwd_blocks(tokens * a.num_heads_k, a.head_dim)) * a.head_dim * sizeof(float);
}

hipError_t launch_norm_rope_bwd(const fa_norm_rope_bwd_args& a, void* ws, hipStream_t st) {
  Params p = {};
  const int64_t tokens = (int64_t)a.batch * a.seqlen;
  set_rows(p.q, a.q, a.q_stride, a.dq, a.dq_stride, a.q_weight, tokens, a.num_heads, 3, 3);
  set_rows(p.k, a.k, a.k_stride, a.dk, a.dk_stride, a.k_weight, tokens, a.num_heads_k, 3, 3);
  p.q.dy = static_cast<const uint16_t*>(a.dq_out);
  p.k.dy = static_cast<const uint16_t*>(a.dk_out);
  for (int i = 0; i < 3; ++i) {
    p.q.gs[i] = a.dqo_stride[i];
    p.k.gs[i] = a.dko_stride[i];
  }
  p.q.blocks = bwd_blocks(p.q.count, a.head_dim);
  p.k.blocks = bwd_blocks(p.k.count, a.head_dim);
  set_common(p, a, a.seqlen);
  p.pos = a.positions;
  p.ps[0] = a.pos_stride[0];
  p.ps[1] = a.pos_stride[1];
  p.partial = static_cast<float*>(ws);
  const uint32_t n = p.q.blocks + p.k.blocks;
  const hipError_t e = n == 0 ? hipSuccess : by_lanes(a.head_dim, [&](auto lanes) {
    constexpr int LPR = decltype(lanes)::value;
    if (a.dtype == FA_DTYPE_F16)
      hipLaunchKernelGGL((norm_rope_bwd_kernel<Half, LPR>), dim3(n), dim3(kThreads), 0, st, p);
    else
      hipLaunchKernelGGL((norm_rope_bwd_kernel<BFloat16, LPR>), dim3(n), dim3(kThreads), 0, st, p);
    return hipGetLastError();
  });
  if (e != hipSuccess || (!a.q_weight && !a.k_weight)) return e;
  hipLaunchKernelGGL(weight_grad_kernel, dim3((a.head_dim + 15) / 16, 2), dim3(1024), 0, st,
                     p.partial, a.head_dim, (int)p.q.blocks, (int)p.k.blocks, a.dq_weight,
                     a.dk_weight, a.weight_f32, a.dtype == FA_DTYPE_BF16);
  return hipGetLastError();
}

}  // namespace fa
