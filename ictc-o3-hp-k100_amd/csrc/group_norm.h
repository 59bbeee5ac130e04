// Group norm with an activation, channels last: x [samples, positions, channels], statistics over all positions and the
// channels of a group,
//   h = (x - mean) r,  r = 1 / sqrt(var + eps),  z = h w + b,  y = act(z)          (act: z, or z / (1 + exp(-z)))
// with ga = g act'(z), u = ga w and <.> the mean over a sample's group its gradients
//   dx = r (u - <u> - h <u h>),  dw = sum ga h,  db = sum ga                       (sums over samples and positions)
// and, for a loss that depends on dx itself, the gradients of <v, dx> + <vw, dw> + <vb, db>:
//   pv = r (v - <v> - h <v h>),  e = w pv + h vw + vb,  zz = e g act''(z)
//   dg' = e act'(z),  dw' = sum ga pv + zz h,  db' = sum zz
//   t  = ga vw + zz w - r (<v h> u + <u h> v),   q = <u v> - <u> <v> - <u h> <v h>
//   dx' = r (t - <t> - h <t h>) - r^2 q h
// <zz w> and <zz w h> hold <v> and <v h>, in which they are linear, so all of the means come of sums of one read.
// Where x is kept in 8 bits (codes.h) its values stand in h; mean and r are those of x itself.
//
// All of it is bound by memory.  Three forms, by the size of a sample's group:
//  * Rows: up to 256 chunks of it.  A team of up to 64 lanes holds it in registers: one read, no barrier.  A team keeps its
//    group, so the parameters stay in registers and their gradients are added per lane.
//  * Tiles: a block takes some whole groups of a sample and reads them twice, for the sums and for the result, the second
//    time from the caches; one launch.
//  * Parts: few large samples.  The sums by many blocks, a small kernel that adds their parts in order, and the result by
//    as many blocks again.
// A chunk is the largest power of two of a group's channels up to 16 bytes, so each lies in one group and in one block of
// codes.  Statistics of tiles and parts are sums of x and of its squares in FP64, which costs nothing beside memory,
// loses nothing to a mean far from zero and holds squares past FP32's range.  Every sum has a fixed order.
#pragma once
#include <algorithm>

#include "codes.h"

namespace ictc {

struct GroupNormCall {
  int64_t samples, positions;
  int channels, groups;
  const void *x, *g, *v, *w, *b, *vw, *vb;   // v, vw, vb: of the second derivative; w, b, vw, vb may be null
  const int8_t* codes;                       // in place of x
  const float* scales;
  int8_t* codes_out;                         // of the forward pass where x is kept in 8 bits
  float* scales_out;
  float eps;
  int silu;
  float *mean, *rstd;   // [samples, groups]; forward writes them (null: nobody wants them)
  void *out, *out_g, *out_w, *out_b;
  void* ws;
  int64_t ws_bytes;
  hipStream_t stream;
};

template <typename T>
void group_norm_fwd(const GroupNormCall& a);
template <typename T>
void group_norm_bwd(const GroupNormCall& a);
template <typename T>
void group_norm_bwd2(const GroupNormCall& a);

}  // namespace ictc

namespace {

// ---------------------------------------------------------------------------
// Chunks
// ---------------------------------------------------------------------------

// p[0 .. EV), or `none` throughout
template <typename T, int EV>
__device__ __forceinline__ void parameter(const T* __restrict__ p, int64_t at, bool ok, float none, float (&v)[EV]) {
  if (p && ok) {
    get<T, EV>(load_pack<T, EV>(p + at, true), v);
  } else {
#pragma unroll
    for (int e = 0; e < EV; ++e) v[e] = none;
  }
}

// A chunk of x as it lies in memory: elements, or codes and their scale.  from: its first element; block: its code block.
template <typename T, int EV, bool EIGHT>
struct Source {
  Pack<T, EV> raw;
  __device__ __forceinline__ void load(const ictc::GroupNormCall& a, int64_t from, int64_t, bool ok) {
    raw = load_pack<T, EV>((const T*)a.x + (ok ? from : 0), ok);
  }
  __device__ __forceinline__ void values(float (&v)[EV]) const { get<T, EV>(raw, v); }
};

typedef uint16_t u16_byte __attribute__((aligned(1)));

template <typename T, int EV>
struct Source<T, EV, true> {
  union {
    int8_t e[8];
    uint16_t b2;
    uint32_t b4, word[2];
    u32x2 b8;
  } raw;
  float scale;
  __device__ Source() {}
  __device__ __forceinline__ void load(const ictc::GroupNormCall& a, int64_t from, int64_t block, bool ok) {
    raw.b8 = u32x2{0, 0};
    scale = 0.f;
    if (!ok) return;
    const int8_t* p = a.codes + from;
    if constexpr (EV == 8) raw.b8 = *reinterpret_cast<const u32x2_byte*>(p);
    if constexpr (EV == 4) raw.b4 = *reinterpret_cast<const u32_byte*>(p);
    if constexpr (EV == 2) raw.b2 = *reinterpret_cast<const u16_byte*>(p);
    if constexpr (EV == 1) raw.e[0] = *p;
    scale = a.scales[block];
  }
  __device__ __forceinline__ void values(float (&v)[EV]) const {
    code_products<EV>(raw.word, scale, v);
#pragma unroll
    for (int e = 0; e < EV; ++e) v[e] = (float)(T)v[e];
  }
};

__device__ __forceinline__ int code_blocks(int C) { return (C + kCodeBlock - 1) / kCodeBlock; }

// ---------------------------------------------------------------------------
// The formulas, element by element
// ---------------------------------------------------------------------------

// act(z), and its derivatives.  (An exponential past FP32 makes the sigmoid zero, as it is to within 2^-128.)
template <bool SILU>
struct Act {
  float s, z;
  __device__ __forceinline__ Act(float z_) : z(z_) {
    constexpr float LOG2E = 1.44269504f;
    s = SILU ? __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-LOG2E * z)) : 1.f;
  }
  __device__ __forceinline__ float value() const { return SILU ? z * s : z; }
  __device__ __forceinline__ float slope() const { return SILU ? __builtin_fmaf(z * s, 1.f - s, s) : 1.f; }
  __device__ __forceinline__ float bend() const {
    return SILU ? s * (1.f - s) * __builtin_fmaf(z, 1.f - 2.f * s, 2.f) : 0.f;
  }
};

// Sums of a group that its gradients need (u, u h), and those that the gradients of the gradients need.
constexpr int kSums = 12;

template <bool SILU>
__device__ __forceinline__ void add_sums(float h, float r, float g, float v, float w, float b, float vw, float vb,
                                         float (&s)[kSums]) {
  const Act<SILU> a(h * w + b);
  const float ga = g * a.slope(), u = ga * w, t = ga * vw;
  s[0] += u;
  s[1] += u * h;
  s[2] += v;
  s[3] += v * h;
  s[4] += u * v;
  s[5] += t;
  s[6] += t * h;
  if (SILU) {
    const float wk = w * (g * a.bend()), part = wk * (w * r * v + h * vw + vb), wwk = w * wk, wwkh = wwk * h;
    s[7] += part;
    s[8] += part * h;
    s[9] += wwk;
    s[10] += wwkh;
    s[11] += wwkh * h;
  }
}

// What the second derivative's result needs of a group's sums.
struct Seconds {
  float v, vh, uh, tm, th, q;
  __device__ __forceinline__ Seconds() {}
  __device__ __forceinline__ Seconds(const float (&s)[kSums], float inv, float r) {
    float m[kSums];
#pragma unroll
    for (int k = 0; k < kSums; ++k) m[k] = s[k] * inv;
    v = m[2];
    vh = m[3];
    uh = m[1];
    tm = m[5] + (m[7] - r * (m[2] * m[9] + m[3] * m[10])) - r * (m[3] * m[0] + m[1] * m[2]);
    th = m[6] + (m[8] - r * (m[2] * m[10] + m[3] * m[11])) - 2.f * r * m[1] * m[3];
    q = m[4] - m[0] * m[2] - m[1] * m[3];
  }
  // (dx', dg') of an element, and its parts of dw' and db'
  template <bool SILU>
  __device__ __forceinline__ void element(float h, float r, float g, float vx, float w, float b, float vw, float vb,
                                          float& dx, float& dg, float& dw, float& db) const {
    const Act<SILU> a(h * w + b);
    const float slope = a.slope(), ga = g * slope, u = ga * w;
    const float pv = r * (vx - v - h * vh), e = w * pv + h * vw + vb, zz = e * (g * a.bend());
    const float t = ga * vw + zz * w - r * (vh * u + uh * vx);
    dx = r * (t - tm - h * th) - r * r * q * h;
    dg = e * slope;
    dw = ga * pv + zz * h;
    db = zz;
  }
};

// 1 / sqrt(var + eps) of a variance that may be past FP32
__device__ __forceinline__ float deviation(double var, float eps) { return (float)(1.0 / sqrt(var + (double)eps)); }

// ---------------------------------------------------------------------------
// Sums over lanes
// ---------------------------------------------------------------------------

template <int CTRL, typename V>
__device__ __forceinline__ V dpp_of(V x) {
  if constexpr (sizeof(V) == 4) {
    return dpp<CTRL>(x);
  } else {
    const u32x2 b = __builtin_bit_cast(u32x2, x);
    const u32x2 c = {(uint32_t)__builtin_amdgcn_mov_dpp((int)b[0], CTRL, 0xf, 0xf, false),
                     (uint32_t)__builtin_amdgcn_mov_dpp((int)b[1], CTRL, 0xf, 0xf, false)};
    return __builtin_bit_cast(V, c);
  }
}

#define GN_STEP(condition, value)                                \
  if (condition) {                                               \
    _Pragma("unroll") for (int k = 0; k < K; ++k) s[k] += value; \
  }
// Sums over aligned groups of n lanes, a power of two, in each of them.
template <int K, typename V>
__device__ __forceinline__ void sum_low(V (&s)[K], int n) {
  GN_STEP(n >= 2, dpp_of<0xB1>(s[k]))
  GN_STEP(n >= 4, dpp_of<0x4E>(s[k]))
  GN_STEP(n >= 8, dpp_of<0x141>(s[k]))
  GN_STEP(n >= 16, dpp_of<0x140>(s[k]))
  GN_STEP(n >= 32, __shfl_xor(s[k], 16))
  GN_STEP(n >= 64, __shfl_xor(s[k], 32))
}
// Sums over the lanes of a wave that agree modulo n, a power of two, in each of them.  (A rotation within 16 lanes is an
// exchange where the halves above it agree already.)
template <int K, typename V>
__device__ __forceinline__ void sum_high(V (&s)[K], int n) {
  GN_STEP(n <= 32, __shfl_xor(s[k], 32))
  GN_STEP(n <= 16, __shfl_xor(s[k], 16))
  GN_STEP(n <= 8, dpp_of<0x128>(s[k]))
  GN_STEP(n <= 4, dpp_of<0x124>(s[k]))
  GN_STEP(n <= 2, dpp_of<0x122>(s[k]))
  GN_STEP(n <= 1, dpp_of<0x121>(s[k]))
}
#undef GN_STEP

// ---------------------------------------------------------------------------
// Rows
// ---------------------------------------------------------------------------

// How the teams of a block are dealt out: `groups` of them side by side, `slots` samples at once; of a team's lanes `across`
// along a position's chunks, the rest along positions; a lane's next chunk is `rows` positions or `columns` chunks on.
struct RowsPlan {
  int team, shift, across, rows, columns;
  int groups, slots;
  int blocks_x, blocks_y;
};

struct RowsAt {
  int group, lane;
  bool on;
  int64_t sample, gap;
  __device__ __forceinline__ RowsAt(const RowsPlan& p, int G) {
    lane = threadIdx.x & (p.team - 1);
    const int t = threadIdx.x >> p.shift, slot = t / p.groups;
    group = blockIdx.y * p.groups + t % p.groups;
    on = slot < p.slots && group < G;
    sample = (int64_t)blockIdx.x * p.slots + slot;
    gap = (int64_t)gridDim.x * p.slots;
  }
};

// A lane's chunks: whether there is one, its channel, and where it is within its sample's elements and code blocks.
template <int EV, int N>
struct RowsChunks {
  bool ok[N];
  int c[N], from[N], block[N];
  __device__ __forceinline__ RowsChunks(const RowsPlan& p, const RowsAt& at, int per, int S, int C) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int row = at.lane / p.across + i * p.rows, col = ((at.lane & (p.across - 1)) + i * p.columns) * EV;
      ok[i] = at.on && row < S && col < per;
      c[i] = at.group * per + col;
      from[i] = row * C + c[i];
      block[i] = row * code_blocks(C) + c[i] / kCodeBlock;
    }
  }
};

// ENCODE: x to 8 bits as well, where the lanes of a code block are an aligned power of two of a wave's: `coded` lanes.
template <typename T, int EV, int N, bool SILU, bool ENCODE>
__global__ __launch_bounds__(256) void gn_rows_fwd_kernel(ictc::GroupNormCall a, RowsPlan p, int per, int coded) {
  const RowsAt at(p, a.groups);
  const int C = a.channels, S = (int)a.positions;
  const float inv = 1.f / ((float)per * (float)S);
  const RowsChunks<EV, N> k(p, at, per, S, C);
  float w[N][EV], b[N][EV];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    parameter<T, EV>((const T*)a.w, k.c[i], k.ok[i], 1.f, w[i]);
    parameter<T, EV>((const T*)a.b, k.c[i], k.ok[i], 0.f, b[i]);
  }
  if (!at.on) return;
  const int64_t size = (int64_t)S * C, blocks = (int64_t)S * code_blocks(C);
  for (int64_t n = at.sample; n < a.samples; n += at.gap) {
    const int64_t base = n * size;
    Pack<T, EV> raw[N];
#pragma unroll
    for (int i = 0; i < N; ++i) raw[i] = load_pack<T, EV>((const T*)a.x + (k.ok[i] ? base + k.from[i] : 0), k.ok[i]);
    float v[N][EV], s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < N; ++i) {
      get<T, EV>(raw[i], v[i]);
#pragma unroll
      for (int e = 0; e < EV; ++e) s[0] += v[i][e];
    }
    if constexpr (ENCODE) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < EV; ++e) top = max(top, magnitude(v[i][e]));
        const float scale = code_scale(lanes_top(top, coded)), inverse = 1.f / scale;
        Codes<EV> q;
#pragma unroll
        for (int e = 0; e < EV; ++e) q.e[e] = (int8_t)code_of(v[i][e], inverse);
        if (k.ok[i]) store_codes<EV>(a.codes_out + base + k.from[i], EV, q);
        if (k.ok[i] && (threadIdx.x & (coded - 1)) == 0) a.scales_out[n * blocks + k.block[i]] = scale;
      }
    }
    sum_low(s, p.team);
    // The deviations' own mean corrects the rounded one (a group of one value far from zero has no deviation left).
    const float first = s[0] * inv;
    float q[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int e = 0; e < EV; ++e) {
        v[i][e] = k.ok[i] ? v[i][e] - first : 0.f;
        q[0] += v[i][e];
        q[1] += v[i][e] * v[i][e];
      }
    sum_low(q, p.team);
    const float rest = q[0] * inv, mu = first + rest;
    float r = 1.f / sqrtf(fmaxf(q[1] * inv - rest * rest, 0.f) + a.eps);
    if (q[1] == __builtin_inff()) {   // finite deviations whose squares are past FP32: added again, scaled
      constexpr float SCALE = 0x1p-80f;
      s[0] = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int e = 0; e < EV; ++e) {
          const float d = (v[i][e] - rest) * SCALE;
          s[0] += k.ok[i] ? d * d : 0.f;
        }
      sum_low(s, p.team);
      r = SCALE / sqrtf(s[0] * inv + a.eps * SCALE * SCALE);
    }
    if (q[1] != q[1]) r = q[1];   // (fmaxf drops a NaN)
#pragma unroll
    for (int i = 0; i < N; ++i) {
#pragma unroll
      for (int e = 0; e < EV; ++e) v[i][e] = Act<SILU>((v[i][e] - rest) * r * w[i][e] + b[i][e]).value();
      if (k.ok[i]) store_pack<T, EV>((T*)a.out + base + k.from[i], v[i]);
    }
    if (at.lane == 0 && a.mean) {
      a.mean[n * a.groups + at.group] = mu;
      a.rstd[n * a.groups + at.group] = r;
    }
  }
}

// A block's sums by channel: acc of every lane, over the chunks of a channel (not where a lane's chunks are of other
// channels), a position's lanes and the slots, to part [channels].
template <int EV, int N>
__device__ __forceinline__ void rows_channels(float (&acc)[N][EV], const RowsPlan& p, const RowsAt& at, int per, int G,
                                              float* __restrict__ part, float* lds) {
  if (p.columns == 0) {
#pragma unroll
    for (int i = 1; i < N; ++i)
#pragma unroll
      for (int e = 0; e < EV; ++e) acc[0][e] += acc[i][e];
  }
  const int strips = p.team / p.across, lanes = p.groups * p.team;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (i > 0 && p.columns == 0) break;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < EV; ++e) lds[e * 256 + threadIdx.x] = acc[i][e];
    __syncthreads();
    for (int k = threadIdx.x; k < p.groups * p.across * EV; k += 256) {
      const int e = k % EV, lane = k / EV % p.across, gi = k / EV / p.across;
      const int col = (lane + i * p.columns) * EV + e, group = blockIdx.y * p.groups + gi;
      if (col >= per || group >= G) continue;
      float s = 0.f;
      for (int slot = 0; slot < p.slots; ++slot)
        for (int j = 0; j < strips; ++j) s += lds[e * 256 + slot * lanes + gi * p.team + j * p.across + lane];
      part[(int64_t)group * per + col] = s;
    }
  }
}

template <typename T, int EV, int N, bool SILU, bool EIGHT>
__global__ __launch_bounds__(256) void gn_rows_bwd_kernel(ictc::GroupNormCall a, RowsPlan p, int per,
                                                          float* __restrict__ part_w, float* __restrict__ part_b) {
  __shared__ float lds[EV * 256];
  const RowsAt at(p, a.groups);
  const int C = a.channels, S = (int)a.positions;
  const float inv = 1.f / ((float)per * (float)S);
  const RowsChunks<EV, N> k(p, at, per, S, C);
  float w[N][EV], b[N][EV], dw[N][EV], db[N][EV];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    parameter<T, EV>((const T*)a.w, k.c[i], k.ok[i], 1.f, w[i]);
    parameter<T, EV>((const T*)a.b, k.c[i], k.ok[i], 0.f, b[i]);
#pragma unroll
    for (int e = 0; e < EV; ++e) dw[i][e] = db[i][e] = 0.f;
  }
  const int64_t size = (int64_t)S * C, blocks = (int64_t)S * code_blocks(C);
  for (int64_t n = at.on ? at.sample : a.samples; n < a.samples; n += at.gap) {
    const int64_t base = n * size;
    Source<T, EV, EIGHT> rx[N];
    Pack<T, EV> rg[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      rx[i].load(a, base + k.from[i], n * blocks + k.block[i], k.ok[i]);
      rg[i] = load_pack<T, EV>((const T*)a.g + (k.ok[i] ? base + k.from[i] : 0), k.ok[i]);
    }
    const float mu = a.mean[n * a.groups + at.group], r = a.rstd[n * a.groups + at.group];
    float h[N][EV], u[N][EV], s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < N; ++i) {
      rx[i].values(h[i]);
      get<T, EV>(rg[i], u[i]);
#pragma unroll
      for (int e = 0; e < EV; ++e) {
        h[i][e] = (h[i][e] - mu) * r;
        const float ga = u[i][e] * Act<SILU>(h[i][e] * w[i][e] + b[i][e]).slope();
        dw[i][e] += ga * h[i][e];
        db[i][e] += ga;
        u[i][e] = ga * w[i][e];
        s[0] += u[i][e];
        s[1] += u[i][e] * h[i][e];
      }
    }
    if (!a.out) continue;
    sum_low(s, p.team);
    const float m = s[0] * inv, mh = s[1] * inv;
#pragma unroll
    for (int i = 0; i < N; ++i) {
#pragma unroll
      for (int e = 0; e < EV; ++e) u[i][e] = r * (u[i][e] - m - h[i][e] * mh);
      if (k.ok[i]) store_pack<T, EV>((T*)a.out + base + k.from[i], u[i]);
    }
  }
  if (part_w) rows_channels<EV, N>(dw, p, at, per, a.groups, part_w + (int64_t)blockIdx.x * C, lds);
  if (part_b) rows_channels<EV, N>(db, p, at, per, a.groups, part_b + (int64_t)blockIdx.x * C, lds);
}

template <typename T, int EV, int N, bool SILU, bool EIGHT>
__global__ __launch_bounds__(256) void gn_rows_bwd2_kernel(ictc::GroupNormCall a, RowsPlan p, int per,
                                                           float* __restrict__ part_w, float* __restrict__ part_b) {
  __shared__ float lds[EV * 256];
  const RowsAt at(p, a.groups);
  const int C = a.channels, S = (int)a.positions;
  const float inv = 1.f / ((float)per * (float)S);
  const RowsChunks<EV, N> k(p, at, per, S, C);
  float dw[N][EV], db[N][EV];
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int e = 0; e < EV; ++e) dw[i][e] = db[i][e] = 0.f;
  const int64_t size = (int64_t)S * C, blocks = (int64_t)S * code_blocks(C);
  for (int64_t n = at.on ? at.sample : a.samples; n < a.samples; n += at.gap) {
    const int64_t base = n * size;
    Source<T, EV, EIGHT> rx[N];
    Pack<T, EV> rg[N], rv[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int64_t from = k.ok[i] ? base + k.from[i] : 0;
      rx[i].load(a, base + k.from[i], n * blocks + k.block[i], k.ok[i]);
      rg[i] = load_pack<T, EV>((const T*)a.g + from, k.ok[i]);
      rv[i] = load_pack<T, EV>((const T*)a.v + from, k.ok[i]);
    }
    const float mu = a.mean[n * a.groups + at.group], r = a.rstd[n * a.groups + at.group];
    float s[kSums] = {};
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float x[EV], g[EV], v[EV], w[EV], b[EV], vw[EV], vb[EV];
      rx[i].values(x);
      get<T, EV>(rg[i], g);
      get<T, EV>(rv[i], v);
      parameter<T, EV>((const T*)a.w, k.c[i], k.ok[i], 1.f, w);
      parameter<T, EV>((const T*)a.b, k.c[i], k.ok[i], 0.f, b);
      parameter<T, EV>((const T*)a.vw, k.c[i], k.ok[i], 0.f, vw);
      parameter<T, EV>((const T*)a.vb, k.c[i], k.ok[i], 0.f, vb);
#pragma unroll
      for (int e = 0; e < EV; ++e) add_sums<SILU>((x[e] - mu) * r, r, g[e], v[e], w[e], b[e], vw[e], vb[e], s);
    }
    sum_low(s, p.team);
    const Seconds of(s, inv, r);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float x[EV], g[EV], v[EV], w[EV], b[EV], vw[EV], vb[EV], pw, pb;
      rx[i].values(x);
      get<T, EV>(rg[i], g);
      get<T, EV>(rv[i], v);
      parameter<T, EV>((const T*)a.w, k.c[i], k.ok[i], 1.f, w);
      parameter<T, EV>((const T*)a.b, k.c[i], k.ok[i], 0.f, b);
      parameter<T, EV>((const T*)a.vw, k.c[i], k.ok[i], 0.f, vw);
      parameter<T, EV>((const T*)a.vb, k.c[i], k.ok[i], 0.f, vb);
#pragma unroll
      for (int e = 0; e < EV; ++e) {
        of.element<SILU>((x[e] - mu) * r, r, g[e], v[e], w[e], b[e], vw[e], vb[e], x[e], v[e], pw, pb);
        dw[i][e] += k.ok[i] ? pw : 0.f;
        db[i][e] += k.ok[i] ? pb : 0.f;
      }
      if (!k.ok[i]) continue;
      if (a.out) store_pack<T, EV>((T*)a.out + base + k.from[i], x);
      if (a.out_g) store_pack<T, EV>((T*)a.out_g + base + k.from[i], v);
    }
  }
  if (part_w) rows_channels<EV, N>(dw, p, at, per, a.groups, part_w + (int64_t)blockIdx.x * C, lds);
  if (part_b) rows_channels<EV, N>(db, p, at, per, a.groups, part_b + (int64_t)blockIdx.x * C, lds);
}

// ---------------------------------------------------------------------------
// Tiles and parts
// ---------------------------------------------------------------------------

constexpr int kThreads = 256;

// Positions that a thread asks for at once: four, two of eight channels.  (More take registers that more waves need.)
template <int EV>
constexpr int kRowsAtOnce = EV >= 8 ? 2 : 4;

// A block's tile: `groups` whole groups of `chunks` chunks each, or where a group has more than a block's threads one of
// the group's `tiles_per` columns; `lanes` threads along it, `rows` positions at once; positions in `splits` of `per_split`.
// It takes every `slots`-th sample, so a thread's channels stay and their gradients are added over its samples.
struct TilePlan {
  int groups, chunks, lanes, rows, tiles, tiles_per;
  int splits, slots;
  int64_t per_split;
  int powers;   // lanes and chunks are powers of two within a wave
};

struct TileAt {
  int lane, row, c, group, local;   // thread's chunk and first position; first channel, its group, that group in the tile
  bool on, first;                   // whether it has a chunk; whether it is its group's first of the tile
  int64_t sample, begin, end;
  int split, slot, part;            // part: of a sample's group
  __device__ __forceinline__ TileAt(const TilePlan& p, int EV, int per, int G, int64_t S) {
    lane = threadIdx.x % p.lanes;
    row = threadIdx.x / p.lanes;
    const int b = die_order(blockIdx.x, gridDim.x);   // (tiles side by side share lines of a die's cache)
    const int tile = b % p.tiles, rest = b / p.tiles;
    split = rest % p.splits;
    sample = slot = rest / p.splits;
    if (p.tiles_per == 1) {
      local = lane / p.chunks;
      group = tile * p.groups + local;
      c = group * per + lane % p.chunks * EV;
      on = row < p.rows && group < G;
      first = on && row == 0 && lane == local * p.chunks;
      part = split;
    } else {
      local = 0;
      group = tile / p.tiles_per;
      const int column = tile % p.tiles_per, chunk = column * p.lanes + lane;
      c = group * per + chunk * EV;
      on = row < p.rows && chunk < p.chunks;
      first = on && row == 0 && lane == 0;
      part = split * p.tiles_per + column;
    }
    begin = split * p.per_split;
    end = min(S, begin + p.per_split);
  }
};

// K values of every thread, added over the positions' threads: in those of row 0, left in lds [K][256].
template <typename V, int K>
__device__ __forceinline__ void sum_rows(V (&s)[K], const TilePlan& p, const TileAt& at, V* lds) {
  __syncthreads();
  if (p.powers) {   // over a wave's lanes, then the waves in order
    sum_high(s, p.lanes);
    if ((int)(threadIdx.x & 63) < p.lanes) {
#pragma unroll
      for (int k = 0; k < K; ++k) lds[k * kThreads + threadIdx.x] = s[k];
    }
    __syncthreads();
    if ((int)threadIdx.x < p.lanes) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        V* q = lds + k * kThreads + threadIdx.x;
        q[0] = q[0] + q[64] + q[128] + q[192];
      }
    }
    __syncthreads();
    return;
  }
#pragma unroll
  for (int k = 0; k < K; ++k) lds[k * kThreads + threadIdx.x] = at.on ? s[k] : (V)0;
  __syncthreads();
  int step = 1;
  while (step < p.rows) step *= 2;
  for (step /= 2; step > 0; step /= 2) {
    if (at.row < step && at.row + step < p.rows) {
#pragma unroll
      for (int k = 0; k < K; ++k) lds[k * kThreads + threadIdx.x] += lds[k * kThreads + threadIdx.x + step * p.lanes];
    }
    __syncthreads();
  }
}

// lds [K][256]'s row 0, added over each group's threads: the sums in every thread of the group, whatever its row.
template <typename V, int K>
__device__ __forceinline__ void sum_groups(V (&s)[K], const TilePlan& p, const TileAt& at, V* lds) {
  const int chunks = p.tiles_per == 1 ? p.chunks : p.lanes, place = at.lane - at.local * chunks;
  int step = 1;
  while (step < chunks) step *= 2;
  for (step /= 2; step > 0; step /= 2) {
    if (at.row == 0 && place < step && place + step < chunks) {
#pragma unroll
      for (int k = 0; k < K; ++k) lds[k * kThreads + at.lane] += lds[k * kThreads + at.lane + step];
    }
    __syncthreads();
  }
#pragma unroll
  for (int k = 0; k < K; ++k) s[k] = lds[k * kThreads + at.local * chunks];
}

// K values of every thread, added over its group's threads of all positions, in each of them.
template <typename V, int K>
__device__ __forceinline__ void sum_all(V (&s)[K], const TilePlan& p, const TileAt& at, V* lds) {
  if (p.powers) {
    sum_low(s, p.chunks);
    sum_high(s, p.lanes);
    __syncthreads();
    if ((int)(threadIdx.x & 63) < p.lanes) {
#pragma unroll
      for (int k = 0; k < K; ++k) lds[k * kThreads + threadIdx.x] = s[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const V* q = lds + k * kThreads + at.lane;
      s[k] = q[0] + q[64] + q[128] + q[192];
    }
    return;
  }
  sum_rows(s, p, at, lds);
  sum_groups(s, p, at, lds);
}

// A thread's walk over its positions, U of them at once: f(first element of each, which of them there are, how many).
template <int U, typename F>
__device__ __forceinline__ void walk(const TilePlan& p, const TileAt& at, int64_t S, int C, F&& f) {
  if (!at.on) return;
  const int64_t step = (int64_t)p.rows * C, bstep = (int64_t)p.rows * code_blocks(C);
  const int64_t row = at.sample * S + at.begin + at.row;
  int64_t from = row * C + at.c, block = row * code_blocks(C) + at.c / kCodeBlock;
  for (int64_t left = at.end - at.begin - at.row; left > 0; left -= U * p.rows, from += U * step, block += U * bstep)
    f(from, step, block, bstep, (int)min<int64_t>(U, (left + p.rows - 1) / p.rows));
}

template <typename T, int EV>
__device__ __forceinline__ void tile_statistics(const ictc::GroupNormCall& a, const TilePlan& p, const TileAt& at,
                                                double (&s)[2], double* lds) {
  constexpr int U = kRowsAtOnce<EV>;
  s[0] = s[1] = 0.0;
  walk<U>(p, at, a.positions, a.channels, [&](int64_t from, int64_t step, int64_t, int64_t, int count) {
    Pack<T, EV> raw[U];
#pragma unroll
    for (int i = 0; i < U; ++i)
      raw[i] = load_pack<T, EV>((const T*)a.x + (i < count ? from + i * step : from), i < count);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      float v[EV];
      get<T, EV>(raw[i], v);
#pragma unroll
      for (int e = 0; e < EV; ++e) {
        const double d = v[e];
        s[0] += d;
        s[1] += d * d;
      }
    }
  });
  sum_all(s, p, at, lds);
}

struct Moments {
  float mean, rstd;
};

__device__ __forceinline__ Moments moments(double sum, double squares, double count, float eps) {
  const double mean = sum / count, var = squares / count - mean * mean;
  return {(float)mean, deviation(var < 0.0 ? 0.0 : var, eps)};
}

template <typename T, int EV, bool SILU>
__device__ __forceinline__ void tile_result(const ictc::GroupNormCall& a, const TilePlan& p, const TileAt& at,
                                            const Moments& m) {
  constexpr int U = kRowsAtOnce<EV>;
  float w[EV], b[EV];
  parameter<T, EV>((const T*)a.w, at.c, at.on, 1.f, w);
  parameter<T, EV>((const T*)a.b, at.c, at.on, 0.f, b);
  walk<U>(p, at, a.positions, a.channels, [&](int64_t from, int64_t step, int64_t, int64_t, int count) {
    Pack<T, EV> raw[U];
#pragma unroll
    for (int i = 0; i < U; ++i)
      raw[i] = load_pack<T, EV>((const T*)a.x + (i < count ? from + i * step : from), i < count);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (i >= count) break;
      float v[EV];
      get<T, EV>(raw[i], v);
#pragma unroll
      for (int e = 0; e < EV; ++e) v[e] = Act<SILU>((v[e] - m.mean) * m.rstd * w[e] + b[e]).value();
      store_pack<T, EV>((T*)a.out + from + i * step, v);
    }
  });
}

template <typename T, int EV, bool SILU>
__global__ __launch_bounds__(kThreads) void gn_tile_fwd_kernel(ictc::GroupNormCall a, TilePlan p, int per) {
  __shared__ double lds[2 * kThreads];
  TileAt at(p, EV, per, a.groups, a.positions);
  for (; at.sample < a.samples; at.sample += p.slots) {
    double s[2];
    tile_statistics<T, EV>(a, p, at, s, lds);
    const Moments m = moments(s[0], s[1], (double)per * (double)a.positions, a.eps);
    if (a.mean && at.first) {
      a.mean[at.sample * a.groups + at.group] = m.mean;
      a.rstd[at.sample * a.groups + at.group] = m.rstd;
    }
    tile_result<T, EV, SILU>(a, p, at, m);
  }
}

// part [samples][groups][splits tiles_per][2]
template <typename T, int EV>
__global__ __launch_bounds__(kThreads) void gn_part_stats_kernel(ictc::GroupNormCall a, TilePlan p, int per,
                                                                 double* __restrict__ part) {
  __shared__ double lds[2 * kThreads];
  TileAt at(p, EV, per, a.groups, a.positions);
  for (; at.sample < a.samples; at.sample += p.slots) {
    double s[2];
    tile_statistics<T, EV>(a, p, at, s, lds);
    if (at.first) {
      double* to = part + ((at.sample * a.groups + at.group) * (p.splits * p.tiles_per) + at.part) * 2;
      to[0] = s[0];
      to[1] = s[1];
    }
  }
}

// A wave's sum of K values of each of `parts` parts, lane by lane and then over the lanes, in each of them.
template <int K, typename V>
__device__ __forceinline__ void wave_parts(const V* __restrict__ part, int parts, V (&s)[K]) {
#pragma unroll
  for (int i = 0; i < K; ++i) s[i] = (V)0;
  for (int k = threadIdx.x & 63; k < parts; k += 64) {
#pragma unroll
    for (int i = 0; i < K; ++i) s[i] += part[(int64_t)k * K + i];
  }
#pragma unroll
  for (int i = 0; i < K; ++i)
    for (int d = 32; d > 0; d /= 2) s[i] += __shfl_xor(s[i], d);
}

// A wave a sample's group.
__global__ __launch_bounds__(256) void gn_part_moments_kernel(const double* __restrict__ part, int64_t units, int parts,
                                                              double count, float eps, float* __restrict__ mean,
                                                              float* __restrict__ rstd) {
  for (int64_t u = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); u < units; u += (int64_t)gridDim.x * 4) {
    double s[2];
    wave_parts<2>(part + u * parts * 2, parts, s);
    if ((threadIdx.x & 63) == 0) {
      const Moments m = moments(s[0], s[1], count, eps);
      mean[u] = m.mean;
      rstd[u] = m.rstd;
    }
  }
}

template <int K>
__global__ __launch_bounds__(256) void gn_part_sums_kernel(const float* __restrict__ part, int64_t units, int parts,
                                                           float* __restrict__ sums) {
  for (int64_t u = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); u < units; u += (int64_t)gridDim.x * 4) {
    float s[K];
    wave_parts<K>(part + u * parts * K, parts, s);
#pragma unroll
    for (int i = 0; i < K; ++i)
      if ((threadIdx.x & 63) == i) sums[u * K + i] = s[i];
  }
}

// Few parts (a lane each) are added by every block that needs them, for its tile's groups, without a launch of their own: K
// sums of the thread's group.  (Blocks of whole groups.)
constexpr int kOwnParts = 64, kOwnGroups = 16;

template <int K, typename V>
__device__ __forceinline__ void tile_parts(const V* __restrict__ part, int64_t sample, int groups, const TilePlan& p,
                                           const TileAt& at, V (&s)[K], V (*lds)[K]) {
  const int g0 = (at.group - at.local), wave = threadIdx.x >> 6;
  __syncthreads();
  for (int g = wave; g < p.groups && g0 + g < groups; g += kThreads / 64) {
    wave_parts<K>(part + ((sample * groups + g0 + g) * p.splits) * K, p.splits, s);
#pragma unroll
    for (int i = 0; i < K; ++i)
      if ((threadIdx.x & 63) == 0) lds[g][i] = s[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < K; ++i) s[i] = lds[at.local][i];
}

// part: the statistics' parts where the blocks add them themselves (and then those of split 0 write mean and rstd, if they
// are wanted); else null, and mean and rstd are read
template <typename T, int EV, bool SILU>
__global__ __launch_bounds__(kThreads) void gn_part_fwd_kernel(ictc::GroupNormCall a, TilePlan p, int per,
                                                               const double* __restrict__ part,
                                                               const float* __restrict__ mean,
                                                               const float* __restrict__ rstd) {
  __shared__ double lds[kOwnGroups][2];
  TileAt at(p, EV, per, a.groups, a.positions);
  for (; at.sample < a.samples; at.sample += p.slots) {
    Moments m = {0.f, 0.f};
    const int64_t u = at.sample * a.groups + at.group;
    if (part) {
      double s[2];
      tile_parts(part, at.sample, a.groups, p, at, s, lds);
      m = moments(s[0], s[1], (double)per * (double)a.positions, a.eps);
      if (a.mean && at.first && at.split == 0) {
        a.mean[u] = m.mean;
        a.rstd[u] = m.rstd;
      }
    } else if (at.on) {
      m = {mean[u], rstd[u]};
    }
    tile_result<T, EV, SILU>(a, p, at, m);
  }
}

// Sums over the tile's positions of ga and ga h by channel, left in lds [2 EV][256] (row 0).
template <typename T, int EV, bool SILU, bool EIGHT>
__device__ __forceinline__ void tile_channels(const ictc::GroupNormCall& a, const TilePlan& p, const TileAt& at,
                                              const Moments& m, const float (&w)[EV], const float (&b)[EV], float* lds) {
  constexpr int U = kRowsAtOnce<EV>;
  float s[2 * EV] = {};
  walk<U>(p, at, a.positions, a.channels, [&](int64_t from, int64_t step, int64_t block, int64_t bstep, int count) {
    Source<T, EV, EIGHT> rx[U];
    Pack<T, EV> rg[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      rx[i].load(a, from + i * step, block + i * bstep, i < count);
      rg[i] = load_pack<T, EV>((const T*)a.g + (i < count ? from + i * step : from), i < count);
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      float x[EV], g[EV];
      rx[i].values(x);
      get<T, EV>(rg[i], g);
#pragma unroll
      for (int e = 0; e < EV; ++e) {
        const float h = (x[e] - m.mean) * m.rstd, ga = g[e] * Act<SILU>(h * w[e] + b[e]).slope();
        s[e] += ga;
        s[EV + e] += ga * h;
      }
    }
  });
  sum_rows(s, p, at, lds);
}

template <typename T, int EV, bool SILU, bool EIGHT>
__device__ __forceinline__ void tile_gradient(const ictc::GroupNormCall& a, const TilePlan& p, const TileAt& at,
                                              const Moments& m, const float (&w)[EV], const float (&b)[EV], float mu,
                                              float muh) {
  constexpr int U = kRowsAtOnce<EV>;
  walk<U>(p, at, a.positions, a.channels, [&](int64_t from, int64_t step, int64_t block, int64_t bstep, int count) {
    Source<T, EV, EIGHT> rx[U];
    Pack<T, EV> rg[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      rx[i].load(a, from + i * step, block + i * bstep, i < count);
      rg[i] = load_pack<T, EV>((const T*)a.g + (i < count ? from + i * step : from), i < count);
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (i >= count) break;
      float x[EV], g[EV];
      rx[i].values(x);
      get<T, EV>(rg[i], g);
#pragma unroll
      for (int e = 0; e < EV; ++e) {
        const float h = (x[e] - m.mean) * m.rstd, ga = g[e] * Act<SILU>(h * w[e] + b[e]).slope();
        x[e] = m.rstd * (ga * w[e] - mu - h * muh);
      }
      store_pack<T, EV>((T*)a.out + from + i * step, x);
    }
  });
}

// A block's sums by channel over its samples, to the row of its slot and split of part_w and part_b.
template <int EV>
struct ChannelSums {
  float s[2 * EV];   // of row 0's threads: db, dw
  __device__ __forceinline__ ChannelSums() {
#pragma unroll
    for (int k = 0; k < 2 * EV; ++k) s[k] = 0.f;
  }
  __device__ __forceinline__ void add(const float* lds) {
#pragma unroll
    for (int k = 0; k < 2 * EV; ++k) s[k] += lds[k * kThreads + threadIdx.x];
  }
  __device__ __forceinline__ void write(const TilePlan& p, const TileAt& at, int C, float* __restrict__ part_w,
                                        float* __restrict__ part_b) const {
    if (!at.on || at.row != 0) return;
    const int64_t to = ((int64_t)at.slot * p.splits + at.split) * C + at.c;
#pragma unroll
    for (int e = 0; e < EV; ++e) {
      if (part_b) part_b[to + e] = s[e];
      if (part_w) part_w[to + e] = s[EV + e];
    }
  }
};

// FUSED: the row gradient follows at once; else sums [samples][groups][splits tiles_per][2] of u and u h.
// part_w, part_b [slots splits][channels]
template <typename T, int EV, bool SILU, bool EIGHT, bool FUSED>
__global__ __launch_bounds__(kThreads) void gn_tile_bwd_kernel(ictc::GroupNormCall a, TilePlan p, int per,
                                                               float* __restrict__ sums, float* __restrict__ part_w,
                                                               float* __restrict__ part_b) {
  __shared__ float lds[2 * EV * kThreads];
  TileAt at(p, EV, per, a.groups, a.positions);
  float w[EV], b[EV];
  parameter<T, EV>((const T*)a.w, at.c, at.on, 1.f, w);
  parameter<T, EV>((const T*)a.b, at.c, at.on, 0.f, b);
  const float inv = 1.f / ((float)per * (float)a.positions);
  ChannelSums<EV> channels;
  for (; at.sample < a.samples; at.sample += p.slots) {
    const int64_t u = at.on ? at.sample * a.groups + at.group : 0;
    const Moments m = {a.mean[u], a.rstd[u]};
    tile_channels<T, EV, SILU, EIGHT>(a, p, at, m, w, b, lds);
    float s[2] = {0.f, 0.f};
    if (at.on && at.row == 0) {
      channels.add(lds);
#pragma unroll
      for (int e = 0; e < EV; ++e) {
        s[0] += w[e] * lds[e * kThreads + threadIdx.x];
        s[1] += w[e] * lds[(EV + e) * kThreads + threadIdx.x];
      }
    }
    if (!a.out) continue;
    __syncthreads();
    lds[threadIdx.x] = s[0];
    lds[kThreads + threadIdx.x] = s[1];
    __syncthreads();
    sum_groups(s, p, at, lds);
    if constexpr (FUSED) {
      tile_gradient<T, EV, SILU, EIGHT>(a, p, at, m, w, b, s[0] * inv, s[1] * inv);
    } else if (at.first) {
      float* to = sums + (u * (p.splits * p.tiles_per) + at.part) * 2;
      to[0] = s[0];
      to[1] = s[1];
    }
  }
  channels.write(p, at, a.channels, part_w, part_b);
}

// own: sums are the parts', and the blocks add them themselves
template <typename T, int EV, bool SILU, bool EIGHT>
__global__ __launch_bounds__(kThreads) void gn_part_bwd_kernel(ictc::GroupNormCall a, TilePlan p, int per,
                                                               const float* __restrict__ sums, bool own) {
  __shared__ float lds[kOwnGroups][2];
  TileAt at(p, EV, per, a.groups, a.positions);
  float w[EV], b[EV];
  parameter<T, EV>((const T*)a.w, at.c, at.on, 1.f, w);
  parameter<T, EV>((const T*)a.b, at.c, at.on, 0.f, b);
  const float inv = 1.f / ((float)per * (float)a.positions);
  for (; at.sample < a.samples; at.sample += p.slots) {
    const int64_t u = at.on ? at.sample * a.groups + at.group : 0;
    float s[2];
    if (own) {
      tile_parts(sums, at.sample, a.groups, p, at, s, lds);
    } else {
      s[0] = sums[u * 2];
      s[1] = sums[u * 2 + 1];
    }
    tile_gradient<T, EV, SILU, EIGHT>(a, p, at, Moments{a.mean[u], a.rstd[u]}, w, b, s[0] * inv, s[1] * inv);
  }
}

// The second derivative's sums over the tile by group, in every thread of the group.
template <typename T, int EV, bool SILU, bool EIGHT>
__device__ __forceinline__ void tile_sums(const ictc::GroupNormCall& a, const TilePlan& p, const TileAt& at,
                                          const Moments& m, const float (&w)[EV], const float (&b)[EV],
                                          const float (&vw)[EV], const float (&vb)[EV], float (&s)[kSums], float* lds) {
#pragma unroll
  for (int k = 0; k < kSums; ++k) s[k] = 0.f;
  constexpr int U = 2;
  walk<U>(p, at, a.positions, a.channels, [&](int64_t from, int64_t step, int64_t block, int64_t bstep, int count) {
    Source<T, EV, EIGHT> rx[U];
    Pack<T, EV> rg[U], rv[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int64_t f = i < count ? from + i * step : from;
      rx[i].load(a, f, block + i * bstep, i < count);
      rg[i] = load_pack<T, EV>((const T*)a.g + f, i < count);
      rv[i] = load_pack<T, EV>((const T*)a.v + f, i < count);
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      float x[EV], g[EV], v[EV];
      rx[i].values(x);
      get<T, EV>(rg[i], g);
      get<T, EV>(rv[i], v);
#pragma unroll
      for (int e = 0; e < EV; ++e)
        add_sums<SILU>((x[e] - m.mean) * m.rstd, m.rstd, g[e], v[e], w[e], b[e], vw[e], vb[e], s);
    }
  });
  sum_all(s, p, at, lds);
}

// The second derivative's results over the tile, and its sums of db' and dw' by channel, left in lds [2 EV][256] (row 0).
template <typename T, int EV, bool SILU, bool EIGHT>
__device__ __forceinline__ void tile_second(const ictc::GroupNormCall& a, const TilePlan& p, const TileAt& at,
                                            const Moments& m, const float (&w)[EV], const float (&b)[EV],
                                            const float (&vw)[EV], const float (&vb)[EV], const Seconds& of, float* lds) {
  float s[2 * EV] = {};
  constexpr int U = 2;
  walk<U>(p, at, a.positions, a.channels, [&](int64_t from, int64_t step, int64_t block, int64_t bstep, int count) {
    Source<T, EV, EIGHT> rx[U];
    Pack<T, EV> rg[U], rv[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int64_t f = i < count ? from + i * step : from;
      rx[i].load(a, f, block + i * bstep, i < count);
      rg[i] = load_pack<T, EV>((const T*)a.g + f, i < count);
      rv[i] = load_pack<T, EV>((const T*)a.v + f, i < count);
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (i >= count) break;
      float x[EV], g[EV], v[EV], pw, pb;
      rx[i].values(x);
      get<T, EV>(rg[i], g);
      get<T, EV>(rv[i], v);
#pragma unroll
      for (int e = 0; e < EV; ++e) {
        of.element<SILU>((x[e] - m.mean) * m.rstd, m.rstd, g[e], v[e], w[e], b[e], vw[e], vb[e], x[e], v[e], pw, pb);
        s[e] += pb;
        s[EV + e] += pw;
      }
      if (a.out) store_pack<T, EV>((T*)a.out + from + i * step, x);
      if (a.out_g) store_pack<T, EV>((T*)a.out_g + from + i * step, v);
    }
  });
  if (a.out_w || a.out_b) sum_rows(s, p, at, lds);
}

// All in one; or the parts' sums to part [samples][groups][splits tiles_per][12]; or the results from sums
// [samples][groups][12] (own: from the parts', which the blocks add themselves).
enum class Phase { kAll, kSums, kResults };
template <typename T, int EV, bool SILU, bool EIGHT, Phase PHASE>
__global__ __launch_bounds__(kThreads) void gn_tile_bwd2_kernel(ictc::GroupNormCall a, TilePlan p, int per,
                                                                float* __restrict__ part, const float* __restrict__ sums,
                                                                bool own, float* __restrict__ part_w,
                                                                float* __restrict__ part_b) {
  constexpr int K = kSums > 2 * EV ? kSums : 2 * EV;
  __shared__ float lds[K * kThreads];
  TileAt at(p, EV, per, a.groups, a.positions);
  float w[EV], b[EV], vw[EV], vb[EV];
  parameter<T, EV>((const T*)a.w, at.c, at.on, 1.f, w);
  parameter<T, EV>((const T*)a.b, at.c, at.on, 0.f, b);
  parameter<T, EV>((const T*)a.vw, at.c, at.on, 0.f, vw);
  parameter<T, EV>((const T*)a.vb, at.c, at.on, 0.f, vb);
  const float inv = 1.f / ((float)per * (float)a.positions);
  ChannelSums<EV> channels;
  for (; at.sample < a.samples; at.sample += p.slots) {
    const int64_t u = at.on ? at.sample * a.groups + at.group : 0;
    const Moments m = {a.mean[u], a.rstd[u]};
    float s[kSums];
    if constexpr (PHASE != Phase::kResults) {
      tile_sums<T, EV, SILU, EIGHT>(a, p, at, m, w, b, vw, vb, s, lds);
    } else if (own) {
      tile_parts(sums, at.sample, a.groups, p, at, s, reinterpret_cast<float(*)[kSums]>(lds));
    } else {
#pragma unroll
      for (int i = 0; i < kSums; ++i) s[i] = sums[u * kSums + i];
    }
    if constexpr (PHASE == Phase::kSums) {
      if (at.first) {
        float* to = part + (u * (p.splits * p.tiles_per) + at.part) * kSums;
#pragma unroll
        for (int i = 0; i < kSums; ++i) to[i] = s[i];
      }
    } else {
      tile_second<T, EV, SILU, EIGHT>(a, p, at, m, w, b, vw, vb, Seconds(s, inv, m.rstd), lds);
      if ((a.out_w || a.out_b) && at.on && at.row == 0) channels.add(lds);
    }
  }
  if (PHASE != Phase::kSums) channels.write(p, at, a.channels, part_w, part_b);
}

// out[c] = sum over the parts' rows, 16 slices of them added per channel and then in order.
template <typename T>
__global__ __launch_bounds__(256) void gn_channels_kernel(const float* __restrict__ part_a, T* __restrict__ out_a,
                                                          const float* __restrict__ part_b, T* __restrict__ out_b,
                                                          int64_t parts, int C) {
  __shared__ float lds[16][17];
  const float* part = blockIdx.y ? part_b : part_a;
  T* out = blockIdx.y ? out_b : out_a;
  if (!out) return;
  const int col = threadIdx.x & 15, slice = threadIdx.x >> 4, c = blockIdx.x * 16 + col;
  float a = 0.f;
  if (c < C) {
#pragma unroll 8
    for (int64_t b = slice; b < parts; b += 16) a += part[b * C + c];
  }
  lds[slice][col] = a;
  __syncthreads();
  if (slice == 0 && c < C) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) s += lds[i][col];
    out[c] = (T)s;
  }
}

// ---------------------------------------------------------------------------
// Which form, and its launch
// ---------------------------------------------------------------------------

enum class Form { kRows, kTiles, kParts };

struct Plan {
  Form form;
  int ev, n;   // elements of a chunk; rows: chunks a lane
  RowsPlan rows;
  TilePlan tile;
  int64_t parts;   // rows of partial sums by channel
  int coded;       // rows: lanes of a code block where the forward pass makes the codes; 0: a kernel of their own does
};

inline int power_of_two(int64_t n) {
  int p = 1;
  while (p < n) p *= 2;
  return p;
}

inline Plan plan_of(int element, int64_t samples, int64_t positions, int channels, int groups) {
  Plan p = {};
  const int per = channels / groups;
  p.ev = 16 / element;
  while (per % p.ev) p.ev /= 2;
  const int chunks = per / p.ev;
  const int across = std::min(64, power_of_two(chunks));
  const int64_t strips = std::min<int64_t>(64 / across, power_of_two(std::min<int64_t>(positions, 64)));
  const int64_t n = positions == 1 ? (chunks + 63) / 64 : chunks > 64 ? 1 << 20 : (positions + strips - 1) / strips;
  if (n <= 4) {
    p.form = Form::kRows;
    p.n = n <= 1 ? 1 : n <= 2 ? 2 : 4;
    RowsPlan& r = p.rows;
    r.team = across * (int)strips;
    while ((1 << r.shift) < r.team) ++r.shift;
    r.across = across;
    r.rows = positions == 1 ? 0 : (int)strips;
    r.columns = positions == 1 ? across : 0;
    const int teams = 256 / r.team;
    r.groups = std::min(groups, teams);
    r.slots = teams / r.groups;
    r.blocks_y = (groups + r.groups - 1) / r.groups;
    const int64_t want = (samples + r.slots - 1) / r.slots;
    r.blocks_x = (int)std::max<int64_t>(1, std::min<int64_t>(want, std::max(1, 1024 / r.blocks_y)));
    p.parts = r.blocks_x;
    // every lane has a chunk, and a block of codes is an aligned power of two of lanes side by side
    const bool whole = positions == 1 && p.ev == 16 / element && (chunks <= 64 ? chunks == across : per % kCodeBlock == 0);
    const int lanes = std::min(channels, kCodeBlock) / p.ev;
    if (whole && (channels <= kCodeBlock ? power_of_two(lanes) == lanes : channels % kCodeBlock == 0) &&
        r.groups * r.team % lanes == 0)
      p.coded = lanes;
    return p;
  }
  TilePlan& t = p.tile;
  t.chunks = chunks;
  t.tiles_per = (chunks + kThreads - 1) / kThreads;
  if (t.tiles_per == 1) {
    // whole groups of 128 bytes a position or more, where there are
    const int want = std::max(1, 128 / (per * element));
    t.groups = std::min(groups, std::min(want, kThreads / chunks));
    // down to 32 bytes while there are few blocks, of samples that a block takes whole
    while (positions <= 32 * (kThreads / chunks) && t.groups > 1 && t.groups * per * element > 64 && samples * ((groups + t.groups - 1) / t.groups) < 512)
      t.groups = (t.groups + 1) / 2;
    t.lanes = t.groups * chunks;
    t.tiles = (groups + t.groups - 1) / t.groups;
  } else {
    t.groups = 1;
    t.lanes = kThreads;
    t.tiles = groups * t.tiles_per;
  }
  t.rows = (int)std::min<int64_t>(kThreads / t.lanes, positions);
  t.splits = 1;
  t.per_split = positions;
  const int64_t blocks = samples * t.tiles, steps = (positions + t.rows - 1) / t.rows;
  if (t.tiles_per == 1 && (blocks >= 512 || steps <= 32)) {
    p.form = Form::kTiles;
  } else {
    p.form = Form::kParts;
    const int64_t most = (steps + 3) / 4;   // (four positions a thread at least)
    const int64_t splits = std::max<int64_t>(1, std::min<int64_t>(most, (2048 + blocks) / (blocks + 1)));
    t.per_split = (steps + splits - 1) / splits * t.rows;
    t.splits = (int)((positions + t.per_split - 1) / t.per_split);
  }
  t.powers = t.lanes <= 64 && power_of_two(t.lanes) == t.lanes && power_of_two(chunks) == chunks;
  t.slots = (int)std::max<int64_t>(1, std::min<int64_t>(samples, 2048 / (t.tiles * t.splits)));
  p.parts = (int64_t)t.slots * t.splits;
  return p;
}

// Blocks of a wave for each sample's group.
inline dim3 unit_blocks(int64_t units) { return dim3((unsigned)std::max<int64_t>(1, std::min<int64_t>(1 << 20, (units + 3) / 4))); }

// Few parts of a group, for tiles of few whole groups: the blocks that need their sums add them.
inline bool own_parts(const TilePlan& p) { return p.tiles_per == 1 && p.splits <= kOwnParts && p.groups <= kOwnGroups; }

#define GN_ROWS(kernel, ...)                                                                                       \
  if (p.n == 1) {                                                                                                  \
    constexpr int N = 1;                                                                                           \
    hipLaunchKernelGGL((kernel), grid, dim3(256), 0, a.stream, __VA_ARGS__);                                       \
  } else if (p.n == 2) {                                                                                           \
    constexpr int N = 2;                                                                                           \
    hipLaunchKernelGGL((kernel), grid, dim3(256), 0, a.stream, __VA_ARGS__);                                       \
  } else {                                                                                                         \
    constexpr int N = 4;                                                                                           \
    hipLaunchKernelGGL((kernel), grid, dim3(256), 0, a.stream, __VA_ARGS__);                                       \
  }

template <typename T, int EV, bool SILU>
void launch_fwd(const ictc::GroupNormCall& a, const Plan& p) {
  const int per = a.channels / a.groups;
  if (p.form == Form::kRows) {
    const dim3 grid(p.rows.blocks_x, p.rows.blocks_y);
    if constexpr (EV == kChunk<T>) {
      if (a.codes_out && p.coded) {
        GN_ROWS((gn_rows_fwd_kernel<T, EV, N, SILU, true>), a, p.rows, per, p.coded)
        return;
      }
    }
    GN_ROWS((gn_rows_fwd_kernel<T, EV, N, SILU, false>), a, p.rows, per, 0)
    return;
  }
  const dim3 grid((unsigned)p.tile.slots * p.tile.splits * p.tile.tiles);
  if (p.form == Form::kTiles) {
    hipLaunchKernelGGL((gn_tile_fwd_kernel<T, EV, SILU>), grid, dim3(kThreads), 0, a.stream, a, p.tile, per);
    return;
  }
  const int64_t units = a.samples * a.groups;
  const int parts = p.tile.splits * p.tile.tiles_per;
  double* part = (double*)a.ws;
  float* mean = a.mean ? a.mean : (float*)(part + units * parts * 2);
  float* rstd = a.mean ? a.rstd : mean + units;
  hipLaunchKernelGGL((gn_part_stats_kernel<T, EV>), grid, dim3(kThreads), 0, a.stream, a, p.tile, per, part);
  const bool own = own_parts(p.tile);
  if (!own)
    hipLaunchKernelGGL(gn_part_moments_kernel, unit_blocks(units), dim3(256), 0, a.stream, part, units, parts,
                       (double)per * (double)a.positions, a.eps, mean, rstd);
  hipLaunchKernelGGL((gn_part_fwd_kernel<T, EV, SILU>), grid, dim3(kThreads), 0, a.stream, a, p.tile, per,
                     own ? part : nullptr, mean, rstd);
}

template <typename T>
void launch_channels(const ictc::GroupNormCall& a, const Plan& p, const float* part_w, const float* part_b) {
  if (a.out_w || a.out_b)
    hipLaunchKernelGGL(gn_channels_kernel<T>, dim3((unsigned)((a.channels + 15) / 16), 2), dim3(256), 0, a.stream, part_w,
                       (T*)a.out_w, part_b, (T*)a.out_b, p.parts, a.channels);
}

// Where the second and first derivatives' workspace begins: sums by channel; then, of parts, K sums of each part and of
// each sample's group.
struct Workspace {
  float *w, *b, *part, *sums;
  Workspace(const ictc::GroupNormCall& a, const Plan& p, int K) {
    const int64_t size = p.parts * a.channels;
    w = (float*)a.ws;
    b = w + size;
    part = b + size;
    sums = part + a.samples * a.groups * (p.tile.splits * p.tile.tiles_per) * K;
  }
};

// The parts' sums of every sample's group, or the parts themselves for blocks that add them.
template <int K>
const float* launch_sums(const ictc::GroupNormCall& a, const Plan& p, const Workspace& ws, bool own) {
  if (own) return ws.part;
  const int64_t units = a.samples * a.groups;
  hipLaunchKernelGGL(gn_part_sums_kernel<K>, unit_blocks(units), dim3(256), 0, a.stream, ws.part, units,
                     p.tile.splits * p.tile.tiles_per, ws.sums);
  return ws.sums;
}

template <typename T, int EV, bool SILU, bool EIGHT>
void launch_bwd(const ictc::GroupNormCall& a, const Plan& p) {
  const int per = a.channels / a.groups;
  const Workspace ws(a, p, 2);
  float *pw = a.out_w ? ws.w : nullptr, *pb = a.out_b ? ws.b : nullptr;
  if (p.form == Form::kRows) {
    const dim3 grid(p.rows.blocks_x, p.rows.blocks_y);
    GN_ROWS((gn_rows_bwd_kernel<T, EV, N, SILU, EIGHT>), a, p.rows, per, pw, pb)
  } else {
    const bool parts = p.form == Form::kParts, own = own_parts(p.tile);
    const dim3 grid((unsigned)p.tile.slots * p.tile.splits * p.tile.tiles);
    if (parts)
      hipLaunchKernelGGL((gn_tile_bwd_kernel<T, EV, SILU, EIGHT, false>), grid, dim3(kThreads), 0, a.stream, a, p.tile, per,
                         ws.part, pw, pb);
    else
      hipLaunchKernelGGL((gn_tile_bwd_kernel<T, EV, SILU, EIGHT, true>), grid, dim3(kThreads), 0, a.stream, a, p.tile, per,
                         (float*)nullptr, pw, pb);
    if (parts && a.out) {
      const float* sums = launch_sums<2>(a, p, ws, own);
      hipLaunchKernelGGL((gn_part_bwd_kernel<T, EV, SILU, EIGHT>), grid, dim3(kThreads), 0, a.stream, a, p.tile, per, sums,
                         own);
    }
  }
  launch_channels<T>(a, p, pw, pb);
}

template <typename T, int EV, bool SILU, bool EIGHT>
void launch_bwd2(const ictc::GroupNormCall& a, const Plan& p) {
  const int per = a.channels / a.groups;
  const Workspace ws(a, p, kSums);
  float *pw = a.out_w ? ws.w : nullptr, *pb = a.out_b ? ws.b : nullptr;
  if (p.form == Form::kRows) {
    const dim3 grid(p.rows.blocks_x, p.rows.blocks_y);
    GN_ROWS((gn_rows_bwd2_kernel<T, EV, N, SILU, EIGHT>), a, p.rows, per, pw, pb)
  } else {
    const bool own = own_parts(p.tile);
    const dim3 grid((unsigned)p.tile.slots * p.tile.splits * p.tile.tiles);
    float* none = nullptr;
    const float* sums = nullptr;
    if (p.form == Form::kParts) {
      hipLaunchKernelGGL((gn_tile_bwd2_kernel<T, EV, SILU, EIGHT, Phase::kSums>), grid, dim3(kThreads), 0, a.stream, a,
                         p.tile, per, ws.part, sums, false, none, none);
      sums = launch_sums<kSums>(a, p, ws, own);
      hipLaunchKernelGGL((gn_tile_bwd2_kernel<T, EV, SILU, EIGHT, Phase::kResults>), grid, dim3(kThreads), 0, a.stream, a,
                         p.tile, per, none, sums, own, pw, pb);
    } else {
      hipLaunchKernelGGL((gn_tile_bwd2_kernel<T, EV, SILU, EIGHT, Phase::kAll>), grid, dim3(kThreads), 0, a.stream, a,
                         p.tile, per, none, sums, false, pw, pb);
    }
  }
  launch_channels<T>(a, p, pw, pb);
}

}  // namespace

namespace ictc {

#define GN_CHUNKS(launch)                                      \
  const Plan p = plan_of((int)sizeof(T), a.samples, a.positions, a.channels, a.groups); \
  if constexpr (sizeof(T) == 2) {                              \
    if (p.ev == 8) { constexpr int EV = 8; return launch; }    \
  }                                                            \
  if (p.ev == 4) { constexpr int EV = 4; return launch; }      \
  if (p.ev == 2) { constexpr int EV = 2; return launch; }      \
  constexpr int EV = 1;                                        \
  return launch;

template <typename T>
void group_norm_fwd(const GroupNormCall& a) {
  GN_CHUNKS((a.silu ? launch_fwd<T, EV, true>(a, p) : launch_fwd<T, EV, false>(a, p)))
}

#define GN_KIND(f) \
  (a.codes ? a.silu ? f<T, EV, true, true>(a, p) : f<T, EV, false, true>(a, p) \
           : a.silu ? f<T, EV, true, false>(a, p) : f<T, EV, false, false>(a, p))

template <typename T>
void group_norm_bwd(const GroupNormCall& a) {
  GN_CHUNKS(GN_KIND(launch_bwd))
}
template <typename T>
void group_norm_bwd2(const GroupNormCall& a) {
  GN_CHUNKS(GN_KIND(launch_bwd2))
}

}  // namespace ictc
