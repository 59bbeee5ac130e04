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

// A chunk of x as it lies in memory: elements, or codes and their scale.
template <typename T, int EV, bool EIGHT>
struct Source {
  Pack<T, EV> raw;
  __device__ __forceinline__ void load(const T* __restrict__ x, const int8_t*, const float*, int64_t row, int C, int c,
                                       bool ok) {
    raw = load_pack<T, EV>(x + (ok ? row * C + c : 0), ok);
  }
  __device__ __forceinline__ void values(float (&v)[EV]) const { get<T, EV>(raw, v); }
};

template <int EV>
union CodePack {
  int8_t e[EV];
  uint8_t b1;
  uint16_t b2;
  uint32_t b4;
  u32x2 b8;
  __device__ CodePack() {}
};
typedef uint16_t u16_byte __attribute__((aligned(1)));

template <typename T, int EV>
struct Source<T, EV, true> {
  CodePack<(EV < 8 ? 8 : EV)> raw;
  float scale;
  __device__ __forceinline__ void load(const T*, const int8_t* __restrict__ codes, const float* __restrict__ scales,
                                       int64_t row, int C, int c, bool ok) {
    raw.b8 = u32x2{0, 0};
    scale = 0.f;
    if (!ok) return;
    const int8_t* p = codes + row * C + c;
    if constexpr (EV == 8) raw.b8 = *reinterpret_cast<const u32x2_byte*>(p);
    if constexpr (EV == 4) raw.b4 = *reinterpret_cast<const u32_byte*>(p);
    if constexpr (EV == 2) raw.b2 = *reinterpret_cast<const u16_byte*>(p);
    if constexpr (EV == 1) raw.e[0] = *p;
    scale = scales[row * ((C + kCodeBlock - 1) / kCodeBlock) + c / kCodeBlock];
  }
  __device__ __forceinline__ void values(float (&v)[EV]) const {
#pragma unroll
    for (int e = 0; e < EV; ++e) v[e] = code_value<T>(raw.e[e], scale);
  }
};

// ---------------------------------------------------------------------------
// The formulas, element by element
// ---------------------------------------------------------------------------

// act(z), and its derivatives.  (An exponential past FP32 makes the sigmoid zero, as it is to within 2^-128.)
struct Act {
  float s, z;
  int silu;
  __device__ __forceinline__ Act(float z_, int silu_) : z(z_), silu(silu_) {
    s = silu ? __builtin_amdgcn_rcpf(1.f + __expf(-z)) : 1.f;
  }
  __device__ __forceinline__ float value() const { return silu ? z * s : z; }
  __device__ __forceinline__ float slope() const { return silu ? s * (1.f + z * (1.f - s)) : 1.f; }
  __device__ __forceinline__ float bend() const { return silu ? s * (1.f - s) * (2.f + z * (1.f - 2.f * s)) : 0.f; }
};

// Sums of a group that its gradients need (u, u h), and those that the gradients of the gradients need.
constexpr int kSums = 12;

__device__ __forceinline__ void add_sums(float h, float r, float g, float v, float w, float b, float vw, float vb,
                                         int silu, float (&s)[kSums]) {
  const Act a(h * w + b, silu);
  const float ga = g * a.slope(), u = ga * w, t = ga * vw;
  s[0] += u;
  s[1] += u * h;
  s[2] += v;
  s[3] += v * h;
  s[4] += u * v;
  s[5] += t;
  s[6] += t * h;
  if (silu) {
    const float wk = w * (g * a.bend()), part = wk * (w * r * v + h * vw + vb), wwk = w * wk;
    s[7] += part;
    s[8] += part * h;
    s[9] += wwk;
    s[10] += wwk * h;
    s[11] += wwk * h * h;
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
  __device__ __forceinline__ void element(float h, float r, float g, float vx, float w, float b, float vw, float vb,
                                          int silu, float& dx, float& dg, float& dw, float& db) const {
    const Act a(h * w + b, silu);
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
// Rows
// ---------------------------------------------------------------------------

// Sums over the aligned team of lanes (a power of two up to 64), in each of them.
template <int K>
__device__ __forceinline__ void team_sum(float (&s)[K], int team) {
#define GN_STEP(lanes, value)                   \
  if (team >= lanes) {                          \
    _Pragma("unroll") for (int k = 0; k < K; ++k) s[k] += value; \
  }
  GN_STEP(2, dpp<0xB1>(s[k]))
  GN_STEP(4, dpp<0x4E>(s[k]))
  GN_STEP(8, dpp<0x141>(s[k]))
  GN_STEP(16, dpp<0x140>(s[k]))
  GN_STEP(32, __shfl_xor(s[k], 16))
  GN_STEP(64, __shfl_xor(s[k], 32))
#undef GN_STEP
}

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

template <typename T, int EV, int N>
__global__ __launch_bounds__(256) void gn_rows_fwd_kernel(ictc::GroupNormCall a, RowsPlan p, int per) {
  const RowsAt at(p, a.groups);
  const int C = a.channels, S = (int)a.positions;
  const float inv = 1.f / ((float)per * (float)S);
  float w[N][EV], b[N][EV];
  bool ok[N];
  int row[N], c[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    row[i] = at.lane / p.across + i * p.rows;
    const int col = ((at.lane & (p.across - 1)) + i * p.columns) * EV;
    ok[i] = at.on && row[i] < S && col < per;
    c[i] = at.group * per + col;
    parameter<T, EV>((const T*)a.w, c[i], ok[i], 1.f, w[i]);
    parameter<T, EV>((const T*)a.b, c[i], ok[i], 0.f, b[i]);
  }
  if (!at.on) return;
  for (int64_t n = at.sample; n < a.samples; n += at.gap) {
    Pack<T, EV> raw[N];
#pragma unroll
    for (int i = 0; i < N; ++i) raw[i] = load_pack<T, EV>((const T*)a.x + (ok[i] ? (n * S + row[i]) * C + c[i] : 0), ok[i]);
    float v[N][EV], s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < N; ++i) {
      get<T, EV>(raw[i], v[i]);
#pragma unroll
      for (int e = 0; e < EV; ++e) s[0] += v[i][e];
    }
    team_sum(s, p.team);
    // The deviations' own mean corrects the rounded one (a group of one value far from zero has no deviation left).
    const float first = s[0] * inv;
    float q[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int e = 0; e < EV; ++e) {
        v[i][e] = ok[i] ? v[i][e] - first : 0.f;
        q[0] += v[i][e];
        q[1] += v[i][e] * v[i][e];
      }
    team_sum(q, p.team);
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
          s[0] += ok[i] ? d * d : 0.f;
        }
      team_sum(s, p.team);
      r = SCALE / sqrtf(s[0] * inv + a.eps * SCALE * SCALE);
    }
    if (q[1] != q[1]) r = q[1];   // (fmaxf drops a NaN)
#pragma unroll
    for (int i = 0; i < N; ++i) {
#pragma unroll
      for (int e = 0; e < EV; ++e) v[i][e] = Act((v[i][e] - rest) * r * w[i][e] + b[i][e], a.silu).value();
      if (ok[i]) store_pack<T, EV>((T*)a.out + (n * S + row[i]) * C + c[i], v[i]);
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

template <typename T, int EV, int N, bool EIGHT>
__global__ __launch_bounds__(256) void gn_rows_bwd_kernel(ictc::GroupNormCall a, RowsPlan p, int per,
                                                          float* __restrict__ part_w, float* __restrict__ part_b) {
  __shared__ float lds[EV * 256];
  const RowsAt at(p, a.groups);
  const int C = a.channels, S = (int)a.positions;
  const float inv = 1.f / ((float)per * (float)S);
  float w[N][EV], b[N][EV], dw[N][EV], db[N][EV];
  bool ok[N];
  int row[N], c[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    row[i] = at.lane / p.across + i * p.rows;
    const int col = ((at.lane & (p.across - 1)) + i * p.columns) * EV;
    ok[i] = at.on && row[i] < S && col < per;
    c[i] = at.group * per + col;
    parameter<T, EV>((const T*)a.w, c[i], ok[i], 1.f, w[i]);
    parameter<T, EV>((const T*)a.b, c[i], ok[i], 0.f, b[i]);
#pragma unroll
    for (int e = 0; e < EV; ++e) dw[i][e] = db[i][e] = 0.f;
  }
  for (int64_t n = at.on ? at.sample : a.samples; n < a.samples; n += at.gap) {
    Source<T, EV, EIGHT> rx[N];
    Pack<T, EV> rg[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      rx[i].load((const T*)a.x, a.codes, a.scales, n * S + row[i], C, c[i], ok[i]);
      rg[i] = load_pack<T, EV>((const T*)a.g + (ok[i] ? (n * S + row[i]) * C + c[i] : 0), ok[i]);
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
        const float ga = u[i][e] * Act(h[i][e] * w[i][e] + b[i][e], a.silu).slope();
        dw[i][e] += ga * h[i][e];
        db[i][e] += ga;
        u[i][e] = ga * w[i][e];
        s[0] += u[i][e];
        s[1] += u[i][e] * h[i][e];
      }
    }
    if (!a.out) continue;
    team_sum(s, p.team);
    const float m = s[0] * inv, mh = s[1] * inv;
#pragma unroll
    for (int i = 0; i < N; ++i) {
#pragma unroll
      for (int e = 0; e < EV; ++e) u[i][e] = r * (u[i][e] - m - h[i][e] * mh);
      if (ok[i]) store_pack<T, EV>((T*)a.out + (n * S + row[i]) * C + c[i], u[i]);
    }
  }
  if (part_w) rows_channels<EV, N>(dw, p, at, per, a.groups, part_w + (int64_t)blockIdx.x * C, lds);
  if (part_b) rows_channels<EV, N>(db, p, at, per, a.groups, part_b + (int64_t)blockIdx.x * C, lds);
}

template <typename T, int EV, int N, bool EIGHT>
__global__ __launch_bounds__(256) void gn_rows_bwd2_kernel(ictc::GroupNormCall a, RowsPlan p, int per,
                                                           float* __restrict__ part_w, float* __restrict__ part_b) {
  __shared__ float lds[EV * 256];
  const RowsAt at(p, a.groups);
  const int C = a.channels, S = (int)a.positions;
  const float inv = 1.f / ((float)per * (float)S);
  float dw[N][EV], db[N][EV];
  bool ok[N];
  int row[N], c[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    row[i] = at.lane / p.across + i * p.rows;
    const int col = ((at.lane & (p.across - 1)) + i * p.columns) * EV;
    ok[i] = at.on && row[i] < S && col < per;
    c[i] = at.group * per + col;
#pragma unroll
    for (int e = 0; e < EV; ++e) dw[i][e] = db[i][e] = 0.f;
  }
  for (int64_t n = at.on ? at.sample : a.samples; n < a.samples; n += at.gap) {
    Source<T, EV, EIGHT> rx[N];
    Pack<T, EV> rg[N], rv[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int64_t from = ok[i] ? (n * S + row[i]) * C + c[i] : 0;
      rx[i].load((const T*)a.x, a.codes, a.scales, n * S + row[i], C, c[i], ok[i]);
      rg[i] = load_pack<T, EV>((const T*)a.g + from, ok[i]);
      rv[i] = load_pack<T, EV>((const T*)a.v + from, ok[i]);
    }
    const float mu = a.mean[n * a.groups + at.group], r = a.rstd[n * a.groups + at.group];
    float s[kSums] = {};
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float x[EV], g[EV], v[EV], w[EV], b[EV], vw[EV], vb[EV];
      rx[i].values(x);
      get<T, EV>(rg[i], g);
      get<T, EV>(rv[i], v);
      parameter<T, EV>((const T*)a.w, c[i], ok[i], 1.f, w);
      parameter<T, EV>((const T*)a.b, c[i], ok[i], 0.f, b);
      parameter<T, EV>((const T*)a.vw, c[i], ok[i], 0.f, vw);
      parameter<T, EV>((const T*)a.vb, c[i], ok[i], 0.f, vb);
#pragma unroll
      for (int e = 0; e < EV; ++e) add_sums((x[e] - mu) * r, r, g[e], v[e], w[e], b[e], vw[e], vb[e], a.silu, s);
    }
    team_sum(s, p.team);
    const Seconds of(s, inv, r);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float x[EV], g[EV], v[EV], w[EV], b[EV], vw[EV], vb[EV], pw, pb;
      rx[i].values(x);
      get<T, EV>(rg[i], g);
      get<T, EV>(rv[i], v);
      parameter<T, EV>((const T*)a.w, c[i], ok[i], 1.f, w);
      parameter<T, EV>((const T*)a.b, c[i], ok[i], 0.f, b);
      parameter<T, EV>((const T*)a.vw, c[i], ok[i], 0.f, vw);
      parameter<T, EV>((const T*)a.vb, c[i], ok[i], 0.f, vb);
#pragma unroll
      for (int e = 0; e < EV; ++e) {
        of.element((x[e] - mu) * r, r, g[e], v[e], w[e], b[e], vw[e], vb[e], a.silu, x[e], v[e], pw, pb);
        dw[i][e] += ok[i] ? pw : 0.f;
        db[i][e] += ok[i] ? pb : 0.f;
      }
      if (!ok[i]) continue;
      const int64_t to = (n * S + row[i]) * C + c[i];
      if (a.out) store_pack<T, EV>((T*)a.out + to, x);
      if (a.out_g) store_pack<T, EV>((T*)a.out_g + to, v);
    }
  }
  if (part_w) rows_channels<EV, N>(dw, p, at, per, a.groups, part_w + (int64_t)blockIdx.x * C, lds);
  if (part_b) rows_channels<EV, N>(db, p, at, per, a.groups, part_b + (int64_t)blockIdx.x * C, lds);
}

// ---------------------------------------------------------------------------
// Tiles and parts
// ---------------------------------------------------------------------------

constexpr int kRowsAtOnce = 4, kThreads = 256;

// A block's tile: `groups` whole groups of `chunks` chunks each, or where a group has more than a block's threads one of
// the group's `tiles_per` columns; `lanes` threads along it, `rows` positions at once; positions in `splits` of `per_split`.
// It takes every `slots`-th sample, so a thread's channels stay and their gradients are added over its samples.
struct TilePlan {
  int groups, chunks, lanes, rows, tiles, tiles_per;
  int splits, slots;
  int64_t per_split;
};

struct TileAt {
  int lane, row, c, group, local;   // thread's chunk and first position; first channel, its group, that group in the tile
  bool on, first;                   // whether it has a chunk; whether it is its group's first of the tile
  int64_t sample, begin, end;
  int split, slot, part;            // part: of a sample's group
  __device__ __forceinline__ TileAt(const TilePlan& p, int EV, int per, int G, int64_t S) {
    lane = threadIdx.x % p.lanes;
    row = threadIdx.x / p.lanes;
    const int tile = blockIdx.x % p.tiles, rest = blockIdx.x / p.tiles;
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

template <typename T, int EV>
__device__ __forceinline__ void tile_statistics(const ictc::GroupNormCall& a, const TilePlan& p, const TileAt& at,
                                                double (&s)[2], double* lds) {
  const T* x = (const T*)a.x + at.sample * a.positions * a.channels + at.c;
  s[0] = s[1] = 0.0;
  for (int64_t q = at.begin + at.row; at.on && q < at.end; q += kRowsAtOnce * p.rows) {
    Pack<T, EV> raw[kRowsAtOnce];
#pragma unroll
    for (int i = 0; i < kRowsAtOnce; ++i) {
      const int64_t n = q + i * p.rows;
      raw[i] = load_pack<T, EV>(x + (n < at.end ? n : q) * a.channels, n < at.end);
    }
#pragma unroll
    for (int i = 0; i < kRowsAtOnce; ++i) {
      float v[EV];
      get<T, EV>(raw[i], v);
#pragma unroll
      for (int e = 0; e < EV; ++e) {
        const double d = v[e];
        s[0] += d;
        s[1] += d * d;
      }
    }
  }
  sum_rows(s, p, at, lds);
  sum_groups(s, p, at, lds);
}

struct Moments {
  float mean, rstd;
};

__device__ __forceinline__ Moments moments(double sum, double squares, double count, float eps) {
  const double mean = sum / count, var = squares / count - mean * mean;
  return {(float)mean, deviation(var < 0.0 ? 0.0 : var, eps)};
}

template <typename T, int EV>
__device__ __forceinline__ void tile_result(const ictc::GroupNormCall& a, const TilePlan& p, const TileAt& at,
                                            const Moments& m) {
  if (!at.on) return;
  float w[EV], b[EV];
  parameter<T, EV>((const T*)a.w, at.c, true, 1.f, w);
  parameter<T, EV>((const T*)a.b, at.c, true, 0.f, b);
  const int64_t base = at.sample * a.positions * a.channels + at.c;
  for (int64_t q = at.begin + at.row; q < at.end; q += kRowsAtOnce * p.rows) {
    Pack<T, EV> raw[kRowsAtOnce];
#pragma unroll
    for (int i = 0; i < kRowsAtOnce; ++i) {
      const int64_t n = q + i * p.rows;
      raw[i] = load_pack<T, EV>((const T*)a.x + base + (n < at.end ? n : q) * a.channels, n < at.end);
    }
#pragma unroll
    for (int i = 0; i < kRowsAtOnce; ++i) {
      const int64_t n = q + i * p.rows;
      if (n >= at.end) break;
      float v[EV];
      get<T, EV>(raw[i], v);
#pragma unroll
      for (int e = 0; e < EV; ++e) v[e] = Act((v[e] - m.mean) * m.rstd * w[e] + b[e], a.silu).value();
      store_pack<T, EV>((T*)a.out + base + n * a.channels, v);
    }
  }
}

template <typename T, int EV>
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
    tile_result<T, EV>(a, p, at, m);
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

// A wave a sample's group: its parts, lane by lane and then over the lanes.
__global__ __launch_bounds__(256) void gn_part_moments_kernel(const double* __restrict__ part, int64_t units, int parts,
                                                              double count, float eps, float* __restrict__ mean,
                                                              float* __restrict__ rstd) {
  const int lane = threadIdx.x & 63;
  for (int64_t u = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); u < units; u += (int64_t)gridDim.x * 4) {
    double s = 0.0, q = 0.0;
    for (int k = lane; k < parts; k += 64) {
      s += part[(u * parts + k) * 2];
      q += part[(u * parts + k) * 2 + 1];
    }
    for (int d = 32; d > 0; d /= 2) {
      s += __shfl_xor(s, d);
      q += __shfl_xor(q, d);
    }
    if (lane == 0) {
      const Moments m = moments(s, q, count, eps);
      mean[u] = m.mean;
      rstd[u] = m.rstd;
    }
  }
}

template <typename T, int EV>
__global__ __launch_bounds__(kThreads) void gn_part_fwd_kernel(ictc::GroupNormCall a, TilePlan p, int per,
                                                               const float* __restrict__ mean,
                                                               const float* __restrict__ rstd) {
  TileAt at(p, EV, per, a.groups, a.positions);
  if (!at.on) return;
  for (; at.sample < a.samples; at.sample += p.slots) {
    const int64_t u = at.sample * a.groups + at.group;
    tile_result<T, EV>(a, p, at, Moments{mean[u], rstd[u]});
  }
}

// Sums over the tile's positions of ga and ga h by channel, left in lds [2 EV][256] (row 0).
template <typename T, int EV, bool EIGHT>
__device__ __forceinline__ void tile_channels(const ictc::GroupNormCall& a, const TilePlan& p, const TileAt& at,
                                              const Moments& m, const float (&w)[EV], const float (&b)[EV], float* lds) {
  float s[2 * EV] = {};
  const int64_t row0 = at.sample * a.positions;
  for (int64_t q = at.begin + at.row; at.on && q < at.end; q += kRowsAtOnce * p.rows) {
    Source<T, EV, EIGHT> rx[kRowsAtOnce];
    Pack<T, EV> rg[kRowsAtOnce];
#pragma unroll
    for (int i = 0; i < kRowsAtOnce; ++i) {
      const int64_t n = q + i * p.rows;
      rx[i].load((const T*)a.x, a.codes, a.scales, row0 + n, a.channels, at.c, n < at.end);
      rg[i] = load_pack<T, EV>((const T*)a.g + (n < at.end ? (row0 + n) * a.channels + at.c : 0), n < at.end);
    }
#pragma unroll
    for (int i = 0; i < kRowsAtOnce; ++i) {
      float x[EV], g[EV];
      rx[i].values(x);
      get<T, EV>(rg[i], g);
#pragma unroll
      for (int e = 0; e < EV; ++e) {
        const float h = (x[e] - m.mean) * m.rstd, ga = g[e] * Act(h * w[e] + b[e], a.silu).slope();
        s[e] += ga;
        s[EV + e] += ga * h;
      }
    }
  }
  sum_rows(s, p, at, lds);
}

template <typename T, int EV, bool EIGHT>
__device__ __forceinline__ void tile_gradient(const ictc::GroupNormCall& a, const TilePlan& p, const TileAt& at,
                                              const Moments& m, const float (&w)[EV], const float (&b)[EV], float mu,
                                              float muh) {
  const int64_t row0 = at.sample * a.positions;
  for (int64_t q = at.begin + at.row; at.on && q < at.end; q += kRowsAtOnce * p.rows) {
    Source<T, EV, EIGHT> rx[kRowsAtOnce];
    Pack<T, EV> rg[kRowsAtOnce];
#pragma unroll
    for (int i = 0; i < kRowsAtOnce; ++i) {
      const int64_t n = q + i * p.rows;
      rx[i].load((const T*)a.x, a.codes, a.scales, row0 + n, a.channels, at.c, n < at.end);
      rg[i] = load_pack<T, EV>((const T*)a.g + (n < at.end ? (row0 + n) * a.channels + at.c : 0), n < at.end);
    }
#pragma unroll
    for (int i = 0; i < kRowsAtOnce; ++i) {
      const int64_t n = q + i * p.rows;
      if (n >= at.end) break;
      float x[EV], g[EV];
      rx[i].values(x);
      get<T, EV>(rg[i], g);
#pragma unroll
      for (int e = 0; e < EV; ++e) {
        const float h = (x[e] - m.mean) * m.rstd, ga = g[e] * Act(h * w[e] + b[e], a.silu).slope();
        x[e] = m.rstd * (ga * w[e] - mu - h * muh);
      }
      store_pack<T, EV>((T*)a.out + (row0 + n) * a.channels + at.c, x);
    }
  }
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

// sums: null, the row gradient follows at once; else [samples][groups][splits tiles_per][2]: sums of u and u h.
// part_w, part_b [slots splits][channels]
template <typename T, int EV, bool EIGHT>
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
    tile_channels<T, EV, EIGHT>(a, p, at, m, w, b, lds);
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
    if (!sums) {
      tile_gradient<T, EV, EIGHT>(a, p, at, m, w, b, s[0] * inv, s[1] * inv);
    } else if (at.first) {
      float* to = sums + (u * (p.splits * p.tiles_per) + at.part) * 2;
      to[0] = s[0];
      to[1] = s[1];
    }
  }
  channels.write(p, at, a.channels, part_w, part_b);
}

// A wave a sample's group: its parts' K sums, lane by lane and then over the lanes.
template <int K>
__global__ __launch_bounds__(256) void gn_part_sums_kernel(const float* __restrict__ part, int64_t units, int parts,
                                                           float* __restrict__ sums) {
  const int lane = threadIdx.x & 63;
  for (int64_t u = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); u < units; u += (int64_t)gridDim.x * 4) {
    float s[K] = {};
    for (int k = lane; k < parts; k += 64) {
#pragma unroll
      for (int i = 0; i < K; ++i) s[i] += part[(u * parts + k) * K + i];
    }
    team_sum(s, 64);
#pragma unroll
    for (int i = 0; i < K; ++i)
      if (lane == i) sums[u * K + i] = s[i];
  }
}

template <typename T, int EV, bool EIGHT>
__global__ __launch_bounds__(kThreads) void gn_part_bwd_kernel(ictc::GroupNormCall a, TilePlan p, int per,
                                                               const float* __restrict__ sums) {
  TileAt at(p, EV, per, a.groups, a.positions);
  if (!at.on) return;
  float w[EV], b[EV];
  parameter<T, EV>((const T*)a.w, at.c, true, 1.f, w);
  parameter<T, EV>((const T*)a.b, at.c, true, 0.f, b);
  const float inv = 1.f / ((float)per * (float)a.positions);
  for (; at.sample < a.samples; at.sample += p.slots) {
    const int64_t u = at.sample * a.groups + at.group;
    tile_gradient<T, EV, EIGHT>(a, p, at, Moments{a.mean[u], a.rstd[u]}, w, b, sums[u * 2] * inv, sums[u * 2 + 1] * inv);
  }
}

// The second derivative's sums over the tile by group, in every thread of the group.
template <typename T, int EV, bool EIGHT>
__device__ __forceinline__ void tile_sums(const ictc::GroupNormCall& a, const TilePlan& p, const TileAt& at,
                                          const Moments& m, const float (&w)[EV], const float (&b)[EV],
                                          const float (&vw)[EV], const float (&vb)[EV], float (&s)[kSums], float* lds) {
#pragma unroll
  for (int k = 0; k < kSums; ++k) s[k] = 0.f;
  const int64_t row0 = at.sample * a.positions;
  constexpr int U = 2;
  for (int64_t q = at.begin + at.row; at.on && q < at.end; q += U * p.rows) {
    Source<T, EV, EIGHT> rx[U];
    Pack<T, EV> rg[U], rv[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int64_t n = q + i * p.rows, from = n < at.end ? (row0 + n) * a.channels + at.c : 0;
      rx[i].load((const T*)a.x, a.codes, a.scales, row0 + n, a.channels, at.c, n < at.end);
      rg[i] = load_pack<T, EV>((const T*)a.g + from, n < at.end);
      rv[i] = load_pack<T, EV>((const T*)a.v + from, n < at.end);
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      float x[EV], g[EV], v[EV];
      rx[i].values(x);
      get<T, EV>(rg[i], g);
      get<T, EV>(rv[i], v);
#pragma unroll
      for (int e = 0; e < EV; ++e)
        add_sums((x[e] - m.mean) * m.rstd, m.rstd, g[e], v[e], w[e], b[e], vw[e], vb[e], a.silu, s);
    }
  }
  sum_rows(s, p, at, lds);
  sum_groups(s, p, at, lds);
}

// The second derivative's results over the tile, and its sums of db' and dw' by channel, left in lds [2 EV][256] (row 0).
template <typename T, int EV, bool EIGHT>
__device__ __forceinline__ void tile_second(const ictc::GroupNormCall& a, const TilePlan& p, const TileAt& at,
                                            const Moments& m, const float (&w)[EV], const float (&b)[EV],
                                            const float (&vw)[EV], const float (&vb)[EV], const Seconds& of, float* lds) {
  float s[2 * EV] = {};
  const int64_t row0 = at.sample * a.positions;
  constexpr int U = 2;
  for (int64_t q = at.begin + at.row; at.on && q < at.end; q += U * p.rows) {
    Source<T, EV, EIGHT> rx[U];
    Pack<T, EV> rg[U], rv[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int64_t n = q + i * p.rows, from = n < at.end ? (row0 + n) * a.channels + at.c : 0;
      rx[i].load((const T*)a.x, a.codes, a.scales, row0 + n, a.channels, at.c, n < at.end);
      rg[i] = load_pack<T, EV>((const T*)a.g + from, n < at.end);
      rv[i] = load_pack<T, EV>((const T*)a.v + from, n < at.end);
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int64_t n = q + i * p.rows;
      if (n >= at.end) break;
      float x[EV], g[EV], v[EV], pw, pb;
      rx[i].values(x);
      get<T, EV>(rg[i], g);
      get<T, EV>(rv[i], v);
#pragma unroll
      for (int e = 0; e < EV; ++e) {
        of.element((x[e] - m.mean) * m.rstd, m.rstd, g[e], v[e], w[e], b[e], vw[e], vb[e], a.silu, x[e], v[e], pw, pb);
        s[e] += pb;
        s[EV + e] += pw;
      }
      const int64_t to = (row0 + n) * a.channels + at.c;
      if (a.out) store_pack<T, EV>((T*)a.out + to, x);
      if (a.out_g) store_pack<T, EV>((T*)a.out_g + to, v);
    }
  }
  if (a.out_w || a.out_b) sum_rows(s, p, at, lds);
}

// All in one (part and sums null); or the parts' sums to part [samples][groups][splits tiles_per][12]; or the results from
// sums [samples][groups][12].
template <typename T, int EV, bool EIGHT>
__global__ __launch_bounds__(kThreads) void gn_tile_bwd2_kernel(ictc::GroupNormCall a, TilePlan p, int per,
                                                                float* __restrict__ part, const float* __restrict__ sums,
                                                                float* __restrict__ part_w, float* __restrict__ part_b) {
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
    if (sums) {
#pragma unroll
      for (int i = 0; i < kSums; ++i) s[i] = sums[u * kSums + i];
    } else {
      tile_sums<T, EV, EIGHT>(a, p, at, m, w, b, vw, vb, s, lds);
    }
    if (part) {
      if (at.first) {
        float* to = part + (u * (p.splits * p.tiles_per) + at.part) * kSums;
#pragma unroll
        for (int i = 0; i < kSums; ++i) to[i] = s[i];
      }
      continue;
    }
    tile_second<T, EV, EIGHT>(a, p, at, m, w, b, vw, vb, Seconds(s, inv, m.rstd), lds);
    if ((a.out_w || a.out_b) && at.on && at.row == 0) channels.add(lds);
  }
  if (!part) channels.write(p, at, a.channels, part_w, part_b);
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
    return p;
  }
  TilePlan& t = p.tile;
  t.chunks = chunks;
  t.tiles_per = (chunks + kThreads - 1) / kThreads;
  if (t.tiles_per == 1) {
    // whole groups of 128 bytes a position or more, where there are
    const int want = std::max(1, 128 / (per * element));
    t.groups = std::min(groups, std::min(want, kThreads / chunks));
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
  t.slots = (int)std::max<int64_t>(1, std::min<int64_t>(samples, 2048 / (t.tiles * t.splits)));
  p.parts = (int64_t)t.slots * t.splits;
  return p;
}

// Blocks of a wave for each sample's group.
inline dim3 unit_blocks(int64_t units) { return dim3((unsigned)std::max<int64_t>(1, std::min<int64_t>(1 << 20, (units + 3) / 4))); }

#define GN_ROWS(kernel, ...)                                                                          \
  if (p.n == 1) { constexpr int N = 1; hipLaunchKernelGGL((kernel), grid, dim3(256), 0, a.stream, __VA_ARGS__); } \
  else if (p.n == 2) { constexpr int N = 2; hipLaunchKernelGGL((kernel), grid, dim3(256), 0, a.stream, __VA_ARGS__); } \
  else { constexpr int N = 4; hipLaunchKernelGGL((kernel), grid, dim3(256), 0, a.stream, __VA_ARGS__); }

template <typename T, int EV>
void launch_fwd(const ictc::GroupNormCall& a, const Plan& p) {
  const int per = a.channels / a.groups;
  if (p.form == Form::kRows) {
    const dim3 grid(p.rows.blocks_x, p.rows.blocks_y);
    GN_ROWS((gn_rows_fwd_kernel<T, EV, N>), a, p.rows, per)
    return;
  }
  const dim3 grid((unsigned)p.tile.slots * p.tile.splits * p.tile.tiles);
  if (p.form == Form::kTiles) {
    hipLaunchKernelGGL((gn_tile_fwd_kernel<T, EV>), grid, dim3(kThreads), 0, a.stream, a, p.tile, per);
    return;
  }
  const int64_t units = a.samples * a.groups;
  const int parts = p.tile.splits * p.tile.tiles_per;
  double* part = (double*)a.ws;
  float* mean = a.mean ? a.mean : (float*)(part + units * parts * 2);
  float* rstd = a.mean ? a.rstd : mean + units;
  hipLaunchKernelGGL((gn_part_stats_kernel<T, EV>), grid, dim3(kThreads), 0, a.stream, a, p.tile, per, part);
  hipLaunchKernelGGL(gn_part_moments_kernel, unit_blocks(units), dim3(256), 0, a.stream, part, units, parts,
                     (double)per * (double)a.positions, a.eps, mean, rstd);
  hipLaunchKernelGGL((gn_part_fwd_kernel<T, EV>), grid, dim3(kThreads), 0, a.stream, a, p.tile, per, mean, rstd);
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

template <typename T, int EV, bool EIGHT>
void launch_bwd(const ictc::GroupNormCall& a, const Plan& p) {
  const int per = a.channels / a.groups;
  const Workspace ws(a, p, 2);
  float *pw = a.out_w ? ws.w : nullptr, *pb = a.out_b ? ws.b : nullptr;
  if (p.form == Form::kRows) {
    const dim3 grid(p.rows.blocks_x, p.rows.blocks_y);
    GN_ROWS((gn_rows_bwd_kernel<T, EV, N, EIGHT>), a, p.rows, per, pw, pb)
  } else {
    const bool parts = p.form == Form::kParts;
    const dim3 grid((unsigned)p.tile.slots * p.tile.splits * p.tile.tiles);
    hipLaunchKernelGGL((gn_tile_bwd_kernel<T, EV, EIGHT>), grid, dim3(kThreads), 0, a.stream, a, p.tile, per,
                       parts ? ws.part : nullptr, pw, pb);
    if (parts && a.out) {
      const int64_t units = a.samples * a.groups;
      hipLaunchKernelGGL(gn_part_sums_kernel<2>, unit_blocks(units), dim3(256), 0, a.stream, ws.part, units,
                         p.tile.splits * p.tile.tiles_per, ws.sums);
      hipLaunchKernelGGL((gn_part_bwd_kernel<T, EV, EIGHT>), grid, dim3(kThreads), 0, a.stream, a, p.tile, per, ws.sums);
    }
  }
  launch_channels<T>(a, p, pw, pb);
}

template <typename T, int EV, bool EIGHT>
void launch_bwd2(const ictc::GroupNormCall& a, const Plan& p) {
  const int per = a.channels / a.groups;
  const Workspace ws(a, p, kSums);
  float *pw = a.out_w ? ws.w : nullptr, *pb = a.out_b ? ws.b : nullptr;
  if (p.form == Form::kRows) {
    const dim3 grid(p.rows.blocks_x, p.rows.blocks_y);
    GN_ROWS((gn_rows_bwd2_kernel<T, EV, N, EIGHT>), a, p.rows, per, pw, pb)
  } else {
    const bool parts = p.form == Form::kParts;
    const dim3 grid((unsigned)p.tile.slots * p.tile.splits * p.tile.tiles);
    float* none = nullptr;
    if (parts) {
      const int64_t units = a.samples * a.groups;
      hipLaunchKernelGGL((gn_tile_bwd2_kernel<T, EV, EIGHT>), grid, dim3(kThreads), 0, a.stream, a, p.tile, per, ws.part,
                         none, none, none);
      hipLaunchKernelGGL(gn_part_sums_kernel<kSums>, unit_blocks(units), dim3(256), 0, a.stream, ws.part, units,
                         p.tile.splits * p.tile.tiles_per, ws.sums);
    }
    hipLaunchKernelGGL((gn_tile_bwd2_kernel<T, EV, EIGHT>), grid, dim3(kThreads), 0, a.stream, a, p.tile, per, none,
                       parts ? ws.sums : none, pw, pb);
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
  GN_CHUNKS((launch_fwd<T, EV>(a, p)))
}
template <typename T>
void group_norm_bwd(const GroupNormCall& a) {
  GN_CHUNKS((a.codes ? launch_bwd<T, EV, true>(a, p) : launch_bwd<T, EV, false>(a, p)))
}
template <typename T>
void group_norm_bwd2(const GroupNormCall& a) {
  GN_CHUNKS((a.codes ? launch_bwd2<T, EV, true>(a, p) : launch_bwd2<T, EV, false>(a, p)))
}

}  // namespace ictc
