// The group norm of samples that a team of lanes holds in registers (group_norm.h has the formulas).
#pragma once
#include "group_norm.h"

namespace {

// How the teams of a block are dealt out: `groups` of them side by side, `slots` samples at once; of a team's lanes `across`
// along a position's chunks, the rest along positions; a lane's next chunk is `rows` positions or `columns` chunks on.
struct RowsPlan {
  int team, shift, across, rows, columns;
  int groups, slots;
  int blocks_x, blocks_fwd, blocks_y;
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

// A lane's chunks: their elements (0: none), channel, and where they are within the sample's elements and code blocks.
template <int EV, int N, bool PART>
struct RowsChunks {
  int n[N], c[N], from[N], block[N], border[N];
  __device__ __forceinline__ RowsChunks(const RowsPlan& p, const RowsAt& at, int per, int S, int C) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int row = at.lane / p.across + i * p.rows, col = ((at.lane & (p.across - 1)) + i * p.columns) * EV;
      n[i] = at.on && row < S && col < per ? (PART ? min(EV, per - col) : EV) : 0;
      c[i] = at.group * per + col;
      from[i] = row * C + c[i];
      block[i] = row * code_blocks(C) + c[i] / kCodeBlock;
      border[i] = PART ? kCodeBlock - c[i] % kCodeBlock : EV;
    }
  }
};

// Sums over the team, in each of its lanes.  WIDE: the team is the block.
template <bool WIDE, int K>
__device__ __forceinline__ void rows_sum(float (&s)[K], int team, float* cross) {
  if constexpr (!WIDE) {
    sum_low(s, team);
    return;
  }
  sum_low(s, 64);
  if ((threadIdx.x & 63) == 0) {
#pragma unroll
    for (int k = 0; k < K; ++k) cross[(threadIdx.x >> 6) * K + k] = s[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) s[k] = cross[k] + cross[K + k] + cross[2 * K + k] + cross[3 * K + k];
  __syncthreads();
}

// ENCODE: x to 8 bits as well, where the lanes of a code block are an aligned power of two of a wave's: `coded` lanes.
template <typename T, int EV, int N, bool WIDE, bool PART, bool SILU, bool ENCODE>
__global__ __launch_bounds__(256) void gn_rows_fwd_kernel(ictc::GroupNormCall a, RowsPlan p, int per, int coded) {
  __shared__ float cross[WIDE ? 8 : 1];
  const RowsAt at(p, a.groups);
  const int C = a.channels, S = (int)a.positions;
  const float count = (float)per * (float)S, inv = 1.f / count;
  const RowsChunks<EV, N, PART> k(p, at, per, S, C);
  float w[N][EV], b[N][EV];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    parameter<T, EV, PART>((const T*)a.w, k.c[i], k.n[i], 1.f, w[i]);
    parameter<T, EV, PART>((const T*)a.b, k.c[i], k.n[i], 0.f, b[i]);
  }
  if (!WIDE && !at.on) return;
  const int64_t size = (int64_t)S * C, blocks = (int64_t)S * code_blocks(C), end = a.samples * size;
  for (int64_t n = at.sample; n < a.samples; n += at.gap) {
    const int64_t base = n * size;
    Pack<T, EV> raw[N];
#pragma unroll
    for (int i = 0; i < N; ++i) raw[i] = load_part<T, EV, PART>((const T*)a.x, base + k.from[i], k.n[i], end);
    float v[N][EV], s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < N; ++i) {
      get<T, EV>(raw[i], v[i]);
      cut<PART>(v[i], k.n[i]);
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
        if (k.n[i] > 0) store_codes<EV>(a.codes_out + base + k.from[i], EV, q);
        if (k.n[i] > 0 && (threadIdx.x & (coded - 1)) == 0) a.scales_out[n * blocks + k.block[i]] = scale;
      }
    }
    rows_sum<WIDE>(s, p.team, cross);
    // The deviations' own mean corrects the rounded one, a quotient to the last bit (a group of one value far from zero has
    // no deviation left).  (Held: one value wherever it is used, none of them joined with the product.)
    const float first = held(s[0] * inv);
    float q[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int e = 0; e < EV; ++e) {
        v[i][e] = (PART ? e : 0) < k.n[i] ? v[i][e] - first : 0.f;
        q[0] += v[i][e];
        q[1] += v[i][e] * v[i][e];
      }
    rows_sum<WIDE>(q, p.team, cross);
    const float about = q[0] * inv, rest = __builtin_fmaf(__builtin_fmaf(-about, count, q[0]), inv, about);
    float r = 1.f / sqrtf(fmaxf(q[1] * inv - rest * rest, 0.f) + a.eps);
    // (the whole team) squares past FP32 of finite deviations, or hardly any but the mean's: added again, without that, scaled
    if (q[1] == __builtin_inff() || 2.f * rest * rest > q[1] * inv) {
      const bool past = q[1] == __builtin_inff();
      const float scale = past ? 0x1p-80f : 1.f;
      s[0] = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int e = 0; e < EV; ++e) {
          const float d = (v[i][e] - rest) * scale;
          s[0] += (PART ? e : 0) < k.n[i] ? d * d : 0.f;
        }
      rows_sum<WIDE>(s, p.team, cross);
      r = past ? fminf(scale / sqrtf(s[0] * inv), 1.f / sqrtf(a.eps)) : 1.f / sqrtf(s[0] * inv + a.eps);
    }
    if (q[1] != q[1]) r = q[1];   // (fmaxf drops a NaN)
#pragma unroll
    for (int i = 0; i < N; ++i) {
#pragma unroll
      for (int e = 0; e < EV; ++e) v[i][e] = Act<SILU>((v[i][e] - rest) * r * w[i][e] + b[i][e]).value();
      if (k.n[i] > 0) store_part<T, EV, PART>((T*)a.out + base + k.from[i], k.n[i], v[i]);
    }
    if (at.lane == 0 && a.mean) {
      a.mean[n * a.groups + at.group] = first + rest;
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

// The team's mean as the backward passes take it: of FP32 x with what its rounding to `mean` left, the mean of x less it,
// where that counts: half a unit of a mean of up to eight deviations 1 / r is 2^-21 of one.  (425,991 x 64 in eight groups,
// gradients 60 us; looked for by every team, or read from memory, 66.)
template <typename T, int EV, int N, bool WIDE, bool PART, bool EIGHT, typename X>
__device__ __forceinline__ Mean rows_mean(const X (&rx)[N], const int (&n)[N], float mean, float r, float inv, int team,
                                          float* cross) {
  if (sizeof(T) == 2 || EIGHT || !(fabsf(mean) * r > 8.f)) return {mean, 0.f};   // (the whole team)
  float s[1] = {0.f};
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float v[EV];
    rx[i].values(v);
#pragma unroll
    for (int e = 0; e < EV; ++e) s[0] += (PART ? e : 0) < n[i] ? v[e] - mean : 0.f;
  }
  rows_sum<WIDE>(s, team, cross);
  return {mean, s[0] * inv};
}

template <typename T, int EV, int N, bool WIDE, bool PART, bool SILU, bool EIGHT>
__global__ __launch_bounds__(256) void gn_rows_bwd_kernel(ictc::GroupNormCall a, RowsPlan p, int per,
                                                          float* __restrict__ part_w, float* __restrict__ part_b) {
  __shared__ float lds[EV * 256];
  const RowsAt at(p, a.groups);
  const int C = a.channels, S = (int)a.positions;
  const float inv = 1.f / ((float)per * (float)S);
  const RowsChunks<EV, N, PART> k(p, at, per, S, C);
  float w[N][EV], b[N][EV], dw[N][EV], db[N][EV];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    parameter<T, EV, PART>((const T*)a.w, k.c[i], k.n[i], 1.f, w[i]);
    parameter<T, EV, PART>((const T*)a.b, k.c[i], k.n[i], 0.f, b[i]);
#pragma unroll
    for (int e = 0; e < EV; ++e) dw[i][e] = db[i][e] = 0.f;
  }
  const int64_t size = (int64_t)S * C, blocks = (int64_t)S * code_blocks(C), end = a.samples * size;
  for (int64_t n = at.on ? at.sample : a.samples; n < a.samples; n += at.gap) {
    const int64_t base = n * size;
    Source<T, EV, EIGHT, PART> rx[N];
    Pack<T, EV> rg[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      rx[i].load(a, base + k.from[i], n * blocks + k.block[i], k.border[i], k.n[i], end);
      rg[i] = load_part<T, EV, PART>((const T*)a.g, base + k.from[i], k.n[i], end);
    }
    const float r = a.rstd[n * a.groups + at.group];
    const Mean mu = rows_mean<T, EV, N, WIDE, PART, EIGHT>(rx, k.n, a.mean[n * a.groups + at.group], r, inv, p.team, lds);
    float h[N][EV], u[N][EV], s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < N; ++i) {
      rx[i].values(h[i]);
      get<T, EV>(rg[i], u[i]);
      cut<PART>(u[i], k.n[i]);
#pragma unroll
      for (int e = 0; e < EV; ++e) {
        // (what there is not has no deviation: zero less a large mean, times r, may be infinite)
        h[i][e] = ((PART ? e : 0) < k.n[i] ? mu.off(h[i][e]) : 0.f) * r;
        const float ga = u[i][e] * Act<SILU>(h[i][e] * w[i][e] + b[i][e]).slope();
        dw[i][e] += ga * h[i][e];
        db[i][e] += ga;
        u[i][e] = ga * w[i][e];
        s[0] += u[i][e];
        s[1] += u[i][e] * h[i][e];
      }
    }
    if (!a.out) continue;
    rows_sum<WIDE>(s, p.team, lds);
    const float m = s[0] * inv, mh = s[1] * inv;
#pragma unroll
    for (int i = 0; i < N; ++i) {
#pragma unroll
      for (int e = 0; e < EV; ++e) u[i][e] = r * (u[i][e] - m - h[i][e] * mh);
      if (k.n[i] > 0) store_part<T, EV, PART>((T*)a.out + base + k.from[i], k.n[i], u[i]);
    }
  }
  if (part_w) rows_channels<EV, N>(dw, p, at, per, a.groups, part_w + (int64_t)blockIdx.x * C, lds);
  if (part_b) rows_channels<EV, N>(db, p, at, per, a.groups, part_b + (int64_t)blockIdx.x * C, lds);
}

// A chunk's parameters, of which the second derivative needs four: kept in registers where a lane has one chunk, else read
// from the caches for each sample.
template <typename T, int EV, bool PART>
struct Parameters {
  float w[EV], b[EV], vw[EV], vb[EV];
  __device__ __forceinline__ void load(const ictc::GroupNormCall& a, int c, int n) {
    parameter<T, EV, PART>((const T*)a.w, c, n, 1.f, w);
    parameter<T, EV, PART>((const T*)a.b, c, n, 0.f, b);
    parameter<T, EV, PART>((const T*)a.vw, c, n, 0.f, vw);
    parameter<T, EV, PART>((const T*)a.vb, c, n, 0.f, vb);
  }
};

template <typename T, int EV, int N, bool WIDE, bool PART, bool SILU, bool EIGHT>
__global__ __launch_bounds__(256) void gn_rows_bwd2_kernel(ictc::GroupNormCall a, RowsPlan p, int per,
                                                           float* __restrict__ part_w, float* __restrict__ part_b) {
  constexpr bool KEEP = N == 1;   // the elements' points too, over the sums
  __shared__ float lds[EV * 256 > 4 * kSums ? EV * 256 : 4 * kSums];
  const RowsAt at(p, a.groups);
  const int C = a.channels, S = (int)a.positions;
  const float inv = 1.f / ((float)per * (float)S);
  const RowsChunks<EV, N, PART> k(p, at, per, S, C);
  float dw[N][EV], db[N][EV];
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int e = 0; e < EV; ++e) dw[i][e] = db[i][e] = 0.f;
  Parameters<T, EV, PART> q;
  if (KEEP) q.load(a, k.c[0], k.n[0]);
  const int64_t size = (int64_t)S * C, blocks = (int64_t)S * code_blocks(C), end = a.samples * size;
  for (int64_t n = at.on ? at.sample : a.samples; n < a.samples; n += at.gap) {
    const int64_t base = n * size;
    Source<T, EV, EIGHT, PART> rx[N];
    Pack<T, EV> rg[N], rv[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      rx[i].load(a, base + k.from[i], n * blocks + k.block[i], k.border[i], k.n[i], end);
      rg[i] = load_part<T, EV, PART>((const T*)a.g, base + k.from[i], k.n[i], end);
      rv[i] = load_part<T, EV, PART>((const T*)a.v, base + k.from[i], k.n[i], end);
    }
    const float r = a.rstd[n * a.groups + at.group];
    const Mean mu = rows_mean<T, EV, N, WIDE, PART, EIGHT>(rx, k.n, a.mean[n * a.groups + at.group], r, inv, p.team, lds);
    float s[kSums] = {};
    Point kept[KEEP ? EV : 1];
    float x[EV], g[EV], v[EV];
    auto unpack = [&](int i) {
      rx[i].values(x);
      get<T, EV>(rg[i], g);
      get<T, EV>(rv[i], v);
      cut<PART>(g, k.n[i]);
      cut<PART>(v, k.n[i]);
      if (!KEEP) q.load(a, k.c[i], k.n[i]);
    };
#pragma unroll
    for (int i = 0; i < N; ++i) {
      unpack(i);
#pragma unroll
      for (int e = 0; e < EV; ++e) {
        const Point o = point<SILU>(((PART ? e : 0) < k.n[i] ? mu.off(x[e]) : 0.f) * r, g[e], q.w[e], q.b[e]);
        if (KEEP) kept[KEEP ? e : 0] = o;
        add_sums<SILU>(o, r, v[e], q.w[e], q.vw[e], q.vb[e], s);
      }
    }
    rows_sum<WIDE>(s, p.team, lds);
    const Seconds of(s, inv, r);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (!KEEP) unpack(i);
#pragma unroll
      for (int e = 0; e < EV; ++e) {
        const Point o = KEEP ? kept[KEEP ? e : 0]
                             : point<SILU>(((PART ? e : 0) < k.n[i] ? mu.off(x[e]) : 0.f) * r, g[e], q.w[e], q.b[e]);
        float pw, pb;
        of.element(o, r, v[e], q.w[e], q.vw[e], q.vb[e], x[e], v[e], pw, pb);
        dw[i][e] += (PART ? e : 0) < k.n[i] ? pw : 0.f;
        db[i][e] += (PART ? e : 0) < k.n[i] ? pb : 0.f;
      }
      if (k.n[i] <= 0) continue;
      if (a.out) store_part<T, EV, PART>((T*)a.out + base + k.from[i], k.n[i], x);
      if (a.out_g) store_part<T, EV, PART>((T*)a.out_g + base + k.from[i], k.n[i], v);
    }
  }
  if (part_w) rows_channels<EV, N>(dw, p, at, per, a.groups, part_w + (int64_t)blockIdx.x * C, lds);
  if (part_b) rows_channels<EV, N>(db, p, at, per, a.groups, part_b + (int64_t)blockIdx.x * C, lds);
}

}  // namespace
