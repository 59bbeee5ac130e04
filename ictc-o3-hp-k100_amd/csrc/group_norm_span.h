// Tiles of groups whose channels are no whole number of 16-byte chunks: a tile is some whole groups side by side, cut into
// whole chunks whatever the groups (the last one in part), and a chunk's elements have their groups' statistics each.  Sums
// are by channel, and by group once a tile is through. (group_norm_launch.h says where this is
// the faster.)
#pragma once
#include "group_norm_tiles.h"

namespace {

constexpr int kSpanGroups = 64;

template <int EV>
struct SpanAt {
  int lane, row, c, n, first_group, groups;   // n: the chunk's elements
  bool on;
  int64_t sample, begin, end;
  int split, slot, border;
  int local[EV];   // each element's group in the tile
  __device__ __forceinline__ SpanAt(const TilePlan& p, int per, int G, int64_t S) {
    lane = threadIdx.x % p.lanes;
    row = threadIdx.x / p.lanes;
    const int b = die_order(blockIdx.x, gridDim.x), tile = b % p.tiles, rest = b / p.tiles;
    split = rest % p.splits;
    sample = slot = rest / p.splits;
    first_group = tile * p.groups;
    groups = min(p.groups, G - first_group);
    c = first_group * per + lane * EV;
    n = row < p.rows ? min(EV, groups * per - lane * EV) : 0;
    on = n > 0;
    border = kCodeBlock - c % kCodeBlock;
#pragma unroll
    for (int e = 0; e < EV; ++e) local[e] = on && e < n ? (lane * EV + e) / per : 0;
    begin = split * p.per_split;
    end = min(S, begin + p.per_split);
  }
};

// Sums by group, [groups][K], of those by channel in lds [K EV][256] (row 0): eight lanes a group.
template <int K, int EV, typename V>
__device__ __forceinline__ void span_groups(const V* lds, int per, int groups, V (*sums)[K]) {
  const int lane = threadIdx.x & 7;
  for (int g0 = 0; g0 < groups; g0 += kThreads / 8) {
    const int g = g0 + (threadIdx.x >> 3);
    V s[K];
#pragma unroll
    for (int k = 0; k < K; ++k) s[k] = (V)0;
    if (g < groups) {
      for (int j = lane; j < per; j += 8) {
        const int c = g * per + j;
#pragma unroll
        for (int k = 0; k < K; ++k) s[k] += lds[(k * EV + c % EV) * kThreads + c / EV];
      }
    }
    sum_low(s, 8);
    if (g < groups && lane == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) sums[g][k] = s[k];
    }
  }
  __syncthreads();
}

// The same of parts [groups][splits][K] in memory.
template <int K, typename V>
__device__ __forceinline__ void span_parts(const V* __restrict__ part, int splits, int groups, V (*sums)[K]) {
  const int lane = threadIdx.x & 7;
  __syncthreads();
  for (int g0 = 0; g0 < groups; g0 += kThreads / 8) {
    const int g = g0 + (threadIdx.x >> 3);
    V s[K];
#pragma unroll
    for (int k = 0; k < K; ++k) s[k] = (V)0;
    if (g < groups) {
#pragma unroll 4
      for (int j = lane; j < splits; j += 8) {
#pragma unroll
        for (int k = 0; k < K; ++k) s[k] += part[((int64_t)g * splits + j) * K + k];
      }
    }
    sum_low(s, 8);
    if (g < groups && lane == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) sums[g][k] = s[k];
    }
  }
  __syncthreads();
}

// Sums by group of the tile's x less the group's first element and of their squares.
template <typename T, int EV>
__device__ __forceinline__ void span_statistics(const ictc::GroupNormCall& a, const TilePlan& p, const SpanAt<EV>& at, int per,
                                                int64_t total, double* lds, double (*sums)[2]) {
  double s[2 * EV] = {};
  float zero[EV];
#pragma unroll
  for (int e = 0; e < EV; ++e) zero[e] = at.on ? first_of<T>(a, at.sample, at.first_group + at.local[e], per) : 0.f;
  constexpr int U = 2;
  walk<U>(p, at, a.positions, a.channels, [&](int64_t from, int64_t step, int64_t, int64_t, int count) {
    Pack<T, EV> raw[U];
#pragma unroll
    for (int i = 0; i < U; ++i) raw[i] = load_part<T, EV, true>((const T*)a.x, from + i * step, i < count ? at.n : 0, total);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (i >= count) break;   // (past n: sums that nobody reads)
      float v[EV];
      get<T, EV>(raw[i], v);
#pragma unroll
      for (int e = 0; e < EV; ++e) {
        const double d = (double)v[e] - (double)zero[e];
        s[e] += d;
        s[EV + e] += d * d;
      }
    }
  });
  sum_rows(s, p, at, lds);
  span_groups<2, EV>(lds, per, at.groups, sums);
}

template <int EV>
struct SpanMoments {
  Mean mean[EV];
  float rstd[EV];
  __device__ __forceinline__ void load(const Moments* m, const SpanAt<EV>& at) {   // the tile's groups'
#pragma unroll
    for (int e = 0; e < EV; ++e) {
      mean[e] = m[at.local[e]].mean;
      rstd[e] = m[at.local[e]].rstd;
    }
  }
  template <bool TWO>
  __device__ __forceinline__ void load(const ictc::GroupNormCall& a, int64_t u, const SpanAt<EV>& at) {   // u: its first group
#pragma unroll
    for (int e = 0; e < EV; ++e) {
      mean[e] = mean_of<TWO>(a, u + at.local[e]);
      rstd[e] = a.rstd[u + at.local[e]];
    }
  }
};

template <typename T, int EV, bool SILU>
__device__ __forceinline__ void span_result(const ictc::GroupNormCall& a, const TilePlan& p, const SpanAt<EV>& at,
                                            const SpanMoments<EV>& m, int64_t total) {
  float w[EV], b[EV];
  parameter<T, EV, true>((const T*)a.w, at.c, at.n, 1.f, w);
  parameter<T, EV, true>((const T*)a.b, at.c, at.n, 0.f, b);
  constexpr int U = 2;
  walk<U>(p, at, a.positions, a.channels, [&](int64_t from, int64_t step, int64_t, int64_t, int count) {
    Pack<T, EV> raw[U];
#pragma unroll
    for (int i = 0; i < U; ++i) raw[i] = load_part<T, EV, true>((const T*)a.x, from + i * step, i < count ? at.n : 0, total);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (i >= count) break;
      float v[EV];
      get<T, EV>(raw[i], v);
#pragma unroll
      for (int e = 0; e < EV; ++e) v[e] = Act<SILU>(m.mean[e].off(v[e]) * m.rstd[e] * w[e] + b[e]).value();
      store_part<T, EV, true>((T*)a.out + from + i * step, at.n, v);
    }
  });
}

// part: null, all in one; else the statistics' parts [samples][groups][splits][2] alone
template <typename T, int EV, bool SILU>
__global__ __launch_bounds__(kThreads) void gn_span_fwd_kernel(ictc::GroupNormCall a, TilePlan p, int per,
                                                               double* __restrict__ part) {
  __shared__ double lds[2 * EV * kThreads];
  __shared__ double sums[kSpanGroups][2];
  __shared__ Moments groups[kSpanGroups];
  SpanAt<EV> at(p, per, a.groups, a.positions);
  const int64_t total = a.samples * a.positions * a.channels;
  for (; at.sample < a.samples; at.sample += p.slots) {
    const int64_t u = at.sample * a.groups + at.first_group;
    const int g = threadIdx.x;
    span_statistics<T, EV>(a, p, at, per, total, lds, sums);
    if (part) {
      if (g < at.groups) {
        part[((u + g) * p.splits + at.split) * 2] = sums[g][0];
        part[((u + g) * p.splits + at.split) * 2 + 1] = sums[g][1];
      }
      continue;   // (the next sample's sums are behind a barrier)
    }
    if (g < at.groups) {
      const float zero = first_of<T>(a, at.sample, at.first_group + g, per);
      groups[g] = moments<T>(zero, sums[g][0], sums[g][1], (double)per * (double)a.positions, a.eps);
      if (a.mean) keep(a, u + g, groups[g]);
    }
    __syncthreads();
    SpanMoments<EV> m;
    m.load(groups, at);
    span_result<T, EV, SILU>(a, p, at, m, total);
  }
}

// part: the statistics' parts, which the blocks add (those of split 0 write mean and rstd, if they are wanted); or null
template <typename T, int EV, bool SILU>
__global__ __launch_bounds__(kThreads) void gn_span_part_fwd_kernel(ictc::GroupNormCall a, TilePlan p, int per,
                                                                    const double* __restrict__ part) {
  __shared__ double sums[kSpanGroups][2];
  __shared__ Moments groups[kSpanGroups];
  SpanAt<EV> at(p, per, a.groups, a.positions);
  const int64_t total = a.samples * a.positions * a.channels;
  for (; at.sample < a.samples; at.sample += p.slots) {
    const int64_t u = at.sample * a.groups + at.first_group;
    SpanMoments<EV> m;
    if (part) {
      span_parts(part + u * p.splits * 2, p.splits, at.groups, sums);
      const int g = threadIdx.x;
      if (g < at.groups) {
        const float zero = first_of<T>(a, at.sample, at.first_group + g, per);
        groups[g] = moments<T>(zero, sums[g][0], sums[g][1], (double)per * (double)a.positions, a.eps);
        if (a.mean && at.split == 0) keep(a, u + g, groups[g]);
      }
      __syncthreads();
      m.load(groups, at);
    } else {
      m.template load<sizeof(T) == 4>(a, u, at);
    }
    span_result<T, EV, SILU>(a, p, at, m, total);
  }
}

template <typename T, int EV, bool SILU, bool EIGHT>
__device__ __forceinline__ void span_gradient(const ictc::GroupNormCall& a, const TilePlan& p, const SpanAt<EV>& at,
                                              const SpanMoments<EV>& m, const float (&w)[EV], const float (&b)[EV],
                                              const float (*sums)[2], float inv, int64_t total) {
  float u[EV], uh[EV];
#pragma unroll
  for (int e = 0; e < EV; ++e) {
    u[e] = sums[at.local[e]][0] * inv;
    uh[e] = sums[at.local[e]][1] * inv;
  }
  constexpr int U = 2;
  walk<U>(p, at, a.positions, a.channels, [&](int64_t from, int64_t step, int64_t block, int64_t bstep, int count) {
    Source<T, EV, EIGHT, true> rx[U];
    Pack<T, EV> rg[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      rx[i].load(a, from + i * step, block + i * bstep, at.border, i < count ? at.n : 0, total);
      rg[i] = load_part<T, EV, true>((const T*)a.g, from + i * step, i < count ? at.n : 0, total);
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (i >= count) break;
      float x[EV], g[EV];
      rx[i].values(x);
      get<T, EV>(rg[i], g);
#pragma unroll
      for (int e = 0; e < EV; ++e) {
        const float h = m.mean[e].off(x[e]) * m.rstd[e], ga = g[e] * Act<SILU>(h * w[e] + b[e]).slope();
        x[e] = m.rstd[e] * (ga * w[e] - u[e] - h * uh[e]);
      }
      store_part<T, EV, true>((T*)a.out + from + i * step, at.n, x);
    }
  });
}

// FUSED: the row gradient follows at once; else sums of u and u h to part [samples][groups][splits][2].
template <typename T, int EV, bool SILU, bool EIGHT, bool FUSED>
__global__ __launch_bounds__(kThreads) void gn_span_bwd_kernel(ictc::GroupNormCall a, TilePlan p, int per,
                                                               float* __restrict__ part, float* __restrict__ part_w,
                                                               float* __restrict__ part_b) {
  __shared__ float lds[2 * EV * kThreads];
  __shared__ float sums[kSpanGroups][2];
  SpanAt<EV> at(p, per, a.groups, a.positions);
  const int64_t total = a.samples * a.positions * a.channels;
  const float inv = 1.f / ((float)per * (float)a.positions);
  float w[EV], b[EV], kept[2 * EV] = {};   // kept: row 0's sums by channel over the samples
  parameter<T, EV, true>((const T*)a.w, at.c, at.n, 1.f, w);
  parameter<T, EV, true>((const T*)a.b, at.c, at.n, 0.f, b);
  for (; at.sample < a.samples; at.sample += p.slots) {
    const int64_t group = at.sample * a.groups + at.first_group;
    SpanMoments<EV> m;
    m.template load<sizeof(T) == 4 && !EIGHT>(a, group, at);
    float s[2 * EV] = {};
    constexpr int U = 2;
    walk<U>(p, at, a.positions, a.channels, [&](int64_t from, int64_t step, int64_t block, int64_t bstep, int count) {
      Source<T, EV, EIGHT, true> rx[U];
      Pack<T, EV> rg[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        // (x of a position that there is: zero less a large mean may be infinite)
        const int64_t f = i < count ? from + i * step : from;
        rx[i].load(a, f, i < count ? block + i * bstep : block, at.border, at.n, total);
        rg[i] = load_part<T, EV, true>((const T*)a.g, f, i < count ? at.n : 0, total);
      }
#pragma unroll
      for (int i = 0; i < U; ++i) {
        float x[EV], g[EV];
        rx[i].values(x);
        get<T, EV>(rg[i], g);
        cut<true>(x, at.n);
        cut<true>(g, at.n);
#pragma unroll
        for (int e = 0; e < EV; ++e) {
          const float h = m.mean[e].off(x[e]) * m.rstd[e], ga = g[e] * Act<SILU>(h * w[e] + b[e]).slope();
          s[e] += ga;
          s[EV + e] += ga * h;
        }
      }
    });
    sum_rows(s, p, at, lds);
    if (at.on && at.row == 0) {
#pragma unroll
      for (int k = 0; k < 2 * EV; ++k) {
        float* q = lds + k * kThreads + threadIdx.x;
        kept[k] += *q;
        *q *= w[k % EV];
      }
    }
    if (!a.out) continue;
    __syncthreads();
    span_groups<2, EV>(lds, per, at.groups, sums);
    if constexpr (FUSED) {
      span_gradient<T, EV, SILU, EIGHT>(a, p, at, m, w, b, sums, inv, total);
    } else if ((int)threadIdx.x < at.groups) {
      const int g = threadIdx.x;
      part[((group + g) * p.splits + at.split) * 2] = sums[g][0];
      part[((group + g) * p.splits + at.split) * 2 + 1] = sums[g][1];
    }
  }
  if (!at.on || at.row != 0) return;
  const int64_t to = ((int64_t)at.slot * p.splits + at.split) * a.channels + at.c;
#pragma unroll
  for (int e = 0; e < EV; ++e) {
    if (e < at.n && part_b) part_b[to + e] = kept[e];
    if (e < at.n && part_w) part_w[to + e] = kept[EV + e];
  }
}

// own: sums are the parts', and the blocks add them themselves
template <typename T, int EV, bool SILU, bool EIGHT>
__global__ __launch_bounds__(kThreads) void gn_span_part_bwd_kernel(ictc::GroupNormCall a, TilePlan p, int per,
                                                                    const float* __restrict__ sums_, bool own) {
  __shared__ float sums[kSpanGroups][2];
  SpanAt<EV> at(p, per, a.groups, a.positions);
  const int64_t total = a.samples * a.positions * a.channels;
  float w[EV], b[EV];
  parameter<T, EV, true>((const T*)a.w, at.c, at.n, 1.f, w);
  parameter<T, EV, true>((const T*)a.b, at.c, at.n, 0.f, b);
  for (; at.sample < a.samples; at.sample += p.slots) {
    const int64_t group = at.sample * a.groups + at.first_group;
    if (own) {
      span_parts(sums_ + group * p.splits * 2, p.splits, at.groups, sums);
    } else {
      __syncthreads();
      if ((int)threadIdx.x < at.groups) {
        sums[threadIdx.x][0] = sums_[(group + threadIdx.x) * 2];
        sums[threadIdx.x][1] = sums_[(group + threadIdx.x) * 2 + 1];
      }
      __syncthreads();
    }
    SpanMoments<EV> m;
    m.template load<sizeof(T) == 4 && !EIGHT>(a, group, at);
    span_gradient<T, EV, SILU, EIGHT>(a, p, at, m, w, b, sums, 1.f / ((float)per * (float)a.positions), total);
  }
}

}  // namespace
