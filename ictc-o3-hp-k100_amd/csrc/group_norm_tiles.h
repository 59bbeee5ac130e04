// The group norm of larger samples: by blocks that take whole groups of them, or by parts (group_norm.h has the formulas).
#pragma once
#include "group_norm.h"

namespace {

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
template <typename V, int K, typename At>
__device__ __forceinline__ void sum_rows(V (&s)[K], const TilePlan& p, const At& at, V* lds) {
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
template <int U, typename At, typename F>
__device__ __forceinline__ void walk(const TilePlan& p, const At& at, int64_t S, int C, F&& f) {
  if (!at.on) return;
  const int64_t step = (int64_t)p.rows * C, bstep = (int64_t)p.rows * code_blocks(C);
  const int64_t row = at.sample * S + at.begin + at.row;
  int64_t from = row * C + at.c, block = row * code_blocks(C) + at.c / kCodeBlock;
  for (int64_t left = at.end - at.begin - at.row; left > 0; left -= U * p.rows, from += U * step, block += U * bstep)
    f(from, step, block, bstep, (int)min<int64_t>(U, (left + p.rows - 1) / p.rows));
}

// What the statistics of sample n's group are counted from: its first element, zero of 16 bits.
template <typename T>
__device__ __forceinline__ float first_of(const ictc::GroupNormCall& a, int64_t n, int group, int per) {
  if constexpr (sizeof(T) == 2) return 0.f;
  return (float)((const T*)a.x)[n * a.positions * a.channels + (int64_t)group * per];
}

// Sums over the tile's group of x less its first element and of their squares; returns that.
template <typename T, int EV>
__device__ __forceinline__ float tile_statistics(const ictc::GroupNormCall& a, const TilePlan& p, const TileAt& at, int per,
                                                 double (&s)[2], double* lds) {
  constexpr int U = kRowsAtOnce<EV>;
  s[0] = s[1] = 0.0;
  const float zero = at.on ? first_of<T>(a, at.sample, at.group, per) : 0.f;
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
      for (int e = 0; e < EV; ++e) {
        const double d = (double)v[e] - (double)zero;
        s[0] += d;
        s[1] += d * d;
      }
    }
  });
  sum_all(s, p, at, lds);
  return zero;
}

struct Moments {
  Mean mean;
  float rstd;
};

// Of sums of values less `zero`.
template <typename T>
__device__ __forceinline__ Moments moments(float zero, double sum, double squares, double count, float eps) {
  const double off = sum / count, var = squares / count - off * off, mean = zero + off;
  return {{(float)mean, sizeof(T) == 4 ? (float)(mean - (float)mean) : 0.f}, deviation(var < 0.0 ? 0.0 : var, eps)};
}

template <typename T, bool EIGHT>
__device__ __forceinline__ Moments moments_of(const ictc::GroupNormCall& a, int64_t u) {
  return {mean_of<sizeof(T) == 4 && !EIGHT>(a, u), a.rstd[u]};
}

// To where they are wanted.
__device__ __forceinline__ void keep(const ictc::GroupNormCall& a, int64_t u, const Moments& m) {
  a.mean[u] = m.mean.hi;
  if (a.rest) a.rest[u] = m.mean.lo;
  a.rstd[u] = m.rstd;
}

template <typename T, int EV, bool SILU>
__device__ __forceinline__ void tile_result(const ictc::GroupNormCall& a, const TilePlan& p, const TileAt& at,
                                            const Moments& m) {
  constexpr int U = kRowsAtOnce<EV>;
  float w[EV], b[EV];
  parameter<T, EV>((const T*)a.w, at.c, at.on ? EV : 0, 1.f, w);
  parameter<T, EV>((const T*)a.b, at.c, at.on ? EV : 0, 0.f, b);
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
      for (int e = 0; e < EV; ++e) v[e] = Act<SILU>(m.mean.off(v[e]) * m.rstd * w[e] + b[e]).value();
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
    const float zero = tile_statistics<T, EV>(a, p, at, per, s, lds);
    const Moments m = moments<T>(zero, s[0], s[1], (double)per * (double)a.positions, a.eps);
    if (a.mean && at.first) keep(a, at.sample * a.groups + at.group, m);
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
    tile_statistics<T, EV>(a, p, at, per, s, lds);
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

// A wave a sample's group; to a's mean, rest and rstd.
template <typename T>
__global__ __launch_bounds__(256) void gn_part_moments_kernel(ictc::GroupNormCall a, const double* __restrict__ part,
                                                              int64_t units, int parts, int per) {
  for (int64_t u = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); u < units; u += (int64_t)gridDim.x * 4) {
    double s[2];
    wave_parts<2>(part + u * parts * 2, parts, s);
    if ((threadIdx.x & 63) == 0) {
      const int64_t n = u / a.groups;
      const float zero = first_of<T>(a, n, (int)(u - n * a.groups), per);
      keep(a, u, moments<T>(zero, s[0], s[1], (double)per * (double)a.positions, a.eps));
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
                                                               const double* __restrict__ part) {
  __shared__ double lds[kOwnGroups][2];
  TileAt at(p, EV, per, a.groups, a.positions);
  for (; at.sample < a.samples; at.sample += p.slots) {
    Moments m = {{0.f, 0.f}, 0.f};
    const int64_t u = at.sample * a.groups + at.group;
    if (part) {
      double s[2];
      tile_parts(part, at.sample, a.groups, p, at, s, lds);
      const float zero = at.on ? first_of<T>(a, at.sample, at.group, per) : 0.f;
      m = moments<T>(zero, s[0], s[1], (double)per * (double)a.positions, a.eps);
      if (a.mean && at.first && at.split == 0) keep(a, u, m);
    } else if (at.on) {
      m = moments_of<T, false>(a, u);
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
      // (x of a position that there is: zero less a large mean may be infinite)
      const int64_t f = i < count ? from + i * step : from;
      rx[i].load(a, f, i < count ? block + i * bstep : block, EV, EV, 0);
      rg[i] = load_pack<T, EV>((const T*)a.g + f, i < count);
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      float x[EV], g[EV];
      rx[i].values(x);
      get<T, EV>(rg[i], g);
#pragma unroll
      for (int e = 0; e < EV; ++e) {
        const float h = m.mean.off(x[e]) * m.rstd, ga = g[e] * Act<SILU>(h * w[e] + b[e]).slope();
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
      rx[i].load(a, from + i * step, block + i * bstep, EV, i < count ? EV : 0, 0);
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
        const float h = m.mean.off(x[e]) * m.rstd, ga = g[e] * Act<SILU>(h * w[e] + b[e]).slope();
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
  parameter<T, EV>((const T*)a.w, at.c, at.on ? EV : 0, 1.f, w);
  parameter<T, EV>((const T*)a.b, at.c, at.on ? EV : 0, 0.f, b);
  const float inv = 1.f / ((float)per * (float)a.positions);
  ChannelSums<EV> channels;
  for (; at.sample < a.samples; at.sample += p.slots) {
    const int64_t u = at.on ? at.sample * a.groups + at.group : 0;
    const Moments m = moments_of<T, EIGHT>(a, u);
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
  parameter<T, EV>((const T*)a.w, at.c, at.on ? EV : 0, 1.f, w);
  parameter<T, EV>((const T*)a.b, at.c, at.on ? EV : 0, 0.f, b);
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
    tile_gradient<T, EV, SILU, EIGHT>(a, p, at, moments_of<T, EIGHT>(a, u), w, b, s[0] * inv, s[1] * inv);
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
      rx[i].load(a, f, i < count ? block + i * bstep : block, EV, EV, 0);
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
        add_sums<SILU>(point<SILU>(m.mean.off(x[e]) * m.rstd, g[e], w[e], b[e]), m.rstd, v[e], w[e], vw[e], vb[e], s);
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
      rx[i].load(a, f, block + i * bstep, EV, i < count ? EV : 0, 0);
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
        of.element(point<SILU>(m.mean.off(x[e]) * m.rstd, g[e], w[e], b[e]), m.rstd, v[e], w[e], vw[e], vb[e], x[e], v[e], pw,
                   pb);
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
  parameter<T, EV>((const T*)a.w, at.c, at.on ? EV : 0, 1.f, w);
  parameter<T, EV>((const T*)a.b, at.c, at.on ? EV : 0, 0.f, b);
  parameter<T, EV>((const T*)a.vw, at.c, at.on ? EV : 0, 0.f, vw);
  parameter<T, EV>((const T*)a.vb, at.c, at.on ? EV : 0, 0.f, vb);
  const float inv = 1.f / ((float)per * (float)a.positions);
  ChannelSums<EV> channels;
  for (; at.sample < a.samples; at.sample += p.slots) {
    const int64_t u = at.on ? at.sample * a.groups + at.group : 0;
    const Moments m = moments_of<T, EIGHT>(a, u);
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

}  // namespace
