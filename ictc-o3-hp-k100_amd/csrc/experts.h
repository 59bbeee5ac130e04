// What the expert linears' kernels share: matrix instructions, runs of sorted rows, the order of blocks.
#pragma once
#include <algorithm>

#include "dense.h"
#include "split_bf16.h"

namespace {

typedef f16 f16x8 __attribute__((ext_vector_type(8)));

template <typename T>
__device__ __forceinline__ v4f mma(u32x4 a, u32x4 b, v4f c) {
  if constexpr (sizeof(T) == 2 && !__is_same(T, bf16))
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
}

// split8 (split_bf16.h) with each remainder by one instruction, the pair's dot product with (-1, 0) or (0, -1) added to
// the value: it is exact as the subtraction is, subnormal numbers included, and where one value of a pair is beyond
// bfloat16's range the other's remainder is NaN too.  The parts end at bfloat16's last bit, 2^-133: a value under 2^-110
// is held to 2^-134, not to FP32's precision.
__device__ __forceinline__ Split split8_pairs(const float* v) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  uint32_t first = 0x0000bf80u, second = 0xbf800000u;
  asm("" : "+s"(first));   // (registers: as an inline constant of a pair -1 would stand for another)
  asm("" : "+s"(second));
  const bf16x2 m0 = __builtin_bit_cast(bf16x2, first), m1 = __builtin_bit_cast(bf16x2, second);
  Split s;
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const bf16x2 h = {(__bf16)v[e], (__bf16)v[e + 1]};
    const float r0 = __builtin_amdgcn_fdot2_f32_bf16(h, m0, v[e], false);
    const float r1 = __builtin_amdgcn_fdot2_f32_bf16(h, m1, v[e + 1], false);
    const bf16x2 m = {(__bf16)r0, (__bf16)r1};
    const bf16x2 l = {(__bf16)__builtin_amdgcn_fdot2_f32_bf16(m, m0, r0, false),
                      (__bf16)__builtin_amdgcn_fdot2_f32_bf16(m, m1, r1, false)};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      s.hi[e + i] = h[i];
      s.mid[e + i] = m[i];
      s.lo[e + i] = l[i];
    }
  }
  return s;
}

// The product of one 16 x 16 block over 32 reduction indices from the operands' parts.
template <typename T, int NP>
__device__ __forceinline__ v4f product(const u32x4 (&a)[NP], const u32x4 (&b)[NP], v4f c) {
  if constexpr (NP == 3) {
    c = mma<T>(a[2], b[0], c);
    c = mma<T>(a[0], b[2], c);
    c = mma<T>(a[1], b[1], c);
    c = mma<T>(a[1], b[0], c);
    c = mma<T>(a[0], b[1], c);
  }
  return mma<T>(a[0], b[0], c);
}

// Run `t` of groups 0 .. G - 1 cut into runs of `rows` sorted rows: its group, first sorted row and row count.  False
// past the last run.  The same values in every lane of the wave, which has to be whole.
struct Run {
  int group, start, count;
};

// Sum over the wave's lanes up to each lane.
__device__ __forceinline__ int scan_lanes(int x) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int up = __shfl_up(x, d);
    if (lane >= d) x += up;
  }
  return x;
}

// `unit` of groups 0 .. G - 1 cut into units of `rows` sorted rows: its group, the group's first unit, sorted rows
// and units.  False past the last unit, and then `first` is their number.
struct Place {
  int group, first, lo, count, units;
};

__device__ __forceinline__ bool find_unit(const int* __restrict__ off, int G, int rows, int unit, Place& p) {
  const int lane = threadIdx.x & 63;
  int base = 0;
  for (int s0 = 0; s0 < G; s0 += 64) {
    const int s = s0 + lane;
    int lo = 0, n = 0;
    if (s < G) {
      lo = off[s];
      n = off[s + 1] - lo;
    }
    const int units = (n + rows - 1) / rows, sum = scan_lanes(units);
    const int total = __builtin_amdgcn_readlane(sum, 63);
    if (unit < base + total) {
      const int f = __builtin_ctzll(__ballot(base + sum > unit));
      p.group = s0 + f;
      p.units = __builtin_amdgcn_readlane(units, f);
      p.first = base + __builtin_amdgcn_readlane(sum, f) - p.units;
      p.lo = __builtin_amdgcn_readlane(lo, f);
      p.count = __builtin_amdgcn_readlane(n, f);
      return true;
    }
    base += total;
  }
  p.first = base;
  return false;
}

__device__ __forceinline__ bool find_run(const int* __restrict__ off, int G, int rows, int t, Run& r) {
  Place p;
  if (!find_unit(off, G, rows, t, p)) return false;
  const int at = (t - p.first) * rows;
  r.group = p.group;
  r.start = p.lo + at;
  r.count = min(rows, p.count - at);
  return true;
}

// The weights' gradient: the sorted rows of all experts, in steps of `rows` of one expert, are cut into `ranges` of
// equal length; a block takes one tile of the output over one range and meets the experts in it in turn.  An expert
// that lies within a range is done there; one that continues into others leaves FP32 partial sums, in slot 0 of each
// range, or in slot 1 of the range that it begins in behind another.  Every range costs the same whatever the
// experts' sizes, and there are as many partial sums as ranges and experts that cross them, not more.
struct Ranges {
  int steps, per;   // of all experts; of a range
};

__device__ __forceinline__ Ranges find_ranges(const int* __restrict__ off, int experts, int rows, int ranges) {
  Place p;
  find_unit(off, experts, rows, INT32_MAX, p);
  return {p.first, max(1, (p.first + ranges - 1) / ranges)};
}

struct Segment {
  int expert, start, count;   // sorted rows
  int steps;                  // of this segment
  bool whole;                 // the expert has no other
  int slot;
};

// The segment that begins at step `u` of the range q = [q per, q per + per).
__device__ __forceinline__ bool find_segment(const int* __restrict__ off, int experts, int rows, const Ranges& r,
                                             int q, int u, Segment& s) {
  Place p;
  const int end = min(r.steps, (q + 1) * r.per);
  if (u >= end || !find_unit(off, experts, rows, u, p)) return false;
  const int last = min(end, p.first + p.units);
  s.expert = p.group;
  s.steps = last - u;
  s.start = p.lo + (u - p.first) * rows;
  s.count = min(s.steps * rows, p.count - (u - p.first) * rows);
  s.whole = u == p.first && last == p.first + p.units;
  s.slot = u > q * r.per;
  return true;
}

// Block `b` of `blocks` in an order that gives each of the eight dies (blocks go to them in turn) a contiguous part.
__device__ __forceinline__ int die_order(int b, int blocks) {
  const int per = blocks / 8, rest = blocks % 8, die = b & 7;
  return die * per + min(die, rest) + (b >> 3);
}

// Zeros in the tile at (m0, k0) of gW [M, K] and, of the first column tile, of gb [M].
template <typename T, int TILE, int THREADS>
__device__ __forceinline__ void zero_tile(T* __restrict__ gW, T* __restrict__ gb, int M, int K, int m0, int k0) {
  constexpr int V = kChunk<T>, CH = TILE / V;
  const float zero[V] = {};
  for (int i = threadIdx.x; i < TILE * CH; i += THREADS) {
    const int m = m0 + i / CH, k = k0 + i % CH * V;
    if (m < M) store_chunk(gW + (int64_t)m * K + k, K - k, zero);
  }
  if (gb && k0 == 0)
    for (int i = threadIdx.x; i < TILE; i += THREADS)
      if (m0 + i < M) gb[m0 + i] = (T)0.f;
}

}  // namespace

// The kernels of experts_direct.hip, and whether they take these: rows of 16 bytes or more.
bool experts_direct_rows_fit(int dtype, int K, int N, bool transpose);
void experts_direct_rows(int dtype, const void* x, int64_t ldx, int64_t rows, int K, const void* W, const void* bias,
                         int N, int experts, const int* perm, const int* off, bool transpose, void* out,
                         hipStream_t st);

// Most runs of up to `tile` rows of one expert (or of none).
inline int64_t most_runs(int64_t rows, int experts, int tile) {
  return rows / tile + std::min<int64_t>(rows, experts + 1);
}

// About as many tiles of 128 x 128 as the rows' product has.
inline int64_t experts_tiles(int64_t rows, int N, int experts) {
  return (rows / 128 + std::min<int64_t>(rows, experts)) * ((N + 127) / 128);
}

// How the weights' gradient is cut: `tile` columns a side, `rows` of a step, `ranges`; `fill` blocks of a tile share the
// zeros of experts without rows; `sums`: an expert may cross ranges; `direct`: by the kernel of experts_direct.hip.
struct OuterPlan {
  bool direct, sums;
  int tile, rows, ranges, fill;
};
bool experts_direct_outer_fits(int dtype, int M, int K);
void experts_direct_outer(int dtype, const OuterPlan& plan, const void* gy, int64_t ldg, int M, const void* x,
                          int64_t ldx, int K, int experts, const int* perm, const int* off, void* gW, void* gb,
                          float* part, hipStream_t st);
