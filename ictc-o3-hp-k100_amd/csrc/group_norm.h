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
//  * Rows: up to four chunks a lane of up to 64 lanes; of single positions, up to 32 elements a lane of a block.  This team
//    holds it in registers: one read.  It keeps its group, so the parameters stay in registers and their gradients are
//    added per lane.  (425,991 x 64 FP32 in eight groups: forward 48 us, gradients 60, 5.1 and 5.9 TB/s; one position of
//    4,096 bfloat16 channels by a block's team, 8,192 samples: forward 29 us and gradients 72, both by parts 204.)
//  * Tiles: a block takes some whole groups of a sample and reads them twice, for the sums and for the result, the second
//    time from the caches; one launch.  (32 x 256 positions x 128 FP32: forward 6 us, gradients 8, second derivative 13.)
//  * Parts: few large samples.  The sums by many blocks, a small kernel that adds their parts in order (few parts are added
//    by every block that needs them), and the result by as many blocks again.  (One sample of 131,072 x 256 bfloat16:
//    statistics 15 us, 4.5 TB/s; result 25, its x from the caches; gradients' sums 32 and result 37.)
// A chunk is the largest power of two of a group's channels up to 16 bytes, so each lies in one group and in one block of
// codes.  Groups that only small chunks divide are cut into 16-byte chunks, the last in part (rows), or their tile is,
// whatever the groups (group_norm_span.h).
//
// Means far from zero: statistics of tiles and parts are sums in FP64 of x less the group's first element (FP32; the sums
// of 16-bit values near one another and of their squares are exact) and of its squares, which costs little beside memory,
// loses nothing to what all of a group have in common and holds squares past FP32's range.  Of FP32 x a mean has two FP32
// values, itself and what its rounding left, and both are taken from x wherever h is made: x less the rounded mean is
// exact where they are near, so h is as good as x is.  (By the rounded mean alone every h of a group is off by half a
// unit of the mean: with a mean of 2^20 deviations 3 to 8 % of the results.)  The rows' backward passes find the second
// value anew, where it counts, for there is one for every few elements; tiles and parts read it.  Half a unit of the mean
// is at most 2^-13 of the largest deviation of 16-bit x, and 2^-16 of the error of x kept in 8 bits, so there it is left.
// Every sum has a fixed order.
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
  float* rest;          // of the means, their FP32 value taken off (null: nobody wants them, or not taken)
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

// A chunk of EV elements of a group.  Where a group's channels are no multiple of EV (PART) its last chunk has n of them: all
// EV are read, the next group's behind them, unless the tensor ends first, and those past n are dropped.
template <typename T, int EV, bool PART>
__device__ __forceinline__ Pack<T, EV> load_part(const T* __restrict__ p, int64_t from, int n, int64_t end) {
  if constexpr (!PART) return load_pack<T, EV>(p + (n > 0 ? from : 0), n > 0);
  if (n <= 0 || from + EV <= end) return load_pack<T, EV>(p + (n > 0 ? from : 0), n > 0);
  Pack<T, EV> c;
  c.raw = {};
#pragma unroll
  for (int e = 0; e < EV; ++e)
    if (e < n) c.e[e] = p[from + e];
  return c;
}

template <bool PART, int EV>
__device__ __forceinline__ void cut(float (&v)[EV], int n) {
  if constexpr (PART) {
#pragma unroll
    for (int e = 0; e < EV; ++e) v[e] = e < n ? v[e] : 0.f;
  }
}

template <typename T, int EV, bool PART>
__device__ __forceinline__ void store_part(T* __restrict__ p, int n, const float (&v)[EV]) {
  if (n >= EV) {
    store_pack<T, EV>(p, v);
  } else if constexpr (PART) {
    float r[4] = {v[0], EV > 1 ? v[1 % EV] : 0.f, EV > 2 ? v[2 % EV] : 0.f, EV > 3 ? v[3 % EV] : 0.f};
    if constexpr (EV == 8) {
      if (n & 4) {
        store_pack<T, 4>(p, r);
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = v[4 + e];
        p += 4;
      }
    }
    if (n & 2) {
      const float two[2] = {r[0], r[1]};
      store_pack<T, 2>(p, two);
      r[0] = r[2];
      p += 2;
    }
    if (n & 1) *p = (T)r[0];
  }
}

// p[0 .. n), `none` past n and where there is no p
template <typename T, int EV, bool PART = false>
__device__ __forceinline__ void parameter(const T* __restrict__ p, int64_t at, int n, float none, float (&v)[EV]) {
  if (p && n >= EV) {
    get<T, EV>(load_pack<T, EV>(p + at, true), v);
  } else {
#pragma unroll
    for (int e = 0; e < EV; ++e) v[e] = PART && p && e < n ? (float)p[at + e] : none;
  }
}

// A chunk of x as it lies in memory: elements, or codes and their scale.  from: its first element; n: how many it has;
// block: its code block, whose elements from `border` on are the next one's (PART).
template <typename T, int EV, bool EIGHT, bool PART = false>
struct Source {
  Pack<T, EV> raw;
  __device__ __forceinline__ void load(const ictc::GroupNormCall& a, int64_t from, int64_t, int, int n, int64_t end) {
    raw = load_part<T, EV, PART>((const T*)a.x, from, n, end);
  }
  __device__ __forceinline__ void values(float (&v)[EV]) const { get<T, EV>(raw, v); }
};

typedef uint16_t u16_byte __attribute__((aligned(1)));

template <typename T, int EV, bool PART>
struct Source<T, EV, true, PART> {
  union {
    int8_t e[8];
    uint16_t b2;
    uint32_t b4, word[2];
    u32x2 b8;
  } raw;
  float scale, next;
  int split;
  __device__ Source() {}
  __device__ __forceinline__ void load(const ictc::GroupNormCall& a, int64_t from, int64_t block, int border, int n,
                                       int64_t end) {
    raw.b8 = u32x2{0, 0};
    scale = next = 0.f;
    split = border;
    if (n <= 0) return;
    const int8_t* p = a.codes + from;
    if (PART && from + EV > end) {
#pragma unroll
      for (int e = 0; e < EV; ++e)
        if (e < n) raw.e[e] = p[e];
    } else {
      if constexpr (EV == 8) raw.b8 = *reinterpret_cast<const u32x2_byte*>(p);
      if constexpr (EV == 4) raw.b4 = *reinterpret_cast<const u32_byte*>(p);
      if constexpr (EV == 2) raw.b2 = *reinterpret_cast<const u16_byte*>(p);
      if constexpr (EV == 1) raw.e[0] = *p;
    }
    scale = a.scales[block];
    if (PART && border < n) next = a.scales[block + 1];
  }
  __device__ __forceinline__ void values(float (&v)[EV]) const {
    if constexpr (PART) {
#pragma unroll
      for (int e = 0; e < EV; ++e) v[e] = held((float)raw.e[e] * (e < split ? scale : next));
    } else {
      code_products<EV>(raw.word, scale, v);
    }
#pragma unroll
    for (int e = 0; e < EV; ++e) v[e] = (float)(T)v[e];
  }
};

__device__ __forceinline__ int code_blocks(int C) { return (C + kCodeBlock - 1) / kCodeBlock; }

// ---------------------------------------------------------------------------
// The formulas, element by element
// ---------------------------------------------------------------------------

// act(z), and its derivatives.  The sigmoid is the hardware's reciprocal of 1 + its power of two, each off by up to one
// unit of FP32 where a correctly rounded quotient is off by half; with the argument's rounding (1.5 |z| units) FP32
// results are off by 1.0 to 1.6 times what rounded steps give, inside the bounds of the row results.  (An exponential
// past FP32 makes the sigmoid zero, as it is to within 2^-128.)
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

// What an element of the normalised values h and the output gradient g gives: ga = g act'(z), act'(z) and g act''(z).
struct Point {
  float h, ga, slope, gb;
};
template <bool SILU>
__device__ __forceinline__ Point point(float h, float g, float w, float b) {
  const Act<SILU> a(h * w + b);
  const float slope = a.slope();
  return {h, g * slope, slope, g * a.bend()};
}

// Sums of a group that the gradients of the gradients need.
constexpr int kSums = 12;

template <bool SILU>
__device__ __forceinline__ void add_sums(const Point& p, float r, float v, float w, float vw, float vb, float (&s)[kSums]) {
  const float h = p.h, u = p.ga * w, t = p.ga * vw;
  s[0] += u;
  s[1] += u * h;
  s[2] += v;
  s[3] += v * h;
  s[4] += u * v;
  s[5] += t;
  s[6] += t * h;
  if (SILU) {
    const float wk = w * p.gb, part = wk * (w * r * v + h * vw + vb), wwk = w * wk, wwkh = wwk * h;
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
  __device__ __forceinline__ void element(const Point& p, float r, float vx, float w, float vw, float vb, float& dx,
                                          float& dg, float& dw, float& db) const {
    const float h = p.h, pv = r * (vx - v - h * vh), e = w * pv + h * vw + vb, zz = e * p.gb;
    const float t = p.ga * vw + zz * w - r * (vh * (p.ga * w) + uh * vx);
    dx = r * (t - tm - h * th) - r * r * q * h;
    dg = e * p.slope;
    dw = p.ga * pv + zz * h;
    db = zz;
  }
};

// A mean in two FP32 values, and what it leaves of x.
struct Mean {
  float hi, lo;
  __device__ __forceinline__ float off(float x) const { return (x - hi) - lo; }
};

// Of sample's group u, by one value or two.
template <bool TWO>
__device__ __forceinline__ Mean mean_of(const ictc::GroupNormCall& a, int64_t u) {
  return {a.mean[u], TWO && a.rest ? a.rest[u] : 0.f};
}

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

}  // namespace
