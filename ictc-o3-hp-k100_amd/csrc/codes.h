// Activations in 8 bits, as every kernel that writes or reads them has them.  A block is 128 consecutive elements of a
// row, the last one what is left; with top the largest magnitude of a block
//   scale = max(top, 2^-100) c,  c = 1/127 in FP32;   code = x (1 / scale) to the nearest whole number, ties to even;
//   value = code scale, rounded to the type of x
// with every step rounded to FP32, so codes and values are the same wherever they are made.  (1/127 and not a power of
// two: all codes are in use whatever the block's size, which halves the largest error.)  A block that holds an infinity
// or NaN has the scale NaN, and so all of its values.
#pragma once
#include "dense.h"

namespace {

constexpr int kCodeBlock = 128;

// Magnitudes compare as whole numbers, infinity and NaN above all others.
__device__ __forceinline__ uint32_t magnitude(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7fffffffu; }

__device__ __forceinline__ float code_scale(uint32_t top) {
  if (top >= 0x7f800000u) return __builtin_nanf("");
  return fmaxf(__builtin_bit_cast(float, top), 0x1p-100f) * (float)(1.0 / 127.0);
}

__device__ __forceinline__ int code_of(float x, float inverse) {
  return (int)fminf(fmaxf(rintf(held(x * inverse)), -127.f), 127.f);
}

// N code values in FP32, code times scale.  A code is taken as code + 128, which one instruction makes a float of, and the
// product's surplus of 128 scales, a power of two of them, leaves by the same rounding: fma(code + 128, scale, -128 scale)
// is code times scale rounded once.  Where 128 scales are past FP32, code by code.
template <int N>
__device__ __forceinline__ void code_products(const uint32_t* raw, float scale, float (&v)[N]) {
  if (__builtin_amdgcn_ballot_w64(scale > 0x1p120f)) {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = held((float)(int8_t)(raw[e / 4] >> 8 * (e % 4)) * scale);
    return;
  }
  const float surplus = -128.f * scale;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const uint32_t biased = raw[e / 4] ^ 0x80808080u;
    v[e] = held(__builtin_fmaf((float)(biased >> 8 * (e % 4) & 255u), scale, surplus));
  }
}

typedef uint32_t u32_byte __attribute__((aligned(1)));
typedef u32x2 u32x2_byte __attribute__((aligned(1)));

// V codes (four or eight) as they lie in memory.
template <int V>
union Codes {
  int8_t e[V];
  uint32_t raw[V / 4];
  __device__ Codes() {}
};

// p[0 .. n), zero past n
template <int V>
__device__ __forceinline__ Codes<V> load_codes(const int8_t* __restrict__ p, int n) {
  Codes<V> c;
  if (n >= V) {
    if constexpr (V == 8)
      *reinterpret_cast<u32x2*>(c.raw) = *reinterpret_cast<const u32x2_byte*>(p);
    else
      c.raw[0] = *reinterpret_cast<const u32_byte*>(p);
  } else {
#pragma unroll
    for (int i = 0; i < V / 4; ++i) c.raw[i] = 0;
    if (n > 0) {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (i < n) c.e[i] = p[i];
    }
  }
  return c;
}

template <int V>
__device__ __forceinline__ void store_codes(int8_t* __restrict__ p, int n, const Codes<V>& c) {
  if (n >= V) {
    if constexpr (V == 8)
      *reinterpret_cast<u32x2_byte*>(p) = *reinterpret_cast<const u32x2*>(c.raw);
    else
      *reinterpret_cast<u32_byte*>(p) = c.raw[0];
  } else if (n > 0) {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < n) p[i] = c.e[i];
  }
}

// The largest of x over the aligned group of LANES lanes, in each of them.
template <int LANES>
__device__ __forceinline__ uint32_t lane_top(uint32_t x) {
  const auto step = [&](uint32_t y) { x = x > y ? x : y; };
  if (LANES >= 2) step(__builtin_bit_cast(uint32_t, dpp<0xB1>(__builtin_bit_cast(float, x))));
  if (LANES >= 4) step(__builtin_bit_cast(uint32_t, dpp<0x4E>(__builtin_bit_cast(float, x))));
  if (LANES >= 8) step(__builtin_bit_cast(uint32_t, dpp<0x141>(__builtin_bit_cast(float, x))));
  if (LANES >= 16) step(__builtin_bit_cast(uint32_t, dpp<0x140>(__builtin_bit_cast(float, x))));
  if (LANES >= 32) step((uint32_t)__shfl_xor((int)x, 16));
  return x;
}

// The same over `lanes` lanes, a power of two up to 32 that all agree on.
__device__ __forceinline__ uint32_t lanes_top(uint32_t x, int lanes) {
  switch (lanes) {
    case 1: return x;
    case 2: return lane_top<2>(x);
    case 4: return lane_top<4>(x);
    case 8: return lane_top<8>(x);
    case 16: return lane_top<16>(x);
    default: return lane_top<32>(x);
  }
}

}  // namespace
