// Element types, 16-byte chunks and wave sums shared by the dense-layer kernels (layer norm, AdamW, expert linears).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/ictc_mi355x.h"

namespace ictc {
int set_error(int code, const char* msg);
}

namespace {

typedef __bf16 bf16;
typedef _Float16 f16;
typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
// Rows of any pitch: a 16- or 8-byte access that promises the element's alignment only (global memory takes it in
// one instruction either way).
typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef u32x2 u32x2_any __attribute__((aligned(2)));

template <typename T>
constexpr int kChunk = 16 / (int)sizeof(T);   // elements of one 16-byte chunk

template <typename T>
union Chunk {
  u32x4 raw;
  T e[kChunk<T>];
  __device__ Chunk() {}
};

// p[0 .. n), zero past n (n may be zero or negative; lanes that all are skip the element loop).
template <typename T>
__device__ __forceinline__ u32x4 load_raw(const T* __restrict__ p, int n) {
  constexpr int V = kChunk<T>;
  if (n >= V) return *reinterpret_cast<const u32x4_any*>(p);
  Chunk<T> c;
  c.raw = u32x4{0, 0, 0, 0};
  if (n > 0) {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < n) c.e[i] = p[i];
  }
  return c.raw;
}

template <typename T>
__device__ __forceinline__ void widen(u32x4 raw, float* v) {
  Chunk<T> c;
  c.raw = raw;
#pragma unroll
  for (int i = 0; i < kChunk<T>; ++i) v[i] = (float)c.e[i];
}

template <typename T>
__device__ __forceinline__ void load_chunk(const T* __restrict__ p, int n, float* v) {
  widen<T>(load_raw(p, n), v);
}

// p[0 .. n) = v, each value rounded to T once (to nearest even).
template <typename T>
__device__ __forceinline__ void store_chunk(T* __restrict__ p, int n, const float* v) {
  constexpr int V = kChunk<T>;
  if (n <= 0) return;
  Chunk<T> c;
#pragma unroll
  for (int i = 0; i < V; ++i) c.e[i] = (T)v[i];
  if (n >= V) {
    *reinterpret_cast<u32x4_any*>(p) = c.raw;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < n) p[i] = c.e[i];
  }
}

// EV elements, 2 to 16 bytes, at any element's address.
template <int BYTES>
struct RawOf;
template <>
struct RawOf<16> { typedef u32x4 type; typedef u32x4_any any; };
template <>
struct RawOf<8> { typedef u32x2 type; typedef u32x2_any any; };
typedef uint32_t u32_any __attribute__((aligned(2)));
template <>
struct RawOf<4> { typedef uint32_t type; typedef u32_any any; };
template <>
struct RawOf<2> { typedef uint16_t type; typedef uint16_t any; };

template <typename T, int EV>
union Pack {
  typename RawOf<EV * (int)sizeof(T)>::type raw;
  T e[EV];
  __device__ Pack() {}
};

template <typename T, int EV>
__device__ __forceinline__ Pack<T, EV> load_pack(const T* __restrict__ p, bool ok) {
  Pack<T, EV> c;
  if (ok) {
    c.raw = *reinterpret_cast<const typename RawOf<EV * (int)sizeof(T)>::any*>(p);
  } else {
    c.raw = {};
  }
  return c;
}

template <typename T, int EV>
__device__ __forceinline__ void get(const Pack<T, EV>& c, float (&v)[EV]) {
#pragma unroll
  for (int e = 0; e < EV; ++e) v[e] = (float)c.e[e];
}

template <typename T, int EV>
__device__ __forceinline__ void store_pack(T* __restrict__ p, const float (&v)[EV]) {
  Pack<T, EV> c;
#pragma unroll
  for (int e = 0; e < EV; ++e) c.e[e] = (T)v[e];
  *reinterpret_cast<typename RawOf<EV * (int)sizeof(T)>::any*>(p) = c.raw;
}

// x, rounded to FP32 here: what it is computed by is not joined with a conversion that follows (a product to FP16 is
// otherwise one instruction that rounds once, and differs from the FP32 product rounded in one case of some thousand).
__device__ __forceinline__ float held(float x) {
  asm("" : "+v"(x));
  return x;
}

template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), CTRL, 0xf, 0xf, false));
}

// Sum over the aligned group of LANES lanes, the same bits in each of them: every step adds a lane's partner, and
// the partner adds the lane's own value.
template <int LANES>
__device__ __forceinline__ float lane_sum(float x) {
  if (LANES >= 2) x += dpp<0xB1>(x);    // lane ^ 1
  if (LANES >= 4) x += dpp<0x4E>(x);    // lane ^ 2
  if (LANES >= 8) x += dpp<0x141>(x);   // mirrored in eight: the other quad, whose lanes agree
  if (LANES >= 16) x += dpp<0x140>(x);  // mirrored in sixteen
  if (LANES >= 32) x += __shfl_xor(x, 16);
  if (LANES >= 64) x += __shfl_xor(x, 32);
  return x;
}

// Lanes of a wave that hand values to each other through LDS: what was written before is seen after.  (LDS serves a
// wave's accesses in order, so this holds the compiler only.)
__device__ __forceinline__ void wave_meet() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Block `b` of `blocks` in an order that gives each of the eight dies (blocks go to them in turn) a contiguous part.
__device__ __forceinline__ int die_order(int b, int blocks) {
  const int per = blocks / 8, rest = blocks % 8, die = b & 7;
  return die * per + min(die, rest) + (b >> 3);
}

inline int dense_fail(int code, const char* msg) { return ictc::set_error(code, msg); }

inline int dense_status(const char* what) {
  return hipGetLastError() == hipSuccess ? ICTC_OK : dense_fail(ICTC_ERR_RUNTIME, what);
}

}  // namespace
